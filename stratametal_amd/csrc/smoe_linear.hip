// stratametal_amd/csrc/smoe_linear.hip - the dense product with bias, activation and residual in its epilogue (gfx950,
// wave64): y[t][o] = act(sum_i x[t][i] w[o][i] + bias[o]) [* (sum_i x[t][i] w2[o][i] + bias2[o])] [+ residual[t][o]],
// x and w bf16 or fp16, sums in f32 on the matrix cores, one rounding to y's type.
#include "smoe_dma.hpp"
#include "smoe_gemv.hpp"
#include "smoe_launch.hpp"
#include "smoe_rules.hpp"
#include "smoe_types.hpp"

#include <type_traits>

namespace smoe {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <bool F16>
__device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                       0);
}

// smoe.h's SMOE_ACT_*
__device__ __forceinline__ float activate(float a, int act) {
    switch (act) {
        case 1: return a * sigmoid_fast(a);
        // 0.5 a (1 + tanh u) = a sigmoid(2 u), u = sqrt(2 / pi) (a + 0.044715 a^3)
        case 2: return a * sigmoid_fast(1.59576912f * a * __builtin_fmaf(0.044715f * a, a, 1.0f));
        case 3: return a > 0.0f || a != a ? a : 0.0f;
        case 4: return a > 0.0f || a != a ? a * a : 0.0f;
        case 5: return sigmoid_fast(a);
        default: return a;
    }
}

// Four outputs o .. o + 3 of token t (those below n_out): g the sums of w, u of w2.
template <bool PAIR>
__device__ __forceinline__ void finish4(const LinearArgs& a, bool vec, int64_t t, int o, const float (&g)[4],
                                        const float (&u)[4]) {
    float v[4], r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const bool f32 = a.y_type == kF32;
    uint8_t* y = static_cast<uint8_t*>(a.y) + (t * a.y_ld + o) * (f32 ? 4 : 2);
    const uint8_t* res = a.residual ? static_cast<const uint8_t*>(a.residual) + (t * a.r_ld + o) * (f32 ? 4 : 2) : nullptr;
    vec = vec && o + 4 <= a.n_out;
    if (res) {
        if (vec && f32) {
            const float4 q = *reinterpret_cast<const float4*>(res);
            r[0] = q.x, r[1] = q.y, r[2] = q.z, r[3] = q.w;
        } else if (vec) {
            const uint2 q = *reinterpret_cast<const uint2*>(res);
            r[0] = elem_to_f32(q.x & 0xFFFFu, a.y_type), r[1] = elem_to_f32(q.x >> 16, a.y_type);
            r[2] = elem_to_f32(q.y & 0xFFFFu, a.y_type), r[3] = elem_to_f32(q.y >> 16, a.y_type);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (o + i < a.n_out)
                    r[i] = f32 ? reinterpret_cast<const float*>(res)[i]
                               : elem_to_f32(reinterpret_cast<const uint16_t*>(res)[i], a.y_type);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int oc = min(o + i, a.n_out - 1);
        v[i] = activate(a.bias ? g[i] + a.bias[oc] : g[i], a.act);
        if constexpr (PAIR) v[i] = v[i] * (a.bias2 ? u[i] + a.bias2[oc] : u[i]);
        if (res) v[i] = v[i] + r[i];
    }
    if (vec && f32) {
        *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (vec) {
        *reinterpret_cast<uint2*>(y) = make_uint2(pack_half2(v[0], v[1], a.y_type), pack_half2(v[2], v[3], a.y_type));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (o + i < a.n_out) store1(y, i, v[i], a.y_type);
    }
}

// y and residual rows take 4-value vectors.
__device__ __forceinline__ bool rows_vec(const LinearArgs& a) {
    const uintptr_t m = (a.y_type == kF32 ? 16 : 8) - 1;
    return ((reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.residual)) & m) == 0 &&
           ((a.y_ld | (a.residual ? a.r_ld : 0)) & 3) == 0;
}

// buffer_rsrc of a base that is the same in every lane, in scalar registers whatever the compiler sees of that.
__device__ __forceinline__ i32x4 uniform_rsrc(const void* base, uint32_t bytes) {
    i32x4 r = buffer_rsrc(base, bytes);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_readfirstlane(r[i]);
    return r;
}

// The sums of a slice of K: [slice][w, w2][token][n_out rounded up to 4].
template <bool PAIR>
__device__ __forceinline__ f32x4* part_at(const LinearArgs& a, int slice, int which, int64_t t, int o) {
    const int64_t quads = (a.n_out + 3) / 4;
    return reinterpret_cast<f32x4*>(a.part) + (((int64_t)slice * (PAIR ? 2 : 1) + which) * a.n_tokens + t) * quads + (o >> 2);
}
template <bool PAIR>
__device__ __forceinline__ void put_part(const LinearArgs& a, int slice, int64_t t, int o, f32x4 g, f32x4 u) {
    *part_at<PAIR>(a, slice, 0, t, o) = g;
    if constexpr (PAIR) *part_at<PAIR>(a, slice, 1, t, o) = u;
}

}  // namespace

// The K loop's ring of STAGES LDS buffers: a wave waits until its loads of all but the `after` newest steps are done.
template <int SLOTS, int STAGES>
__device__ __forceinline__ void wait_steps(int after) {
    if (STAGES > 2 && after >= STAGES - 2) vmcnt<(STAGES - 2) * SLOTS>();
    else if (STAGES > 3 && after == STAGES - 3) vmcnt<(STAGES - 3) * SLOTS>();
    else vmcnt<0>();
}

// The tile of work-group i of n: consecutive work-groups go to the 8 XCDs in turn, so XCD x takes the x-th eighth of the
// tiles; in it, bands of kBand token tiles are walked output tile by output tile, so that the tiles at work together share
// rows of both matrices in that XCD's L2.
constexpr int kBand = 4;
__device__ __forceinline__ void tile_of(int i, int n, int tiles_o, int tiles_t, int& o, int& t) {
    const int q = n / 8, r = n % 8, x = i % 8;
    const int j = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + i / 8;
    const int band = j / (kBand * tiles_o), in = j % (kBand * tiles_o);
    const int rows = min(kBand, tiles_t - band * kBand);
    t = band * kBand + in % rows;
    o = in / rows;
}

// A tile of BM = 16 MT WM weight rows by BN = 16 NT WN tokens per work-group of WM WN waves, MT x NT fragments of 16 x 16
// to a wave; K in steps of 64 through a ring of STAGES LDS buffers, filled by loads that write LDS directly.  A row's step is
// eight 16-byte pieces, piece c of row r at place c ^ (r & 7), so that the 16 rows of a fragment's read spread over the
// banks.  PAIR: the tile's 16-row sets are w's and w2's in turn, so that a lane holds both sums of its outputs.
// blockIdx.y: a slice of K, whose sums go to `part` ([slice][w, w2][token][n_out]) for k_linear_join.
template <int MT, int NT, int WM, int WN, int STAGES, bool PAIR, bool F16>
__global__ __launch_bounds__(64 * WM * WN) void k_linear_tile(const LinearArgs a, int tiles_o, int tiles_t) {
    constexpr int WAVES = WM * WN, BM = 16 * MT * WM, BN = 16 * NT * WN;
    constexpr int OUTS = PAIR ? BM / 2 : BM;           // outputs of the tile
    constexpr int WS = BM / 8 / WAVES, XS = BN / 8 / WAVES, SLOTS = WS + XS;  // a wave's loads of a step, 8 rows each
    constexpr int STEP = (BM + BN) * 128;              // bytes of a step
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole loads");
    static_assert(!PAIR || (MT % 2 == 0 && WAVES % 4 == 0), "sets in pairs, a wave's loads all of one matrix");
    static_assert(STAGES >= 2 && STAGES <= 4, "wait_steps");
    __shared__ __align__(1024) uint8_t lds[STAGES * STEP];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    int to, tt;
    tile_of(blockIdx.x, gridDim.x, tiles_o, tiles_t, to, tt);
    const int o0 = to * OUTS, t0 = tt * BN;
    const int n_o = min(OUTS, a.n_out - o0), n_t = min(BN, a.n_tokens - t0);
    const uint32_t wrow = 2u * a.n_in;
    // load i of the wave: rows 8 (i WAVES + wave) .. + 7 of the weights, then of the tokens; lane: row l >> 3, place l & 7
    const void* wm_at = PAIR && (wave & 2) ? a.w2 : a.w;
    const i32x4 rw = uniform_rsrc(static_cast<const uint8_t*>(wm_at) + (size_t)o0 * wrow, n_o * wrow);
    const i32x4 rx = uniform_rsrc(static_cast<const uint8_t*>(a.x) + (size_t)t0 * a.x_ld * 2,
                                  (uint32_t)((n_t - 1) * a.x_ld * 2) + wrow);
    uint32_t off[SLOTS];
    const int piece = (lane & 7) ^ (lane >> 3);
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        const int row = 8 * ((i < WS ? i : i - WS) * WAVES + wave) + (lane >> 3);
        const int o = PAIR ? (row >> 5) * 16 + (row & 15) : row;
        if (i < WS) off[i] = o < n_o ? o * wrow + 16u * piece : kOob;
        else off[i] = row < n_t ? (uint32_t)(row * a.x_ld * 2) + 16u * piece : kOob;
    }
    const int all = (a.n_in + 63) / 64;
    const int u0 = (int)((int64_t)all * blockIdx.y / gridDim.y), u1 = (int)((int64_t)all * (blockIdx.y + 1) / gridDim.y);
    const auto load = [&](int u) {
        const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(lds) + (u - u0) % STAGES * STEP + wave * 1024);
        const bool in = u * 64 + 8 * piece < a.n_in;  // (a last short step: zeros past the row)
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)  // (a row past the matrix stays past the buffer)
            dma16(base + (i < WS ? i * WAVES * 1024 : BM * 128 + (i - WS) * WAVES * 1024),
                  in ? off[i] + 128u * u : kOob, i < WS ? rw : rx, 0);
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
        if (u0 + i < u1) load(u0 + i);
    const int fr = lane & 15;
    for (int u = u0; u < u1; ++u) {
        wait_steps<SLOTS, STAGES>(u1 - 1 - u);
        __syncthreads();  // step u is in LDS, and every wave is done with the buffer that the next load overwrites
        if (u + STAGES - 1 < u1) load(u + STAGES - 1);
        const uint8_t* step = lds + (u - u0) % STAGES * STEP;
        const uint8_t* wb = step + (wm * MT * 16 + fr) * 128;
        const uint8_t* xb = step + (BM + wn * NT * 16 + fr) * 128;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int at = ((4 * kk + (lane >> 4)) ^ (fr & 7)) * 16;
            uint4 av[MT], bv[NT];
#pragma unroll
            for (int m = 0; m < MT; ++m) av[m] = *reinterpret_cast<const uint4*>(wb + m * 2048 + at);
#pragma unroll
            for (int n = 0; n < NT; ++n) bv[n] = *reinterpret_cast<const uint4*>(xb + n * 2048 + at);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[m][n] = mfma16<F16>(av[m], bv[n], acc[m][n]);
        }
    }
    // The epilogue by 16 tokens at a time through the wave's own piece of LDS, so that a token's outputs lie in consecutive
    // lanes (and the fragments' registers are named by constants in a short loop).
    constexpr int ROW = 64 * MT + 16;                  // bytes of a token's sums, and 16 that spread the tokens over the banks
    constexpr int QUADS = 4 * MT / (PAIR ? 2 : 1);     // quads of outputs of a token
    static_assert(WAVES * 16 * ROW <= STAGES * STEP, "the waves' pieces");
    __syncthreads();
    uint8_t* mine = lds + wave * 16 * ROW;
    const bool vec = rows_vec(a);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
            *reinterpret_cast<f32x4*>(mine + fr * ROW + m * 64 + (lane >> 4) * 16) = acc[m][n];
#pragma unroll 1
        for (int i = lane; i < 16 * QUADS; i += 64) {
            const int tr = i / QUADS, q = i % QUADS;
            const int t = (wn * NT + n) * 16 + tr, o = o0 + wm * (4 * QUADS) + 4 * q;
            const uint8_t* at = mine + tr * ROW + (PAIR ? (q >> 2) * 128 + (q & 3) * 16 : q * 16);
            const f32x4 g = *reinterpret_cast<const f32x4*>(at), u = *reinterpret_cast<const f32x4*>(at + (PAIR ? 64 : 0));
            if (t < n_t && o < a.n_out) {
                if (gridDim.y == 1)
                    finish4<PAIR>(a, vec, t0 + t, o, {g[0], g[1], g[2], g[3]}, {u[0], u[1], u[2], u[3]});
                else put_part<PAIR>(a, blockIdx.y, t0 + t, o, g, u);
            }
        }
    }
}

// A few tokens: 16 outputs to a work-group (PAIR: of both matrices), its WAVES waves each every WAVES-th 64 of K, straight
// from memory to the matrix instruction's layout: lane l holds row (or token) l & 15, values 8 (l >> 4) .. of a 32-value
// step.  Bound by the weights' bytes: up to LOADS of a lane's weight loads are on their way together.  Tokens in NT sets of 16
// (lanes past the last token hold its values, and their results are dropped); the waves' sums meet in LDS, in wave order.
template <int NT, int WAVES, bool PAIR, bool F16>
__global__ __launch_bounds__(64 * WAVES) void k_linear_few(const LinearArgs a) {
    constexpr int SETS = PAIR ? 2 : 1, BLOCKS = 4;  // blocks of 64 of K on their way
    __shared__ f32x4 sum_s[WAVES][SETS * NT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int o0 = blockIdx.x * 16;
    const int row = min(o0 + (lane & 15), a.n_out - 1), kq = 8 * (lane >> 4);
    const uint16_t* wp[SETS];
    wp[0] = static_cast<const uint16_t*>(a.w) + (size_t)row * a.n_in;
    if constexpr (PAIR) wp[1] = static_cast<const uint16_t*>(a.w2) + (size_t)row * a.n_in;
    const uint16_t* xp[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
        xp[n] = static_cast<const uint16_t*>(a.x) + min(16 * n + (lane & 15), a.n_tokens - 1) * a.x_ld;
    const int all = (a.n_in + 63) / 64;
    const int u0 = (int)((int64_t)all * blockIdx.y / gridDim.y), u1 = (int)((int64_t)all * (blockIdx.y + 1) / gridDim.y);
    f32x4 acc[SETS][NT];
#pragma unroll
    for (int i = 0; i < SETS; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[i][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int u = u0 + wave; u < u1; u += BLOCKS * WAVES) {
        uint4 wv[BLOCKS][2][SETS], xv[BLOCKS][2][NT];
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = min((u + b * WAVES) * 64 + 32 * h + kq, a.n_in - 8);
#pragma unroll
                for (int i = 0; i < SETS; ++i) wv[b][h][i] = *reinterpret_cast<const uint4*>(wp[i] + k);
#pragma unroll
                for (int n = 0; n < NT; ++n) xv[b][h][n] = *reinterpret_cast<const uint4*>(xp[n] + k);
            }
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // (past the slice or the row: zeros of both, whatever the last values are)
                const bool in = u + b * WAVES < u1 && (u + b * WAVES) * 64 + 32 * h + kq < a.n_in;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint4 x = in ? xv[b][h][n] : zero;
#pragma unroll
                    for (int i = 0; i < SETS; ++i) acc[i][n] = mfma16<F16>(in ? wv[b][h][i] : zero, x, acc[i][n]);
                }
            }
    }
#pragma unroll
    for (int i = 0; i < SETS; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) sum_s[wave][i * NT + n][lane] = acc[i][n];
    __syncthreads();
    const bool vec = rows_vec(a);
    for (int n = wave; n < NT; n += WAVES) {
        f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int i = 0; i < SETS; ++i) {
            s[i] = sum_s[0][i * NT + n][lane];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) s[i] = s[i] + sum_s[w][i * NT + n][lane];
        }
        const int t = 16 * n + (lane & 15), o = o0 + 4 * (lane >> 4);
        if (t >= a.n_tokens || o >= a.n_out) continue;
        if (gridDim.y == 1) finish4<PAIR>(a, vec, t, o, {s[0][0], s[0][1], s[0][2], s[0][3]}, {s[1][0], s[1][1], s[1][2], s[1][3]});
        else put_part<PAIR>(a, blockIdx.y, t, o, s[0], s[1]);
    }
}

// The slices' sums added in order, and the epilogue: four outputs of a token to a thread.
template <bool PAIR>
__global__ __launch_bounds__(256) void k_linear_join(const LinearArgs a, int slices) {
    const int quads = (a.n_out + 3) / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.n_tokens * quads) return;
    const int64_t t = i / quads;
    const int o = (int)(i % quads) * 4;
    float g[4] = {0, 0, 0, 0}, u[4] = {0, 0, 0, 0};
    for (int s = 0; s < slices; ++s) {
        const f32x4 q = *part_at<PAIR>(a, s, 0, t, o);
#pragma unroll
        for (int j = 0; j < 4; ++j) g[j] += q[j];
        if constexpr (PAIR) {
            const f32x4 p = *part_at<PAIR>(a, s, 1, t, o);
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] += p[j];
        }
    }
    finish4<PAIR>(a, rows_vec(a), t, o, g, u);
}

size_t linear_part_bytes(int64_t T, int K, int N, bool pair) {
    const int slices = linear_plan(T, K, N, pair).slices;
    return slices > 1 ? (size_t)slices * (pair ? 2 : 1) * T * ((N + 3) / 4) * 16 : 0;
}

namespace {
template <int MT, int NT, int WM, int WN, int STAGES, bool PAIR, bool F16>
hipError_t launch_tile(const LinearArgs& a, int slices, hipStream_t s) {
    constexpr int OUTS = 16 * MT * WM / (PAIR ? 2 : 1), BN = 16 * NT * WN;
    const int tiles_o = (a.n_out + OUTS - 1) / OUTS, tiles_t = (a.n_tokens + BN - 1) / BN;
    hipLaunchKernelGGL((k_linear_tile<MT, NT, WM, WN, STAGES, PAIR, F16>), dim3(tiles_o * tiles_t, slices),
                       dim3(64 * WM * WN), 0, s, a, tiles_o, tiles_t);
    return hipGetLastError();
}
template <bool PAIR, bool F16>
hipError_t launch_linear_as(const LinearArgs& a, const LinearPlan& p, hipStream_t s) {
    hipError_t e = hipErrorInvalidValue;
    const dim3 few((a.n_out + 15) / 16, p.slices);
#define SMOE_FEW(N, W) \
    if (p.kind == kLinearFew && p.a == N && p.b == W) { \
        hipLaunchKernelGGL((k_linear_few<N, W, PAIR, F16>), few, dim3(64 * W), 0, s, a); \
        e = hipGetLastError(); \
    }
    SMOE_FEW(1, 4) SMOE_FEW(1, 8) SMOE_FEW(1, 16) SMOE_FEW(2, 4) SMOE_FEW(2, 8)
#undef SMOE_FEW
    if (p.kind == kLinearTile) {
        if (p.a == 256) e = launch_tile<8, 4, 2, 4, 2, PAIR, F16>(a, p.slices, s);
        else if (p.a == 128 && p.b == 128) e = launch_tile<4, 4, 2, 2, 2, PAIR, F16>(a, p.slices, s);
        else if (p.a == 128 && p.b == 64) e = launch_tile<4, 2, 2, 2, 3, PAIR, F16>(a, p.slices, s);
        else if (p.a == 64 && p.b == 64) e = launch_tile<2, 2, 2, 2, 4, PAIR, F16>(a, p.slices, s);
    }
    if (e != hipSuccess || p.slices == 1) return e;
    const int64_t quads = (int64_t)a.n_tokens * ((a.n_out + 3) / 4);
    hipLaunchKernelGGL(k_linear_join<PAIR>, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, a, p.slices);
    return hipGetLastError();
}
}  // namespace

hipError_t launch_linear(const LinearArgs& a, hipStream_t s) {
    const LinearPlan p = linear_plan(a.n_tokens, a.n_in, a.n_out, a.w2 != nullptr);
    const bool f16 = a.w_type == kF16;
    if (a.w2) return f16 ? launch_linear_as<true, true>(a, p, s) : launch_linear_as<true, false>(a, p, s);
    return f16 ? launch_linear_as<false, true>(a, p, s) : launch_linear_as<false, false>(a, p, s);
}

}  // namespace smoe
