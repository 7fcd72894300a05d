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

}  // namespace

// A tile of BM = 16 MT WM weight rows by BN = 16 NT WN tokens per work-group of WM WN waves, MT x NT fragments of 16 x 16
// to a wave; K in steps of 64 through two LDS buffers, the next step's loads in flight while this one is multiplied.  A row's
// step is eight 16-byte pieces, piece c of row r at place c ^ (r & 7), so that the 16 rows of a fragment's read spread over
// the banks.  PAIR: the tile's 16-row sets are w's and w2's in turn, so that a lane holds both sums of its outputs.
template <int MT, int NT, int WM, int WN, bool PAIR, bool F16>
__global__ __launch_bounds__(64 * WM * WN) void k_linear_tile(const LinearArgs a) {
    constexpr int WAVES = WM * WN, BM = 16 * MT * WM, BN = 16 * NT * WN;
    constexpr int OUTS = PAIR ? BM / 2 : BM;           // outputs of the tile
    constexpr int SLOTS = (BM + BN) / 8 / WAVES;       // loads of a wave per step, 8 rows each
    static_assert((BM + BN) % (8 * WAVES) == 0 && (!PAIR || MT % 2 == 0), "whole loads; sets in pairs");
    __shared__ __align__(1024) uint8_t lds[2][(BM + BN) * 128];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int o0 = blockIdx.x * OUTS, t0 = blockIdx.y * BN;
    const int n_o = min(OUTS, a.n_out - o0), n_t = min(BN, a.n_tokens - t0);
    const uint32_t wrow = 2u * a.n_in;
    const i32x4 rw = buffer_rsrc(static_cast<const uint8_t*>(a.w) + (size_t)o0 * wrow, n_o * wrow);
    const i32x4 rw2 = PAIR ? buffer_rsrc(static_cast<const uint8_t*>(a.w2) + (size_t)o0 * wrow, n_o * wrow) : rw;
    const i32x4 rx = buffer_rsrc(static_cast<const uint8_t*>(a.x) + (size_t)t0 * a.x_ld * 2,
                                 (uint32_t)((n_t - 1) * a.x_ld * 2) + wrow);
    // slot s of the wave: rows 8 (wave SLOTS + s) .. + 7 of the tile; lane: row l >> 3, place l & 7
    uint32_t off[SLOTS];
    const int piece = (lane & 7) ^ (lane >> 3);
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        const int row = 8 * (wave * SLOTS + s) + (lane >> 3);
        if (row < BM) {
            const int o = PAIR ? (row >> 5) * 16 + (row & 15) : row;
            off[s] = o < n_o ? o * wrow + 16u * piece : kOob;
        } else {
            const int t = row - BM;
            off[s] = t < n_t ? (uint32_t)(t * a.x_ld * 2) + 16u * piece : kOob;
        }
    }
    const int steps = (a.n_in + 63) / 64;
    const auto load = [&](int u) {
        const uint32_t base = lds_addr(lds[u & 1]);
        const bool in = u * 64 + 8 * piece < a.n_in;  // (a last short step: zeros past the row)
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int row = 8 * (wave * SLOTS + s);
            const i32x4 r = row >= BM ? rx : PAIR && (row & 16) ? rw2 : rw;
            dma16(base + row * 128, in && off[s] != kOob ? off[s] + 128u * u : kOob, r, 0);
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    load(0);
    const int fr = lane & 15;
    for (int u = 0; u < steps; ++u) {
        vmcnt<0>();
        __syncthreads();  // step u is in LDS, and every wave is done with the buffer that step u + 1 overwrites
        if (u + 1 < steps) load(u + 1);
        const uint8_t* wb = lds[u & 1] + (wm * MT * 16 + fr) * 128;
        const uint8_t* xb = lds[u & 1] + (BM + wn * NT * 16 + fr) * 128;
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
    const bool vec = rows_vec(a);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int t = (wn * NT + n) * 16 + fr;
        if (t >= n_t) continue;
#pragma unroll
        for (int m = 0; m < MT; m += PAIR ? 2 : 1) {
            const int set = wm * MT + m;
            const int o = o0 + (PAIR ? set / 2 : set) * 16 + 4 * (lane >> 4);
            if (o >= a.n_out) continue;
            const f32x4 q = acc[m][n], p = acc[PAIR ? m + 1 : m][n];
            finish4<PAIR>(a, vec, t0 + t, o, {q[0], q[1], q[2], q[3]}, {p[0], p[1], p[2], p[3]});
        }
    }
}

size_t linear_part_bytes(int64_t, int, int, bool) { return 0; }

hipError_t launch_linear(const LinearArgs& a, hipStream_t s) {
    const auto go = [&](auto pair, auto f16) {
        constexpr bool P = decltype(pair)::value;
        const dim3 grid((a.n_out + (P ? 31 : 63)) / (P ? 32 : 64), (a.n_tokens + 63) / 64);
        hipLaunchKernelGGL((k_linear_tile<2, 2, 2, 2, P, decltype(f16)::value>), grid, dim3(256), 0, s, a);
    };
    const std::true_type yes;
    const std::false_type no;
    if (a.w2) a.w_type == kF16 ? go(yes, yes) : go(yes, no);
    else a.w_type == kF16 ? go(no, yes) : go(no, no);
    return hipGetLastError();
}

}  // namespace smoe
