// stratametal_amd/csrc/smoe_linear.hpp - what the dense products share (smoe_linear.hip, smoe_linear4.hip): the matrix
// instruction, the epilogue (bias, activation, gated pair, residual, one rounding to y's type), the tiles' places and loads.
#pragma once

#include "smoe_dma.hpp"
#include "smoe_gemv.hpp"
#include "smoe_launch.hpp"
#include "smoe_rules.hpp"
#include "smoe_types.hpp"

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

// 1 / (1 + e^-x), the quotient by the hardware's reciprocal (1 ulp).  e^-x = 2^t, t = -x log2 e: t's rounding is at most
// |x| 2^-24 of e^-x, so as much of a small sigmoid(x), and of a large one its part e^-x of that.
__device__ __forceinline__ float act_sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f));
}
// smoe.h's SMOE_ACT_*
__device__ __forceinline__ float activate(float a, int act) {
    switch (act) {
        case 1: return a * act_sigmoid(a);
        // 0.5 a (1 + tanh u) = a sigmoid(2 u), u = sqrt(2 / pi) (a + 0.044715 a^3)
        case 2: return a * act_sigmoid(1.59576912f * a * __builtin_fmaf(0.044715f * a, a, 1.0f));
        case 3: return a > 0.0f || a != a ? a : 0.0f;
        case 4: return a > 0.0f || a != a ? a * a : 0.0f;
        case 5: return act_sigmoid(a);
        default: return a;
    }
}

template <int N>
__device__ __forceinline__ void activate_all(float (&v)[N][4], int act) {
    const auto each = [&](auto which) {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[k][j] = activate(v[k][j], decltype(which)::value);
    };
    switch (act) {
        case 1: each(std::integral_constant<int, 1>{}); break;
        case 2: each(std::integral_constant<int, 2>{}); break;
        case 3: each(std::integral_constant<int, 3>{}); break;
        case 4: each(std::integral_constant<int, 4>{}); break;
        case 5: each(std::integral_constant<int, 5>{}); break;
        default: break;
    }
}

// Output o of token t: g the sum of w, u of w2.
template <bool PAIR>
__device__ __forceinline__ void finish1(const LinearArgs& a, int64_t t, int o, float g, float u) {
    float v = activate(a.bias ? g + a.bias[o] : g, a.act);
    if constexpr (PAIR) v = v * (a.bias2 ? u + a.bias2[o] : u);
    if (a.residual) {
        const int64_t at = t * a.r_ld + o;
        v += a.y_type == kF32 ? static_cast<const float*>(a.residual)[at]
                              : elem_to_f32(static_cast<const uint16_t*>(a.residual)[at], a.y_type);
    }
    store1(a.y, t * a.y_ld + o, v, a.y_type);
}

// Four outputs o .. o + 3 of token t (those below n_out).
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

// The same for tokens t, t + PER, ... (those below t_end) of one lane's outputs, all of them there, rows of vectors; b and c
// are their biases.
template <int BATCH, int PER, bool PAIR>
__device__ __forceinline__ void finish_batch(const LinearArgs& a, int64_t t, int64_t t_end, int o, const float (&b)[4],
                                             const float (&c)[4], const f32x4 (&g)[BATCH], const f32x4 (&u)[BATCH]) {
    const bool f32 = a.y_type == kF32;
    u32x4 r[BATCH];
    if (a.residual && f32) {
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
            r[k] = *reinterpret_cast<const u32x4*>(static_cast<const float*>(a.residual) + min(t + k * PER, t_end - 1) * a.r_ld + o);
    } else if (a.residual) {
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
            r[k].xy = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(a.residual) + min(t + k * PER, t_end - 1) * a.r_ld + o);
    }
    float v[BATCH][4];
#pragma unroll
    for (int k = 0; k < BATCH; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k][j] = g[k][j] + b[j];
    activate_all(v, a.act);
    if constexpr (PAIR) {
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[k][j] = v[k][j] * (u[k][j] + c[j]);
    }
    const auto add = [&](auto type) {  // the residual, of one type for all
        constexpr int E = decltype(type)::value;
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[k][j] += E == kF32 ? u2f(r[k][j]) : elem_to_f32(j & 1 ? r[k][j >> 1] >> 16 : r[k][j >> 1] & 0xFFFFu, E);
    };
    if (a.residual) {
        if (f32) add(std::integral_constant<int, kF32>{});
        else if (a.y_type == kBf16) add(std::integral_constant<int, kBf16>{});
        else add(std::integral_constant<int, kF16>{});
    }
    const auto put = [&](auto type) {
        constexpr int E = decltype(type)::value;
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
            if (t + k * PER < t_end)
                store4(static_cast<uint8_t*>(a.y) + ((t + k * PER) * a.y_ld + o) * elem_bytes(E), v[k], E);
    };
    if (f32) put(std::integral_constant<int, kF32>{});
    else if (a.y_type == kBf16) put(std::integral_constant<int, kBf16>{});
    else put(std::integral_constant<int, kF16>{});
}

// The same of one output, rows of any alignment.
template <int BATCH, int PER, bool PAIR>
__device__ __forceinline__ void finish_column(const LinearArgs& a, int64_t t, int64_t t_end, int o, const float (&g)[BATCH],
                                              const float (&u)[BATCH]) {
    const bool f32 = a.y_type == kF32;
    const float b = a.bias ? a.bias[o] : 0.0f, c = PAIR && a.bias2 ? a.bias2[o] : 0.0f;
    uint32_t r[BATCH];
    if (a.residual) {
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int64_t at = min(t + k * PER, t_end - 1) * a.r_ld + o;
            r[k] = f32 ? static_cast<const uint32_t*>(a.residual)[at] : static_cast<const uint16_t*>(a.residual)[at];
        }
    }
    static_assert(BATCH % 4 == 0, "activate_all");
    float v[BATCH / 4][4];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) v[k / 4][k % 4] = g[k] + b;
    activate_all(v, a.act);
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
        float w = v[k / 4][k % 4];
        if constexpr (PAIR) w = w * (u[k] + c);
        if (a.residual) w += f32 ? u2f(r[k]) : elem_to_f32(r[k], a.y_type);
        if (t + k * PER < t_end) store1(a.y, (t + k * PER) * a.y_ld + o, w, a.y_type);
    }
}

// y and residual rows take 4-value vectors.
__host__ __device__ __forceinline__ bool rows_vec(const LinearArgs& a) {
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

// A wave's loads of a step: load i brings rows 8 (i WAVES + wave) .. + 7 of the tile's weights (i < BM / 8 / WAVES, buffer
// rw), then of its tokens (rx), lane l piece (l & 7) ^ (l >> 3) of row l >> 3, from byte off[i] on at K = 0 (past the buffer
// for a row past the matrix).  PAIR: the tile's 16-row sets are w's and w2's in turn, and a wave's loads all of one of them.
template <int BM, int BN, int WAVES, bool PAIR, int SLOTS>
__device__ __forceinline__ void tile_loads(const LinearArgs& a, int o0, int t0, int n_o, int n_t, int wave, int lane, i32x4& rw,
                                           i32x4& rx, uint32_t (&off)[SLOTS]) {
    constexpr int WS = BM / 8 / WAVES;
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0 && SLOTS == WS + BN / 8 / WAVES, "whole loads");
    static_assert(!PAIR || WAVES % 4 == 0, "a wave's loads all of one matrix");
    const uint32_t wrow = 2u * a.n_in;
    rw = uniform_rsrc(static_cast<const uint8_t*>(PAIR && (wave & 2) ? a.w2 : a.w) + (size_t)o0 * wrow, n_o * wrow);
    rx = uniform_rsrc(static_cast<const uint8_t*>(a.x) + (size_t)t0 * a.x_ld * 2, (uint32_t)((n_t - 1) * a.x_ld * 2) + wrow);
    const int piece = (lane & 7) ^ (lane >> 3);
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        const int row = 8 * ((i < WS ? i : i - WS) * WAVES + wave) + (lane >> 3);
        const int o = PAIR ? (row >> 5) * 16 + (row & 15) : row;
        if (i < WS) off[i] = o < n_o ? o * wrow + 16u * piece : kOob;
        else off[i] = row < n_t ? (uint32_t)(row * a.x_ld * 2) + 16u * piece : kOob;
    }
}

// A wave's MT x NT fragments of sums, outputs from o0 and tokens from t0 (those below t_end) on, through the epilogue, NG
// sets of 16 tokens at a time through the wave's own piece of LDS, so that a token's outputs lie in consecutive lanes: a
// lane's outputs are the same four of every token it takes, its bias is loaded once, and the residual's loads and the
// stores of BATCH tokens go together (one at a time the epilogue of a 256 x 256 tile took 36 us).
template <int MT>
constexpr int kStoreRow = 64 * MT + 16;  // bytes of a token's sums, and 16 that spread the tokens over the banks
template <int MT, int NG>
constexpr int kStoreBytes = 16 * NG * kStoreRow<MT>;
template <int MT, int NT, int NG, bool PAIR>
__device__ __forceinline__ void tile_store(const LinearArgs& a, const f32x4 (&acc)[MT][NT], uint8_t* mine, int o0, int t0,
                                           int t_end, int lane) {
    constexpr int ROW = kStoreRow<MT>;
    constexpr int QUADS = 4 * MT / (PAIR ? 2 : 1);  // quads of outputs of a token
    constexpr int PER = 64 / QUADS;                 // tokens of an access
    constexpr int BATCH = 16 * NG / PER < 8 ? 16 * NG / PER : 8;
    static_assert(!PAIR || MT % 2 == 0, "sets in pairs");
    static_assert(NT % NG == 0 && 64 % QUADS == 0 && 16 * NG / PER % BATCH == 0, "whole batches");
    const int q = lane % QUADS, o = o0 + 4 * q;
    const bool vec = rows_vec(a) && a.n_out % 4 == 0 && gridDim.y == 1;
    float b[4], c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int oc = min(o + j, a.n_out - 1);
        b[j] = a.bias ? a.bias[oc] : 0.0f;
        c[j] = PAIR && a.bias2 ? a.bias2[oc] : 0.0f;
    }
#pragma unroll
    for (int n = 0; n < NT; n += NG) {
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int m = 0; m < MT; ++m)
                *reinterpret_cast<f32x4*>(mine + (16 * i + (lane & 15)) * ROW + m * 64 + (lane >> 4) * 16) = acc[m][n + i];
        const uint8_t* at = mine + (lane / QUADS) * ROW + (PAIR ? (q >> 2) * 128 + (q & 3) * 16 : q * 16);
        const int t1 = t0 + n * 16 + lane / QUADS;
        if (vec) {
#pragma unroll 1
            for (int i = 0; i < 16 * NG / PER && o < a.n_out; i += BATCH) {
                f32x4 g[BATCH], u[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    g[k] = *reinterpret_cast<const f32x4*>(at + (i + k) * PER * ROW);
                    u[k] = PAIR ? *reinterpret_cast<const f32x4*>(at + (i + k) * PER * ROW + 64) : g[k];
                }
                finish_batch<BATCH, PER, PAIR>(a, t1 + i * PER, t_end, o, b, c, g, u);
            }
        } else if (gridDim.y > 1) {
#pragma unroll 1
            for (int i = 0; i < 16 * NG / PER; ++i) {
                const int t = t1 + i * PER;
                if (t < t_end && o < a.n_out)
                    put_part<PAIR>(a, blockIdx.y, t, o, *reinterpret_cast<const f32x4*>(at + i * PER * ROW),
                                   *reinterpret_cast<const f32x4*>(at + i * PER * ROW + (PAIR ? 64 : 0)));
            }
        } else {  // rows that take no vectors: lanes take consecutive outputs of a token, a lane the same one of several
            constexpr int OUTS = 4 * QUADS, W = OUTS < 64 ? OUTS : 64, PER1 = 64 / W, ALL = 16 * NG / PER1;
            constexpr int B = ALL < 16 ? ALL : 16;
            const int t2 = t0 + n * 16 + lane / W;
#pragma unroll 1
            for (int oc = lane % W; oc < OUTS && o0 + oc < a.n_out; oc += W) {
                const uint8_t* v = mine + lane / W * ROW + 4 * (PAIR ? oc / 16 * 32 + oc % 16 : oc);
#pragma unroll 1
                for (int i = 0; i < ALL; i += B) {
                    float g[B], u[B];
#pragma unroll
                    for (int k = 0; k < B; ++k) {
                        g[k] = *reinterpret_cast<const float*>(v + (i + k) * PER1 * ROW);
                        u[k] = PAIR ? *reinterpret_cast<const float*>(v + (i + k) * PER1 * ROW + 64) : 0.0f;
                    }
                    finish_column<B, PER1, PAIR>(a, t2 + i * PER1, t_end, o0 + oc, g, u);
                }
            }
        }
    }
}

}  // namespace smoe
