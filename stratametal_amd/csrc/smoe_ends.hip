// stratametal_amd/csrc/smoe_ends.hip - the ends of a block on one residual stream (gfx950, wave64): the norm after the
// block, its gate and the residual scales, and the norm before the next block, in one pass over the rows.
//   z = y, or y rs(y) post;  out = res_scale R + y_scale g z;  x = out rs(out) pre;  rs(v) = 1 / sqrt(mean v^2 + eps)
// Every value is read once and written once: memory bound (a row of n f32 values in and out moves 16 n bytes for some 11 n
// operations), latency bound at a few tokens.
#include "smoe_gemv.hpp"
#include "smoe_launch.hpp"
#include "smoe_rules.hpp"
#include "smoe_types.hpp"

#include <type_traits>

namespace smoe {

// a gate for every row; a row's own values; a row's one value
enum { kEndsNoGate = 0, kEndsGateOnce = 1, kEndsGateRow = 2, kEndsGateToken = 3 };

namespace {

// A row's values in a lane's slots of four, as loaded.  VEC: slot m is the 4 values of chunk l + L m (L lanes to a row: a
// load or store of the wave is one run of bytes for every type); else value j of slot m is element l + L (4 m + j).  Those
// past the row hold its last ones (every load is in bounds).
template <bool VEC>
__device__ __forceinline__ int slot_at(int l, int L, int m, int j) {
    return VEC ? 4 * (l + L * m) + j : l + L * (4 * m + j);
}
template <bool VEC, int L, int NV>
__device__ __forceinline__ void load_row(const void* p, int type, int n, int l, u32x4 (&raw)[NV]) {
    if (type == kF32) {
#pragma unroll
        for (int m = 0; m < NV; ++m) {
            if constexpr (VEC) {
                raw[m] = static_cast<const u32x4*>(p)[min(l + L * m, (n >> 2) - 1)];
            } else {
                const uint32_t* q = static_cast<const uint32_t*>(p);
                raw[m] = u32x4{q[min(l + L * (4 * m), n - 1)], q[min(l + L * (4 * m + 1), n - 1)],
                               q[min(l + L * (4 * m + 2), n - 1)], q[min(l + L * (4 * m + 3), n - 1)]};
            }
        }
    } else {
#pragma unroll
        for (int m = 0; m < NV; ++m) {
            if constexpr (VEC) {
                raw[m].xy = static_cast<const u32x2*>(p)[min(l + L * m, (n >> 2) - 1)];
            } else {
                const uint16_t* q = static_cast<const uint16_t*>(p);
                raw[m] = u32x4{q[min(l + L * (4 * m), n - 1)], q[min(l + L * (4 * m + 1), n - 1)],
                               q[min(l + L * (4 * m + 2), n - 1)], q[min(l + L * (4 * m + 3), n - 1)]};
            }
        }
    }
}
template <bool VEC, int NV>
__device__ __forceinline__ void row_values(const u32x4 (&raw)[NV], int type, float (&v)[NV][4]) {
    const auto all = [&](auto which) {  // (one branch for the row)
        constexpr int E = decltype(which)::value;
#pragma unroll
        for (int m = 0; m < NV; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[m][j] = E == kF32 ? u2f(raw[m][j])
                                    : elem_to_f32(!VEC ? raw[m][j] : j & 1 ? raw[m][j >> 1] >> 16 : raw[m][j >> 1] & 0xFFFFu, E);
    };
    if (type == kF32) all(std::integral_constant<int, kF32>{});
    else if (type == kBf16) all(std::integral_constant<int, kBf16>{});
    else all(std::integral_constant<int, kF16>{});
}
template <bool VEC, int L, int NV>
__device__ __forceinline__ void store_row(void* p, int type, int n, int l, const float (&v)[NV][4]) {
    const auto all = [&](auto which) {
        constexpr int E = decltype(which)::value;
#pragma unroll
        for (int m = 0; m < NV; ++m) {
            if constexpr (VEC) {
                const int c = l + L * m;
                if (4 * c < n) store4(static_cast<uint8_t*>(p) + (size_t)c * (4 * elem_bytes(E)), v[m], E);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int d = slot_at<false>(l, L, m, j);
                    if (d < n) store1(p, d, v[m][j], E);
                }
            }
        }
    };
    if (type == kF32) all(std::integral_constant<int, kF32>{});
    else if (type == kBf16) all(std::integral_constant<int, kBf16>{});
    else all(std::integral_constant<int, kF16>{});
}

// The sum of a value over a row's L lanes, in every one of them (s: L / 64 floats of LDS, the work-group's one row's).
template <int L>
__device__ __forceinline__ float row_sum(float v, float* s) {
    if constexpr (L < 64) {
        if constexpr (L == 32) v = v + xor_swap<16>(v);
        v = v + xor_swap<8>(v);
        v = v + xor_swap<4>(v);
        v = v + xor_swap<2>(v);
        return v + xor_swap<1>(v);
    }
    v = wave_sum_xor_fast(v);
    if constexpr (L > 64) {
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        v = s[0];
#pragma unroll
        for (int w = 1; w < L / 64; ++w) v = v + s[w];
    }
    return v;
}

// 1 / sqrt(mean v^2 + eps) of a row.  The squares are summed in f32: a row whose mean square leaves f32's safe range is
// summed again with its values scaled by 2^-80 or 2^80 (one branch for the row: its lanes all hold the same q).
// s: L / 32 floats of LDS, used once between two other barriers.
template <bool VEC, int L, int NV>
__device__ __forceinline__ float row_scale(const float (&v)[NV][4], int n, int l, float eps, float* s) {
    float acc = 0.0f;
#pragma unroll
    for (int m = 0; m < NV; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (slot_at<VEC>(l, L, m, j) < n) acc = __builtin_fmaf(v[m][j], v[m][j], acc);
    const float q = row_sum<L>(acc, s) / (float)n + eps;
    if (!(q > 0x1p120f || q < 0x1p-100f)) return 1.0f / __builtin_sqrtf(q);
    const float f = q > 1.0f ? 0x1p-80f : 0x1p80f;
    acc = 0.0f;
#pragma unroll
    for (int m = 0; m < NV; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (slot_at<VEC>(l, L, m, j) < n) acc = __builtin_fmaf(v[m][j] * f, v[m][j] * f, acc);
    return f / __builtin_sqrtf(row_sum<L>(acc, s + L / 64) / (float)n + eps * f * f);
}

}  // namespace

// L lanes to a row of up to 4 L NV values: 256 / L rows at a time to a work-group, or from 256 lanes on one.  A work-group
// takes every gridDim.x-th set of rows; the next row's values are loaded before this one's are worked on, and what no row
// changes (y_scale post g of a gate per channel, and pre) stays in registers.  With four slots, or two and a gate of every
// value, neither fits the 128 registers of 16 waves: a row's values are loaded when its turn comes, and the weights each
// time where they are used.  Four slots spill all the same (16 to 101 registers, without vectors 70 to 379), as do two
// without vectors and with a gate of every value (40): joins of 4096 rows of 16384 f32 values 226 us, 4.8 TB/s, with a
// gate per channel 340, with one of every value 388, of 16383 394 to 1398; 8192 rows of 8192 207, 206 and 253 us, 5.2
// TB/s.  4096 rows of 4096 f32 values in and out 45 us, 6.0 TB/s of the copy's 5.1 (from the caches in part; 8192 rows 101
// us, 5.3 TB/s); one row of 2048 3.5 us, a launch's latencies.  (Types chosen per value, not per row: a bf16 batch with a
// gate of every value 155 us for 92.)
template <int L, int NV, bool VEC, int GATE>
__global__ __launch_bounds__(L < 256 ? 256 : L) void k_block_ends(const EndsArgs a) {
    constexpr int ROWS = L < 256 ? 256 / L : 1;
    constexpr bool AHEAD = NV < 4 && !(L == 1024 && GATE == kEndsGateRow);
    static_assert(L <= 64 || L >= 256, "a row's lanes are a wave's, or the work-group");
    __shared__ float sum_s[2][L / 16];  // (two rows' in turn: a wave may be one row ahead of another's last read)
    const int l = threadIdx.x % L, n = a.n;
    const bool write = a.y != nullptr;
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int64_t t = (int64_t)blockIdx.x * ROWS + threadIdx.x / L;
    if (t >= a.n_tokens) return;  // (rows within a wave only, and they meet no barrier)
    u32x4 rr[NV], yr[NV], gr[NV];
    float gt = 1.0f;
    const auto load = [&](int64_t row) {
        load_row<VEC, L, NV>(static_cast<const uint8_t*>(a.R) + row * a.r_ld * elem_bytes(a.r_type), a.r_type, n, l, rr);
        if (write) load_row<VEC, L, NV>(static_cast<const uint8_t*>(a.y) + row * a.y_ld * elem_bytes(a.y_type), a.y_type, n, l, yr);
        const float* g = a.gate + row * a.gate_ld;
        if constexpr (GATE == kEndsGateToken) gt = *g;
        if constexpr (GATE == kEndsGateRow) {
            if (a.gate_unit) {
                load_row<VEC, L, NV>(g, kF32, n, l, gr);
            } else {
#pragma unroll
                for (int m = 0; m < NV; ++m)
#pragma unroll
                    for (int j = 0; j < 4; ++j) gr[m][j] = f2u(g[min(slot_at<VEC>(l, L, m, j), n - 1) * a.gate_step]);
            }
        }
    };
    const auto act = [&](float (&g)[NV][4]) {
        if (!a.gate_sigmoid) return;
#pragma unroll
        for (int m = 0; m < NV; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) g[m][j] = sigmoid_fast(g[m][j]);
    };
    // y_scale post [g]
    const auto branch = [&](float (&c)[NV][4]) {
        u32x4 w[NV];
        if (a.post) {
            load_row<VEC, L, NV>(a.post, kF32, n, l, w);
            row_values<VEC, NV>(w, kF32, c);
        }
        float g[NV][4];
        if constexpr (GATE == kEndsGateOnce) {
#pragma unroll
            for (int m = 0; m < NV; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) g[m][j] = a.gate[min(slot_at<VEC>(l, L, m, j), n - 1) * a.gate_step];
            act(g);
        }
#pragma unroll
        for (int m = 0; m < NV; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                c[m][j] = a.post ? a.y_scale * c[m][j] : a.y_scale;
                if constexpr (GATE == kEndsGateOnce) c[m][j] = c[m][j] * g[m][j];
            }
    };
    const auto weight = [&](float (&p)[NV][4]) {
        u32x4 w[NV];
        if (a.pre) {
            load_row<VEC, L, NV>(a.pre, kF32, n, l, w);
            row_values<VEC, NV>(w, kF32, p);
        } else {
#pragma unroll
            for (int m = 0; m < NV; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) p[m][j] = 1.0f;
        }
    };
    float c[NV][4], p[NV][4];
    load(t);
    if constexpr (AHEAD) {
        if (write) branch(c);
        if (a.x) weight(p);
    }
    for (int it = 0; t < a.n_tokens; t += step, ++it) {
        float* s = sum_s[it & 1];
        float v[NV][4];
        if (!AHEAD && it > 0) load(t);
        row_values<VEC, NV>(rr, a.r_type, v);
        if (write) {
            float z[NV][4];
            row_values<VEC, NV>(yr, a.y_type, z);
            if constexpr (GATE == kEndsGateRow) {  // the row's gate, on the side of y (the norm's sum is of z without it)
                float g[NV][4];
                row_values<VEC, NV>(gr, kF32, g);
                act(g);
                if (AHEAD && t + step < a.n_tokens) load(t + step);
                const float rs = a.post ? row_scale<VEC, L, NV>(z, n, l, a.eps, s) : 1.0f;
#pragma unroll
                for (int m = 0; m < NV; ++m)
#pragma unroll
                    for (int j = 0; j < 4; ++j) z[m][j] = (z[m][j] * rs) * g[m][j];
            } else {
                const float g = GATE == kEndsGateToken && a.gate_sigmoid ? sigmoid_fast(gt) : gt;
                if (AHEAD && t + step < a.n_tokens) load(t + step);
                const float rs = a.post ? row_scale<VEC, L, NV>(z, n, l, a.eps, s) : 1.0f;
#pragma unroll
                for (int m = 0; m < NV; ++m)
#pragma unroll
                    for (int j = 0; j < 4; ++j) z[m][j] = GATE == kEndsGateToken ? (z[m][j] * rs) * g : z[m][j] * rs;
            }
            if constexpr (!AHEAD) branch(c);
#pragma unroll
            for (int m = 0; m < NV; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[m][j] = __builtin_fmaf(z[m][j], c[m][j], a.res_scale * v[m][j]);
            store_row<VEC, L, NV>(static_cast<uint8_t*>(a.out) + t * a.out_ld * elem_bytes(a.r_type), a.r_type, n, l, v);
        } else if (AHEAD && t + step < a.n_tokens) {
            load(t + step);
        }
        if (a.x) {
            const float rs = row_scale<VEC, L, NV>(v, n, l, a.eps, s + L / 32);
            if constexpr (!AHEAD) weight(p);
#pragma unroll
            for (int m = 0; m < NV; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[m][j] = (v[m][j] * rs) * p[m][j];
            store_row<VEC, L, NV>(static_cast<uint8_t*>(a.x) + t * a.x_ld * elem_bytes(a.x_type), a.x_type, n, l, v);
        }
    }
}

hipError_t launch_block_ends(const EndsArgs& args, hipStream_t s) {
    EndsArgs a = args;
    const auto al = [](const void* p, int64_t ld, int type) {  // rows of 4-value vectors
        return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * elem_bytes(type))) & (4 * elem_bytes(type) - 1)) == 0;
    };
    const bool vec = a.n % 4 == 0 && al(a.R, a.r_ld, a.r_type) && al(a.y, a.y_ld, a.y_type) &&
                     al(a.out, a.out_ld, a.r_type) && al(a.x, a.x_ld, a.x_type) && al(a.post, 0, kF32) && al(a.pre, 0, kF32);
    a.gate_unit = a.gate_step == 1 && (!vec || al(a.gate, a.gate_ld, kF32));
    const int mode = !a.gate ? kEndsNoGate : a.gate_ld == 0 ? kEndsGateOnce : a.gate_step == 0 ? kEndsGateToken : kEndsGateRow;
    const EndsShape sh = ends_shape(a.n);
    const dim3 grid((unsigned)ends_groups(a.n_tokens, a.n)), block(sh.lanes < 256 ? 256 : sh.lanes);
#define SMOE_ENDS_K(W, V, G)                                                               \
    if (vec) hipLaunchKernelGGL((k_block_ends<W, V, true, G>), grid, block, 0, s, a);      \
    else hipLaunchKernelGGL((k_block_ends<W, V, false, G>), grid, block, 0, s, a)
#define SMOE_ENDS(W, V)                                                              \
    if (sh.lanes == W && sh.slots == V) {                                            \
        if (mode == kEndsNoGate) { SMOE_ENDS_K(W, V, kEndsNoGate); }                 \
        else if (mode == kEndsGateOnce) { SMOE_ENDS_K(W, V, kEndsGateOnce); }        \
        else if (mode == kEndsGateToken) { SMOE_ENDS_K(W, V, kEndsGateToken); }      \
        else { SMOE_ENDS_K(W, V, kEndsGateRow); }                                    \
        return hipGetLastError();                                                    \
    }
    SMOE_ENDS(16, 1) SMOE_ENDS(32, 1) SMOE_ENDS(64, 1) SMOE_ENDS(64, 2) SMOE_ENDS(256, 1) SMOE_ENDS(256, 2) SMOE_ENDS(512, 2)
    SMOE_ENDS(1024, 2) SMOE_ENDS(1024, 4)
#undef SMOE_ENDS
#undef SMOE_ENDS_K
    return hipErrorInvalidValue;
}

}  // namespace smoe
