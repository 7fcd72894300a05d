// stratametal_amd/csrc/smoe_ends.hip - the ends of a block on one residual stream (gfx950, wave64): the norm after the
// block, its gate and the residual scales, and the norm before the next block, in one pass over the rows.
//   z = y, or y rs(y) post;  out = res_scale R + y_scale g z;  x = out rs(out) pre;  rs(v) = 1 / sqrt(mean v^2 + eps)
// Every value is read once and written once: memory bound (a row of n f32 values in and out moves 16 n bytes for some 11 n
// operations), latency bound at a few tokens.
#include "smoe_gemv.hpp"
#include "smoe_launch.hpp"
#include "smoe_rules.hpp"
#include "smoe_types.hpp"

namespace smoe {

namespace {

// A row's values in a lane's slots, as loaded.  VEC: slot m is the 8 values of chunk l + L m (L lanes to a row); else
// value j of slot m is element l + L (8 m + j).  Those past the row hold its last ones (every load is in bounds).
template <bool VEC>
__device__ __forceinline__ int slot_at(int l, int L, int m, int j) {
    return VEC ? 8 * (l + L * m) + j : l + L * (8 * m + j);
}
template <bool VEC, int L, int NV>
__device__ __forceinline__ void load_row(const void* p, int type, int n, int l, Raw8 (&raw)[NV]) {
    if constexpr (VEC) {
        const int last = (n >> 3) - 1;
        if (type == kF32) {
#pragma unroll
            for (int m = 0; m < NV; ++m) {
                const uint4* q = static_cast<const uint4*>(p) + 2 * min(l + L * m, last);
                raw[m].a = q[0];
                raw[m].b = q[1];
            }
        } else {
#pragma unroll
            for (int m = 0; m < NV; ++m) raw[m].a = static_cast<const uint4*>(p)[min(l + L * m, last)];
        }
    } else {
#pragma unroll
        for (int m = 0; m < NV; ++m) {
            uint32_t v[8];
            if (type == kF32) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = static_cast<const uint32_t*>(p)[min(slot_at<false>(l, L, m, j), n - 1)];
                raw[m].a = make_uint4(v[0], v[1], v[2], v[3]);
                raw[m].b = make_uint4(v[4], v[5], v[6], v[7]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = static_cast<const uint16_t*>(p)[min(slot_at<false>(l, L, m, j), n - 1)];
                raw[m].a = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
            }
        }
    }
}
template <bool VEC, int L, int NV>
__device__ __forceinline__ void store_row(void* p, int type, int n, int l, const float (&v)[NV][8]) {
#pragma unroll
    for (int m = 0; m < NV; ++m) {
        if constexpr (VEC) {
            const int c = l + L * m;
            if (8 * c < n) store8(static_cast<uint8_t*>(p) + (size_t)c * (8 * elem_bytes(type)), v[m], type);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int d = slot_at<false>(l, L, m, j);
                if (d < n) store1(p, d, v[m][j], type);
            }
        }
    }
}

// The sum of a value over a row's WAVES waves, in every lane (s: WAVES floats of LDS, the work-group's one row's).
template <int WAVES>
__device__ __forceinline__ float row_sum(float v, float* s) {
    v = wave_sum_xor_fast(v);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        v = s[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v = v + s[w];
    }
    return v;
}

// 1 / sqrt(mean v^2 + eps) of a row.  The squares are summed in f32: a row whose mean square leaves f32's safe range is
// summed again with its values scaled by 2^-80 or 2^80 (one branch for the row: its lanes all hold the same q).
// s: 2 WAVES floats of LDS, used once.
template <int WAVES, bool VEC, int L, int NV>
__device__ __forceinline__ float row_scale(const float (&v)[NV][8], int n, int l, float eps, float* s) {
    float acc = 0.0f;
#pragma unroll
    for (int m = 0; m < NV; ++m)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (slot_at<VEC>(l, L, m, j) < n) acc = __builtin_fmaf(v[m][j], v[m][j], acc);
    const float q = row_sum<WAVES>(acc, s) / (float)n + eps;
    if (!(q > 0x1p120f || q < 0x1p-100f)) return 1.0f / __builtin_sqrtf(q);
    const float f = q > 1.0f ? 0x1p-80f : 0x1p80f;
    acc = 0.0f;
#pragma unroll
    for (int m = 0; m < NV; ++m)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (slot_at<VEC>(l, L, m, j) < n) acc = __builtin_fmaf(v[m][j] * f, v[m][j] * f, acc);
    return f / __builtin_sqrtf(row_sum<WAVES>(acc, s + WAVES) / (float)n + eps * f * f);
}

}  // namespace

// WAVES waves to a row of up to 512 WAVES NV values: four rows to a work-group of one-wave rows, else one.
template <int WAVES, int NV, bool VEC>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void k_block_ends(const EndsArgs a) {
    constexpr int L = 64 * WAVES, ROWS = WAVES == 1 ? 4 : 1;
    __shared__ float sum_s[4 * WAVES];
    const int l = threadIdx.x % L, n = a.n;
    const int64_t t = (int64_t)blockIdx.x * ROWS + threadIdx.x / L;
    if (t >= a.n_tokens) return;  // (one-wave rows only, and they meet no barrier)
    const bool write = a.y != nullptr;
    Raw8 rr[NV], yr[NV];
    load_row<VEC, L, NV>(static_cast<const uint8_t*>(a.R) + t * a.r_ld * elem_bytes(a.r_type), a.r_type, n, l, rr);
    if (write) load_row<VEC, L, NV>(static_cast<const uint8_t*>(a.y) + t * a.y_ld * elem_bytes(a.y_type), a.y_type, n, l, yr);
    float v[NV][8];
    if (!write) {
#pragma unroll
        for (int m = 0; m < NV; ++m)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[m][j] = raw8_value(rr[m], j, a.r_type);
    } else {
        float z[NV][8];
#pragma unroll
        for (int m = 0; m < NV; ++m)
#pragma unroll
            for (int j = 0; j < 8; ++j) z[m][j] = raw8_value(yr[m], j, a.y_type);
        if (a.post) {
            const float rs = row_scale<WAVES, VEC, L, NV>(z, n, l, a.eps, sum_s);
#pragma unroll
            for (int m = 0; m < NV; ++m)
#pragma unroll
                for (int j = 0; j < 8; ++j) z[m][j] = (z[m][j] * rs) * a.post[min(slot_at<VEC>(l, L, m, j), n - 1)];
        }
        if (a.gate) {
            const float* g = a.gate + t * a.gate_ld;
#pragma unroll
            for (int m = 0; m < NV; ++m)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float w = g[min(slot_at<VEC>(l, L, m, j), n - 1) * a.gate_step];
                    z[m][j] = z[m][j] * (a.gate_sigmoid ? sigmoid_fast(w) : w);
                }
        }
#pragma unroll
        for (int m = 0; m < NV; ++m)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[m][j] = __builtin_fmaf(a.y_scale, z[m][j], a.res_scale * raw8_value(rr[m], j, a.r_type));
        store_row<VEC, L, NV>(static_cast<uint8_t*>(a.out) + t * a.out_ld * elem_bytes(a.r_type), a.r_type, n, l, v);
    }
    if (a.x) {
        const float rs = row_scale<WAVES, VEC, L, NV>(v, n, l, a.eps, sum_s + 2 * WAVES);
#pragma unroll
        for (int m = 0; m < NV; ++m)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[m][j] = v[m][j] * rs;
                if (a.pre) v[m][j] = v[m][j] * a.pre[min(slot_at<VEC>(l, L, m, j), n - 1)];
            }
        store_row<VEC, L, NV>(static_cast<uint8_t*>(a.x) + t * a.x_ld * elem_bytes(a.x_type), a.x_type, n, l, v);
    }
}

hipError_t launch_block_ends(const EndsArgs& a, hipStream_t s) {
    const auto al = [](const void* p, int64_t ld, int type) {
        return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * elem_bytes(type))) & 15) == 0;
    };
    const bool vec = a.n % 8 == 0 && al(a.R, a.r_ld, a.r_type) && al(a.y, a.y_ld, a.y_type) &&
                     al(a.out, a.out_ld, a.r_type) && al(a.x, a.x_ld, a.x_type) && al(a.post, 0, kF32) && al(a.pre, 0, kF32);
    const EndsShape sh = ends_shape(a.n_tokens, a.n);
    const dim3 grid((unsigned)ends_groups(a.n_tokens, a.n)), block(sh.waves == 1 ? 256 : 64 * sh.waves);
#define SMOE_ENDS(W, V)                                                                    \
    if (sh.waves == W && sh.slots == V) {                                                  \
        if (vec) hipLaunchKernelGGL((k_block_ends<W, V, true>), grid, block, 0, s, a);     \
        else hipLaunchKernelGGL((k_block_ends<W, V, false>), grid, block, 0, s, a);        \
        return hipGetLastError();                                                          \
    }
    SMOE_ENDS(1, 1) SMOE_ENDS(1, 2) SMOE_ENDS(1, 4) SMOE_ENDS(4, 1) SMOE_ENDS(4, 2) SMOE_ENDS(4, 4) SMOE_ENDS(16, 2)
#undef SMOE_ENDS
    return hipErrorInvalidValue;
}

}  // namespace smoe
