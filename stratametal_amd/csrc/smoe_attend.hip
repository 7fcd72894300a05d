// stratametal_amd/csrc/smoe_attend.hip - attention of each sequence's new tokens over its pages of the cache (gfx950, wave64):
// out = sum_j w_j v_j, w = softmax of scale q k_j over the keys that the query sees.
#include "smoe_launch.hpp"
#include "smoe_types.hpp"

namespace smoe {

namespace {

// Scores travel in units of ln 2 (scale times log2 e), so that weights are 2^(score - top).
constexpr float kLn2 = 0.693147181f;
constexpr int kMaxDim = 256;

// The sequence that holds query row t, and its first row and key count; b < 0: none.
struct Sequence {
    int b, t0, n, len;
};
__device__ __forceinline__ Sequence sequence_at(const AttendArgs& a, int b, int t0, int t1) {
    const int len = min(max(a.kv_len[b], 0), a.max_len);
    return {b, t0, t1 - t0, len};
}
__device__ __forceinline__ Sequence sequence_of(const AttendArgs& a, int t, int lane) {
    for (int at = 0; at < a.n_seqs; at += 64) {
        const int b = min(at + lane, a.n_seqs - 1);
        const int t0 = a.q_start[b], t1 = min(a.q_start[b + 1], a.n_tokens);
        const uint64_t in = __ballot(t0 <= t && t < t1);
        if (in) {
            const int l = __builtin_ctzll(in);
            return sequence_at(a, __shfl(b, l), max(__shfl(t0, l), 0), __shfl(t1, l));
        }
    }
    return {-1, 0, 0, 0};
}

__device__ __forceinline__ float half_value(uint32_t bits, bool f16) { return elem_to_f32(bits, f16 ? kF16 : kBf16); }

// One query row by one wave, 64 keys at a time, a key to a lane for its score and 64 values of the head to the wave for the
// sum: keys that the query does not see are skipped, not weighted by 0.  out[i]: value lane + 64 i.
__device__ __forceinline__ void row_alone(const AttendArgs& a, const Sequence& s, int t, int head, int k0, int k1, float* q_s,
                                       float (&out)[kMaxDim / 64], float& top, float& sum, int lane) {
    const int D = a.head_dim, kvh = head / (a.n_heads / a.n_kv);
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)t * a.q_ld + (int64_t)head * D;
    for (int d = lane; d < D; d += 64) q_s[d] = half_value(q[d], a.f16);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int p = s.len - s.n + (t - s.t0);
    if (a.causal) k1 = min(k1, p + 1);
    k1 = min(k1, s.len);
    if (a.window) k0 = max(k0, p - a.window + 1);
    k0 = max(k0, 0);
    const int32_t* pages = a.pages + s.b * a.pages_ld;
    top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i) out[i] = 0.0f;
    for (int at = k0; at < k1; at += 64) {
        const int j = at + lane, page = j < k1 ? pages[j / a.page_size] : -1;
        const bool there = page >= 0 && page < a.n_pages;
        const int64_t row = there ? ((int64_t)page * a.n_kv + kvh) * a.page_size + j % a.page_size : 0;
        float score = 0.0f;
        if (there) {
            const uint16_t* k = reinterpret_cast<const uint16_t*>(a.k) + row * D;
            for (int d = 0; d < D; d += 8) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(k + d);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    score = __builtin_fmaf(q_s[d + 2 * i], half_value(w[i] & 0xFFFFu, a.f16), score);
                    score = __builtin_fmaf(q_s[d + 2 * i + 1], half_value(w[i] >> 16, a.f16), score);
                }
            }
        }
        score = there ? score * a.scale : -__builtin_inff();
        float m = score;
        for (int x = 32; x > 0; x >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, x));
        m = __builtin_fmaxf(m, top);
        const float base = m == -__builtin_inff() ? 0.0f : m;
        const float keep = __builtin_amdgcn_exp2f(top - base), w = there ? __builtin_amdgcn_exp2f(score - base) : 0.0f;
        top = m;
        sum = __builtin_fmaf(sum, keep, w);
#pragma unroll
        for (int i = 0; i < kMaxDim / 64; ++i) out[i] *= keep;
        for (uint64_t left = __ballot(there); left; left &= left - 1) {
            const int l = __builtin_ctzll(left);
            const float wl = __shfl(w, l);
            const uint16_t* v = reinterpret_cast<const uint16_t*>(a.v) + __shfl(row, l) * D;
#pragma unroll
            for (int i = 0; i < kMaxDim / 64; ++i)
                if (lane + 64 * i < D) out[i] = __builtin_fmaf(wl, half_value(v[lane + 64 * i], a.f16), out[i]);
        }
    }
    for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x);
}

__device__ __forceinline__ float lse_of(float top, float sum) {
    return sum == 0.0f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

}  // namespace

// A wave to a query row.
__global__ __launch_bounds__(256) void k_attend_rows(const AttendArgs a) {
    __shared__ float q_s[4][kMaxDim];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t i = (int64_t)blockIdx.x * 4 + wave;
    if (i >= (int64_t)a.n_tokens * a.n_heads) return;
    const int t = (int)(i / a.n_heads), head = (int)(i % a.n_heads);
    const Sequence s = sequence_of(a, t, lane);
    if (s.b < 0) return;
    float out[kMaxDim / 64], top, sum;
    row_alone(a, s, t, head, 0, s.len, q_s[wave], out, top, sum, lane);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t* o = static_cast<uint16_t*>(a.out) + (int64_t)t * a.out_ld + (int64_t)head * a.head_dim;
#pragma unroll
    for (int d = 0; d < kMaxDim / 64; ++d)
        if (lane + 64 * d < a.head_dim) o[lane + 64 * d] = f32_to_half_bits(out[d] * inv, a.f16 ? kF16 : kBf16);
    if (a.lse && lane == 0) a.lse[i] = lse_of(top, sum);
}

size_t attend_part_bytes(int64_t, int, int, int, int, int, int64_t) { return 0; }

hipError_t launch_attend(const AttendArgs& a, hipStream_t s) {
    const int64_t rows = (int64_t)a.n_tokens * a.n_heads;
    hipLaunchKernelGGL(k_attend_rows, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace smoe
