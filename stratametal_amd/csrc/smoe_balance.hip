// stratametal_amd/csrc/smoe_balance.hip - the router's balance loss, its per-expert counts and its gradients (gfx950,
// wave64).
//   p = softmax(logits); f_e = counts_e / (n k), P_e = mean_t p_te over the n tokens of the mask;
//   balance = E sum_e f_e P_e, z = mean_t lse_t^2, loss = cb balance + cz z
//   dlogits_tj = (cb E p_tj (f_j - sum_e f_e p_te) + 2 cz lse_t p_tj) / n, dbias_j = sum_t dlogits_tj
// The gradient needs f, and f needs the ids alone: the counts come first (k_balance_counts, T k integers), so the logits
// are read once, and their gradient is written in the same pass (k_balance_rows).  Sums over tokens: a wave's rows in
// registers, a work-group's waves through LDS in wave order, the work-groups' partial rows in k_balance_sums in index order
// and in 64 bits; the counts are integers: every result is the same bits in every run.
#include "smoe_gemv.hpp"
#include "smoe_launch.hpp"
#include "smoe_rules.hpp"
#include "smoe_types.hpp"

#include <type_traits>

namespace smoe {

namespace {

constexpr int kThreads = 256, kBalanceWaves = kThreads / 64;
constexpr int kSumCols = 64;  // columns of a work-group of k_balance_sums

// The scratch: per work-group of the rows kernel E sums of p, E of dlogits, the sum of lse^2; per work-group of the counts
// kernel E counts and its tokens; k_balance_sums' partial sums of f P and its ticket.
struct Work {
    float *psum, *dsum;
    double *zsum, *fp;
    int32_t *counts, *tokens, *ticket;
};
__host__ __device__ inline size_t balance_up(size_t v) { return (v + 255) & ~(size_t)255; }
inline size_t work_layout(int64_t T, int E, uint8_t* base, Work* w) {
    const int64_t G = balance_groups(T), C = balance_count_groups(T);
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        uint8_t* p = base + at;
        at += balance_up(bytes);
        return p;
    };
    Work v;
    v.psum = reinterpret_cast<float*>(take((size_t)G * E * 4));
    v.dsum = reinterpret_cast<float*>(take((size_t)G * E * 4));
    v.zsum = reinterpret_cast<double*>(take((size_t)G * 8));
    v.fp = reinterpret_cast<double*>(take((size_t)(E + kSumCols - 1) / kSumCols * 8));
    v.counts = reinterpret_cast<int32_t*>(take((size_t)C * E * 4));
    v.tokens = reinterpret_cast<int32_t*>(take((size_t)C * 4));
    v.ticket = reinterpret_cast<int32_t*>(take(4));
    if (w) *w = v;
    return at;
}

}  // namespace

// Pairs per expert and tokens of the mask in C pieces of the batch, a work-group each.
__global__ __launch_bounds__(kThreads) void k_balance_counts(const int32_t* __restrict__ ids, const uint8_t* __restrict__ mask,
                                                             int T, int E, int k, Work w) {
    extern __shared__ int32_t hist[];  // E + 1
    const int tid = threadIdx.x, C = gridDim.x;
    for (int e = tid; e <= E; e += kThreads) hist[e] = 0;
    __syncthreads();
    const int t0 = (int)((int64_t)T * blockIdx.x / C), t1 = (int)((int64_t)T * (blockIdx.x + 1) / C);
    const int64_t i1 = (int64_t)t1 * k;
    for (int64_t i = (int64_t)t0 * k + tid; i < i1; i += kThreads) {
        const int e = ids[i];
        if ((uint32_t)e < (uint32_t)E && (!mask || mask[i / k])) atomicAdd(&hist[e], 1);
    }
    int n = 0;
    for (int t = t0 + tid; t < t1; t += kThreads) n += !mask || mask[t];
    if (n) atomicAdd(&hist[E], n);
    __syncthreads();
    for (int e = tid; e < E; e += kThreads) w.counts[(size_t)blockIdx.x * E + e] = hist[e];
    if (tid == 0) {
        w.tokens[blockIdx.x] = hist[E];
        if (blockIdx.x == 0) *w.ticket = 0;
    }
}

// One wave per row at a time, rows blockIdx.x * 4 + wave, then 4 gridDim.x further: column lane + 64 j in slot j of NJ.
// The next row is on its way while this one is worked on.  dlogits may be logits: a row is written by the wave that read it.
template <int NJ, bool GRAD>
__global__ __launch_bounds__(kThreads) void k_balance_rows(const float* logits, int64_t ld,
                                                           const uint8_t* __restrict__ mask, int T, int E, int k, float cb,
                                                           float cz, float* dlogits, int64_t ld_d, int C, Work w) {
    __shared__ float col_s[kBalanceWaves][64 * NJ];
    __shared__ double z_s[kBalanceWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int step = gridDim.x * kBalanceWaves;
    float f[NJ], psum[NJ], dsum[NJ];
    float inv_n = 0.0f;
    if constexpr (GRAD) {
        int n = 0;
        for (int c = 0; c < C; ++c) n += w.tokens[c];
        inv_n = n > 0 ? 1.0f / (float)n : 0.0f;
        const float inv_nk = inv_n / (float)k;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int e = min(lane + 64 * j, E - 1);
            int cnt = 0;
            for (int c = 0; c < C; ++c) cnt += w.counts[(size_t)c * E + e];
            f[j] = (float)cnt * inv_nk;
        }
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) psum[j] = dsum[j] = 0.0f;
    double zsum = 0.0;
    int64_t t = (int64_t)blockIdx.x * kBalanceWaves + wave;
    float next[NJ];
    const auto load = [&](int64_t row) {
        const float* p = logits + min(row, (int64_t)T - 1) * ld;
#pragma unroll
        for (int j = 0; j < NJ; ++j) next[j] = p[min(lane + 64 * j, E - 1)];
    };
    load(t);
    for (; t < T; t += step) {
        float v[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) v[j] = lane + 64 * j < E ? next[j] : -__builtin_inff();
        load(t + step);
        const bool used = !mask || mask[t];
        float* d = GRAD ? dlogits + t * ld_d : nullptr;
        if (!used) {  // (a masked row's values, whatever they are, go nowhere)
            if constexpr (GRAD) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    if (lane + 64 * j < E) d[lane + 64 * j] = 0.0f;
            }
            continue;
        }
        float top = v[0];
#pragma unroll
        for (int j = 1; j < NJ; ++j) top = __builtin_fmaxf(top, v[j]);
        top = wave_max_fast(top);
        const float shift = top == -__builtin_inff() ? 0.0f : top;  // a row of -inf alone: every e^v is 0
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            v[j] = exp_fast(v[j] - shift);
            sum += v[j];
        }
        sum = wave_sum_xor_fast(sum);
        const bool none = sum == 0.0f;
        const float inv = none ? 0.0f : 1.0f / sum;
        const float lse = none ? 0.0f : top + __builtin_logf(sum);
        zsum += (double)lse * (double)lse;
        float fp = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            v[j] = v[j] * inv;
            psum[j] += v[j];
            if constexpr (GRAD) fp = __builtin_fmaf(f[j], v[j], fp);
        }
        if constexpr (GRAD) {
            fp = wave_sum_xor_fast(fp);
            const float zc = 2.0f * cz * lse, bc = cb * (float)E;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const float g = v[j] * __builtin_fmaf(bc, f[j] - fp, zc) * inv_n;
                dsum[j] += g;
                if (lane + 64 * j < E) d[lane + 64 * j] = g;
            }
        }
    }
    // the waves' column sums, in wave order
    const auto fold = [&](const float (&a)[NJ], float* out) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) col_s[wave][lane + 64 * j] = a[j];
        __syncthreads();
        for (int e = threadIdx.x; e < E; e += kThreads)
            out[(size_t)blockIdx.x * E + e] = ((col_s[0][e] + col_s[1][e]) + col_s[2][e]) + col_s[3][e];
    };
    fold(psum, w.psum);
    if (lane == 0) z_s[wave] = zsum;
    __syncthreads();
    if (threadIdx.x == 0) w.zsum[blockIdx.x] = ((z_s[0] + z_s[1]) + z_s[2]) + z_s[3];
    if constexpr (GRAD) fold(dsum, w.dsum);
}

// 64 columns to a work-group: the partial rows summed (wave s takes every fourth), counts, P and dbias written; the last
// work-group to arrive forms the loss from the others' sums of f P.
__global__ __launch_bounds__(kThreads) void k_balance_sums(int T, int E, int k, float cb, float cz, int G, int C,
                                                           float* __restrict__ loss, int32_t* __restrict__ counts,
                                                           float* __restrict__ mean_p, float* __restrict__ dbias, Work w) {
    __shared__ double part_s[kBalanceWaves][kSumCols];
    __shared__ int last_s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int e = blockIdx.x * kSumCols + lane, ec = min(e, E - 1);
    int n = 0;
    for (int c = 0; c < C; ++c) n += w.tokens[c];
    const double inv_n = n > 0 ? 1.0 / (double)n : 0.0;
    const auto column = [&](const float* rows) {
        double a = 0.0;
        for (int g = wave; g < G; g += kBalanceWaves) a += (double)rows[(size_t)g * E + ec];
        part_s[wave][lane] = a;
        __syncthreads();
        const double r = ((part_s[0][lane] + part_s[1][lane]) + part_s[2][lane]) + part_s[3][lane];
        __syncthreads();
        return r;
    };
    const double P = column(w.psum) * inv_n;
    if (dbias) {
        const double db = column(w.dsum);
        if (wave == 0 && e < E) dbias[e] = (float)db;
    }
    if (wave == 0) {
        int cnt = 0;
        for (int c = 0; c < C; ++c) cnt += w.counts[(size_t)c * E + ec];
        if (e < E) {
            counts[e] = cnt;
            mean_p[e] = (float)P;
        }
        double fp = e < E ? (double)cnt * inv_n / (double)k * P : 0.0;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) fp += __shfl_xor(fp, o, 64);
        if (lane == 0) {
            __hip_atomic_store(w.fp + blockIdx.x, fp, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last_s = __hip_atomic_fetch_add(w.ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!last_s || wave != 0) return;
    double z = 0.0;
    for (int g = lane; g < G; g += 64) z += w.zsum[g];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
    if (lane == 0) {
        double b = 0.0;
        for (int i = 0; i < (int)gridDim.x; ++i)
            b += __hip_atomic_load(w.fp + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        b *= (double)E;
        z *= inv_n;
        loss[0] = (float)((double)cb * b + (double)cz * z);
        loss[1] = (float)b;
        loss[2] = (float)z;
        loss[3] = (float)n;
    }
}

size_t balance_work_bytes(int64_t T, int E) { return work_layout(T, E, nullptr, nullptr); }

namespace {
template <bool GRAD>
void launch_rows(const BalanceArgs& a, int G, int C, const Work& w, hipStream_t s) {
    const auto go = [&](auto nj) {
        hipLaunchKernelGGL((k_balance_rows<decltype(nj)::value, GRAD>), dim3(G), dim3(kThreads), 0, s, a.logits, a.ld, a.mask,
                           a.n_tokens, a.n_expert, a.k, a.balance_coef, a.z_coef, a.dlogits, a.ld_d, C, w);
    };
    const int E = a.n_expert;
    if (E <= 64) go(std::integral_constant<int, 1>{});
    else if (E <= 128) go(std::integral_constant<int, 2>{});
    else if (E <= 256) go(std::integral_constant<int, 4>{});
    else if (E <= 512) go(std::integral_constant<int, 8>{});
    else go(std::integral_constant<int, 16>{});
}
}  // namespace

hipError_t launch_balance(const BalanceArgs& a, hipStream_t s) {
    const int T = a.n_tokens, E = a.n_expert;
    const int G = (int)balance_groups(T), C = (int)balance_count_groups(T);
    Work w;
    work_layout(T, E, static_cast<uint8_t*>(a.work), &w);
    hipLaunchKernelGGL(k_balance_counts, dim3(C), dim3(kThreads), (E + 1) * 4, s, a.ids, a.mask, T, E, a.k, w);
    if (a.dlogits) launch_rows<true>(a, G, C, w, s);
    else launch_rows<false>(a, G, C, w, s);
    hipLaunchKernelGGL(k_balance_sums, dim3((E + kSumCols - 1) / kSumCols), dim3(kThreads), 0, s, T, E, a.k, a.balance_coef,
                       a.z_coef, G, C, a.loss, a.counts, a.mean_p, a.dlogits ? a.dbias : nullptr, w);
    return hipGetLastError();
}

}  // namespace smoe
