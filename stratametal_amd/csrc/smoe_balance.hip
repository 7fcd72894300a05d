// stratametal_amd/csrc/smoe_balance.hip - the router's balance loss, its per-expert counts and its gradients (gfx950,
// wave64).
//   p = softmax(logits); f_e = counts_e / (n k), P_e = mean_t p_te over the n tokens of the mask;
//   balance = E sum_e f_e P_e, z = mean_t lse_t^2, loss = cb balance + cz z
//   dlogits_tj = (cb E p_tj (f_j - sum_e f_e p_te) + 2 cz lse_t p_tj) / n, dbias_j = sum_t dlogits_tj
// The gradient needs f, and f needs the ids alone: the counts come first (T k integers), so the logits are read once, and
// their gradient is written in the same pass (k_balance_rows).  Sums over tokens: a wave's rows in registers, a work-group's
// waves through LDS in wave order, the work-groups' partial rows in k_balance_sums in a fixed order and in 64 bits; the
// counts are integers: every result is the same bits in every run.
//   k_balance_one                                    a few tokens: one work-group does it all
//   k_balance_rows, k_balance_sums                   some pairs: each work-group that needs the counts counts for itself
//   k_balance_counts, k_balance_rows, k_balance_sums a batch
// Bound by the logits' and the gradient's bytes in a large batch (32768 tokens of 1024 experts 72 us among other calls, 268 MB),
// by the launches' chains of latencies else: 4096 tokens of 512 experts, 10 each, 24.5 us, without gradients 18, 64 tokens
// without gradients 10.  Rows of more than 512 experts without vectors and with gradients spill in their loop (22 registers of
// the 128): 32768 tokens of 1001 experts 200 us, of 1024 66, both among calls of their own kind.
#include "smoe_gemv.hpp"
#include "smoe_launch.hpp"
#include "smoe_rules.hpp"
#include "smoe_types.hpp"

#include <type_traits>

namespace smoe {

namespace {

constexpr int kRowWaves = 4, kOneWaves = 16;  // waves of k_balance_rows and k_balance_one
constexpr int kSumCols = 16, kSumGroups = 64;     // columns of a work-group of k_balance_sums, groups of its lanes
static_assert(1024 / kSumCols <= 64, "a wave holds the work-groups' sums");

// The scratch: per work-group of the rows kernel E sums of p, E of dlogits and the sum of lse^2; per work-group of the
// counts kernel E counts and its tokens; k_balance_sums' sums of f P and its ticket.
struct Work {
    float *psum, *dsum;
    double *zsum, *fp;
    int32_t *counts, *tokens, *ticket;
};
size_t work_layout(int64_t T, int E, uint8_t* base, Work* w) {
    const int64_t G = balance_groups(T), C = balance_count_groups(T);
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        uint8_t* p = base + at;
        at += (bytes + 255) & ~(size_t)255;
        return p;
    };
    Work v;
    v.psum = reinterpret_cast<float*>(take((size_t)G * E * 4));
    v.dsum = reinterpret_cast<float*>(take((size_t)G * E * 4));
    v.zsum = reinterpret_cast<double*>(take((size_t)G * 8));
    v.fp = reinterpret_cast<double*>(take(64 * 8));
    v.counts = reinterpret_cast<int32_t*>(take((size_t)C * E * 4));
    v.tokens = reinterpret_cast<int32_t*>(take((size_t)C * 4));
    v.ticket = reinterpret_cast<int32_t*>(take(4));
    if (w) *w = v;
    return at;
}

// The pairs of tokens t0 .. t1 - 1 per expert into hist[0 .. E - 1] and the tokens that count into hist[E] (LDS; every
// thread of the work-group calls it): 16 ids of a thread on their way together.
__device__ __forceinline__ void histogram(const int32_t* __restrict__ ids, const uint8_t* __restrict__ mask, int t0, int t1,
                                          int E, int k, int32_t* hist) {
    constexpr int kIds = 16;
    const int tid = threadIdx.x;
    const uint32_t threads = blockDim.x;
    for (int e = tid; e <= E; e += threads) hist[e] = 0;
    __syncthreads();
    const uint32_t i1 = (uint32_t)t1 * k;  // (at most 2^24 pairs)
    for (uint32_t i0 = (uint32_t)t0 * k; i0 < i1; i0 += threads * kIds) {
        int e[kIds];
        uint8_t on[kIds];
#pragma unroll
        for (int j = 0; j < kIds; ++j) e[j] = ids[min(i0 + tid + threads * j, i1 - 1)];
#pragma unroll
        for (int j = 0; j < kIds; ++j) on[j] = mask ? mask[min(i0 + tid + threads * j, i1 - 1) / (uint32_t)k] : 1;
#pragma unroll
        for (int j = 0; j < kIds; ++j)
            if (i0 + tid + threads * j < i1 && on[j] && (uint32_t)e[j] < (uint32_t)E) atomicAdd(&hist[e[j]], 1);
    }
    int n = 0;
    for (int t = t0 + tid; t < t1; t += threads) n += !mask || mask[t];
    if (n) atomicAdd(&hist[E], n);
    __syncthreads();
}

// The sum of column e of C rows of counts: eight loads on their way at a time.
__device__ __forceinline__ int count_of(const int32_t* __restrict__ counts, int e, int E, int C) {
    int n = 0;
    for (int c0 = 0; c0 < C; c0 += 8) {
        int v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = counts[(size_t)min(c0 + c, C - 1) * E + e];
#pragma unroll
        for (int c = 0; c < 8; ++c) n += c0 + c < C ? v[c] : 0;
    }
    return n;
}

// A wave's rows t, t + step, ...: the sums over them of p (psum), of their gradient (dsum) and of lse^2 (returned).  The
// next row is on its way while this one is worked on.  VEC (E % 4 == 0, aligned rows): slot j of a lane is column
// 4 (lane + 64 (j / 4)) + j % 4, else lane + 64 j.  dlogits may be logits: a row is written by the wave that read it.
template <int NJ, bool GRAD, bool VEC>
struct Rows {
    const float* logits;
    const uint8_t* mask;
    float* dlogits;
    int64_t ld, ld_d;
    int T, E;
    float cz;
    float next[NJ];
    uint8_t next_on;

    static __device__ __forceinline__ int col(int j) {
        const int lane = threadIdx.x & 63;
        return VEC ? 4 * (lane + 64 * (j >> 2)) + (j & 3) : lane + 64 * j;
    }
    __device__ __forceinline__ void load(int64_t row) {
        row = min(row, (int64_t)T - 1);
        const float* p = logits + row * ld;
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < NJ; j += 4) {
                const float4 q = *reinterpret_cast<const float4*>(p + min(col(j), E - 4));
                next[j] = q.x, next[j + 1] = q.y, next[j + 2] = q.z, next[j + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < NJ; ++j) next[j] = p[min(col(j), E - 1)];
        }
        next_on = mask ? mask[row] : 1;
    }
    __device__ __forceinline__ void store(int64_t row, const float (&g)[NJ]) {
        float* d = dlogits + row * ld_d;
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < NJ; j += 4)
                if (col(j) < E) *reinterpret_cast<float4*>(d + col(j)) = make_float4(g[j], g[j + 1], g[j + 2], g[j + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                if (col(j) < E) d[col(j)] = g[j];
        }
    }
    // bf: cb E f / n.  A row's e^(v - top) is 2^(v log2 e - c), c = top log2 e as rounded: every e^v and their sum share a
    // factor 2^d, d the rounding of c, that p is free of and lse takes back.  d grows with top (past 2^31 the factor itself
    // leaves f32), so a row whose top is beyond kFar, where |d| is at most 1/16, takes v - top first.
    __device__ __forceinline__ double run(int64_t t, int64_t step, const float (&bf)[NJ], float inv_n, float (&psum)[NJ],
                                          float (&dsum)[NJ]) {
        constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f, kFar = 0x1p20f;
        double zsum = 0.0;
#pragma unroll
        for (int j = 0; j < NJ; ++j) psum[j] = dsum[j] = 0.0f;
        for (; t < T; t += step) {
            float v[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j) v[j] = col(j) < E ? next[j] : -__builtin_inff();
            const bool used = next_on != 0;
            if (t + step < T) load(t + step);
            if (!used) {  // (a masked row's values, whatever they are, go nowhere)
                if constexpr (GRAD) {
#pragma unroll
                    for (int j = 0; j < NJ; ++j) v[j] = 0.0f;
                    store(t, v);
                }
                continue;
            }
            float top = v[0];
#pragma unroll
            for (int j = 1; j < NJ; ++j) top = __builtin_fmaxf(top, v[j]);
            top = wave_max_fast(top);
            float c = top * kLog2e;
            const bool far = __builtin_fabsf(top) > kFar;  // (the same in every lane)
            if (far) {
                const float shift = top == -__builtin_inff() ? 0.0f : top;  // a row of -inf alone: every e^v is 0
#pragma unroll
                for (int j = 0; j < NJ; ++j) v[j] = v[j] - shift;
                c = 0.0f;
            }
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                v[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(v[j], kLog2e, -c));
                sum += v[j];
            }
            sum = wave_sum_xor_fast(sum);
            const bool none = sum == 0.0f;
            const float inv = none ? 0.0f : 1.0f / sum;
            const float log_sum = __builtin_logf(sum);
            const float lse = none ? 0.0f : far ? top + log_sum : __builtin_fmaf(c, kLn2, log_sum);
            zsum += (double)lse * (double)lse;
            float fp = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                v[j] = v[j] * inv;
                psum[j] += v[j];
                if constexpr (GRAD) fp = __builtin_fmaf(bf[j], v[j], fp);
            }
            if constexpr (GRAD) {
                fp = wave_sum_xor_fast(fp);
                const float k = __builtin_fmaf(2.0f * cz * inv_n, lse, -fp);
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    v[j] = v[j] * (bf[j] + k);
                    dsum[j] += v[j];
                }
                store(t, v);
            }
        }
        return zsum;
    }
};

__device__ __forceinline__ double wave_sum_double(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Values between work-groups of one launch: written and read past the XCD's L2 (device scope), and the writer waits for its
// stores before it takes a ticket.  A release fence would write back the whole L2 instead, dirty with the gradients of the
// launch before (k_balance_sums of 1024 partial rows by 1024 columns 23 us with fences).
__device__ __forceinline__ void put_shared(double* p, double v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double get_shared(double* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ int take_ticket(int32_t* p) {
    const int t = __hip_atomic_fetch_add(p, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("" ::: "memory");
    return t;
}
__device__ __forceinline__ void write_loss(float* loss, float cb, float cz, double balance, double z, int n) {
    loss[0] = (float)((double)cb * balance + (double)cz * z);
    loss[1] = (float)balance;
    loss[2] = (float)z;
    loss[3] = (float)n;
}

}  // namespace

// C pieces of the batch, a work-group each.
__global__ __launch_bounds__(1024) void k_balance_counts(const BalanceArgs a, Work w) {
    extern __shared__ int32_t hist[];  // E + 1
    const int C = gridDim.x, E = a.n_expert;
    const int t0 = (int)((int64_t)a.n_tokens * blockIdx.x / C), t1 = (int)((int64_t)a.n_tokens * (blockIdx.x + 1) / C);
    histogram(a.ids, a.mask, t0, t1, E, a.k, hist);
    for (int e = threadIdx.x; e < E; e += 1024) w.counts[(size_t)blockIdx.x * E + e] = hist[e];
    if (threadIdx.x == 0) w.tokens[blockIdx.x] = hist[E];
}

// Rows blockIdx.x * 4 + wave, then 4 gridDim.x further.  C > 0: the counts are k_balance_counts'; 0: counted here.
template <int NJ, bool GRAD, bool VEC>
__global__ __launch_bounds__(64 * kRowWaves, 4) void k_balance_rows(const BalanceArgs a, int C, Work w) {
    __shared__ float col_s[kRowWaves][64 * NJ + 1];
    __shared__ double z_s[kRowWaves];
    const int wave = threadIdx.x >> 6, tid = threadIdx.x, E = a.n_expert;
    const int64_t step = (int64_t)gridDim.x * kRowWaves, t = (int64_t)blockIdx.x * kRowWaves + wave;
    Rows<NJ, GRAD, VEC> r{a.logits, a.mask, a.dlogits, a.ld, a.ld_d, a.n_tokens, E, a.z_coef, {}, 1};
    r.load(t);
    if (blockIdx.x == 0 && tid == 0) *w.ticket = 0;
    float bf[NJ], psum[NJ], dsum[NJ];
    float inv_n = 0.0f;
    if constexpr (GRAD) {
        int32_t* hist = reinterpret_cast<int32_t*>(&col_s[0][0]);
        if (C == 0) {
            histogram(a.ids, a.mask, 0, a.n_tokens, E, a.k, hist);
        } else {
            for (int e = tid; e < E; e += 64 * kRowWaves) hist[e] = count_of(w.counts, e, E, C);
            if (tid == 0) hist[E] = count_of(w.tokens, 0, 1, C);
            __syncthreads();
        }
        const int n = hist[E];
        inv_n = n > 0 ? 1.0f / (float)n : 0.0f;
        const float scale = inv_n / (float)a.k * (a.balance_coef * (float)E) * inv_n;
#pragma unroll
        for (int j = 0; j < NJ; ++j) bf[j] = (float)hist[min(r.col(j), E - 1)] * scale;
        __syncthreads();
    }
    const double zsum = r.run(t, step, bf, inv_n, psum, dsum);
    // the waves' column sums, in wave order
    const auto fold = [&](const float (&v)[NJ], float* out) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) col_s[wave][r.col(j)] = v[j];
        __syncthreads();
        for (int e = tid; e < E; e += 64 * kRowWaves)
            out[(size_t)blockIdx.x * E + e] = ((col_s[0][e] + col_s[1][e]) + col_s[2][e]) + col_s[3][e];
    };
    fold(psum, w.psum);
    if ((tid & 63) == 0) z_s[wave] = zsum;
    __syncthreads();
    if (tid == 0) w.zsum[blockIdx.x] = ((z_s[0] + z_s[1]) + z_s[2]) + z_s[3];
    if constexpr (GRAD) fold(dsum, w.dsum);
}

// 16 columns to a work-group: its 64 groups of 16 lanes each take every 64th partial row, eight of them on their way at a
// time, and what the end needs is loaded beside them.  Writes counts, P and dbias; the last work-group to arrive forms the
// loss from all of their sums of f P.  A chain of latencies: the partial rows, the ticket, the others' sums.
__global__ __launch_bounds__(1024) void k_balance_sums(const BalanceArgs a, int G, int C, Work w) {
    __shared__ double part_s[2][kSumGroups][kSumCols];
    __shared__ double z_s[16];
    __shared__ int hist_s[1025];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E = a.n_expert;
    const int cl = tid % kSumCols, grp = tid / kSumCols;
    const int e = blockIdx.x * kSumCols + cl, ec = min(e, E - 1);
    const bool grad = a.dlogits && a.dbias;
    int n = 0, cnt = 0;
    if (C) {
        n = count_of(w.tokens, 0, 1, C);
        cnt = count_of(w.counts, ec, E, C);
    }
    double z = tid < G ? w.zsum[tid] : 0.0;  // (balance_groups: at most 512 partial rows)
    double pa = 0.0, da = 0.0;
    for (int g = grp; g < G; g += 8 * kSumGroups) {
        float pv[8], dv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const size_t at = (size_t)min(g + kSumGroups * i, G - 1) * E + ec;
            pv[i] = w.psum[at];
            dv[i] = grad ? w.dsum[at] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (g + kSumGroups * i < G) pa += (double)pv[i], da += (double)dv[i];
    }
    if (C == 0) {
        histogram(a.ids, a.mask, 0, a.n_tokens, E, a.k, hist_s);
        n = hist_s[E];
        cnt = hist_s[ec];
    }
    part_s[0][grp][cl] = pa;
    part_s[1][grp][cl] = da;
    z = wave_sum_double(z);
    if (lane == 0) z_s[wave] = z;
    __syncthreads();
    if (wave != 0) return;
    // lanes 0 .. 15: P of a column; 16 .. 31: its dbias
    const double inv_n = n > 0 ? 1.0 / (double)n : 0.0;
    double v = 0.0;
    if (lane < 2 * kSumCols)
        for (int i = 0; i < kSumGroups; ++i) v += part_s[lane / kSumCols][i][cl];
    double fp = 0.0;
    if (lane < kSumCols && e < E) {
        const double P = v * inv_n;
        a.counts[e] = cnt;
        a.mean_p[e] = (float)P;
        fp = (double)cnt * inv_n / (double)a.k * P;
    } else if (lane < 2 * kSumCols && grad && e < E) {
        a.dbias[e] = (float)v;
    }
    fp = wave_sum_double(fp);
    int last = 0;
    if (lane == 0) {
        put_shared(w.fp + blockIdx.x, fp);
        arrived();
        last = take_ticket(w.ticket) == (int)gridDim.x - 1;
    }
    if (!__shfl(last, 0, 64)) return;
    const double b = wave_sum_double(lane < (int)gridDim.x ? get_shared(w.fp + lane) : 0.0);
    z = wave_sum_double(lane < 16 ? z_s[lane] : 0.0);
    if (lane == 0) write_loss(a.loss, a.balance_coef, a.z_coef, b * (double)E, z * inv_n, n);
}

// A few tokens: one work-group of 16 waves, one launch.
template <int NJ, bool GRAD, bool VEC>
__global__ __launch_bounds__(64 * kOneWaves) void k_balance_one(const BalanceArgs a) {
    __shared__ float col_s[kOneWaves][64 * NJ];
    __shared__ int32_t hist[64 * NJ + 1];
    __shared__ double z_s[kOneWaves], b_s[kOneWaves];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, tid = threadIdx.x, E = a.n_expert;
    Rows<NJ, GRAD, VEC> r{a.logits, a.mask, a.dlogits, a.ld, a.ld_d, a.n_tokens, E, a.z_coef, {}, 1};
    r.load(wave);
    histogram(a.ids, a.mask, 0, a.n_tokens, E, a.k, hist);
    const int n = hist[E];
    const float inv_n = n > 0 ? 1.0f / (float)n : 0.0f;
    float bf[NJ], psum[NJ], dsum[NJ];
    if constexpr (GRAD) {
        const float scale = inv_n / (float)a.k * (a.balance_coef * (float)E) * inv_n;
#pragma unroll
        for (int j = 0; j < NJ; ++j) bf[j] = (float)hist[min(r.col(j), E - 1)] * scale;
    }
    const double zsum = r.run(wave, kOneWaves, bf, inv_n, psum, dsum);
    const double over = n > 0 ? 1.0 / (double)n : 0.0;
    const auto put = [&](const float (&v)[NJ]) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) col_s[wave][r.col(j)] = v[j];
        __syncthreads();
    };
    const auto column = [&](int e) {
        double v = 0.0;
        for (int i = 0; i < kOneWaves; ++i) v += (double)col_s[i][e];
        return v;
    };
    put(psum);
    double b = 0.0;
    if (tid < E) {
        const double P = column(tid) * over;
        a.counts[tid] = hist[tid];
        a.mean_p[tid] = (float)P;
        b = (double)hist[tid] * over / (double)a.k * P;
    }
    b = wave_sum_double(b);
    if (lane == 0) {
        z_s[wave] = zsum;
        b_s[wave] = b;
    }
    __syncthreads();
    if (GRAD && a.dbias) {
        put(dsum);
        if (tid < E) a.dbias[tid] = (float)column(tid);
    }
    if (tid == 0) {
        double z = 0.0, s = 0.0;
        for (int i = 0; i < kOneWaves; ++i) z += z_s[i], s += b_s[i];
        write_loss(a.loss, a.balance_coef, a.z_coef, s * (double)E, z * over, n);
    }
}

size_t balance_work_bytes(int64_t T, int E) { return work_layout(T, E, nullptr, nullptr); }

namespace {
template <bool GRAD, bool VEC>
void launch_rows(const BalanceArgs& a, int G, int C, const Work& w, hipStream_t s) {
    const auto go = [&](auto nj) {
        constexpr int NJ = decltype(nj)::value;
        if (balance_one(a.n_tokens, a.k))
            hipLaunchKernelGGL((k_balance_one<NJ, GRAD, VEC>), dim3(1), dim3(64 * kOneWaves), 0, s, a);
        else
            hipLaunchKernelGGL((k_balance_rows<NJ, GRAD, VEC>), dim3(G), dim3(64 * kRowWaves), 0, s, a, C, w);
    };
    const int E = a.n_expert;
    if (!VEC && E <= 64) go(std::integral_constant<int, VEC ? 4 : 1>{});
    else if (!VEC && E <= 128) go(std::integral_constant<int, VEC ? 4 : 2>{});
    else if (E <= 256) go(std::integral_constant<int, 4>{});
    else if (E <= 512) go(std::integral_constant<int, 8>{});
    else go(std::integral_constant<int, 16>{});
}
}  // namespace

hipError_t launch_balance(const BalanceArgs& a, hipStream_t s) {
    const int T = a.n_tokens, E = a.n_expert;
    const int G = (int)balance_groups(T);
    const int C = balance_counts_apart(T, a.k, a.dlogits != nullptr) ? (int)balance_count_groups(T) : 0;
    Work w;
    work_layout(T, E, static_cast<uint8_t*>(a.work), &w);
    const bool one = balance_one(T, a.k);
    if (C) hipLaunchKernelGGL(k_balance_counts, dim3(C), dim3(1024), (E + 1) * 4, s, a, w);
    const bool vec = E % 4 == 0 && a.ld % 4 == 0 && (!a.dlogits || a.ld_d % 4 == 0) && E > 128 &&
                     ((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.dlogits)) & 15) == 0;
    if (a.dlogits) vec ? launch_rows<true, true>(a, G, C, w, s) : launch_rows<true, false>(a, G, C, w, s);
    else vec ? launch_rows<false, true>(a, G, C, w, s) : launch_rows<false, false>(a, G, C, w, s);
    if (!one)
        hipLaunchKernelGGL(k_balance_sums, dim3((E + kSumCols - 1) / kSumCols), dim3(1024), 0, s, a, G, C, w);
    return hipGetLastError();
}

}  // namespace smoe
