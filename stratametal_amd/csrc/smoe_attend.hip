// stratametal_amd/csrc/smoe_attend.hip - attention of each sequence's new tokens over its pages of the cache (gfx950, wave64):
// out = sum_j w_j v_j, w = softmax of scale q k_j over the keys that the query sees.
#include "smoe_dma.hpp"
#include "smoe_launch.hpp"
#include "smoe_rules.hpp"
#include "smoe_types.hpp"

#include <type_traits>

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

// ------------------------------------------------------------------------------------------------ tiles

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <bool F16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Two f32 to the type's pair, round to nearest even.
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {a, b};
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
// Four 16-bit values by columns: the 16 lanes of a quarter give four rows of 16 values, four lanes and 8 bytes each to a row, and
// lane i receives value i of each of the four rows.
__device__ __forceinline__ u32x2 read_columns(const uint8_t* at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at));
}
// The larger of a lane's value and of the lane 32 on (16 on, within the half) from it.
__device__ __forceinline__ float max_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    return __builtin_fmaxf(u2f(r[0]), u2f(r[1]));
}
__device__ __forceinline__ float add_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    return u2f(r[0]) + u2f(r[1]);
}
__device__ __forceinline__ float max_quarters(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
    return max_halves(__builtin_fmaxf(u2f(r[0]), u2f(r[1])));
}
__device__ __forceinline__ float add_quarters(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
    return add_halves(u2f(r[0]) + u2f(r[1]));
}

// 16 (dword: 4) bytes a lane from memory to LDS, lane l's at lds + 16 l (4 l); asynchronous, counted by vmcnt.
__device__ __forceinline__ void to_lds16(uint32_t lds, const void* p) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
__device__ __forceinline__ void to_lds4(uint32_t lds, const void* p) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}

// A row of keys or values in LDS is DIM / 8 pieces of 16 bytes, piece c of row r at place c ^ spread(r): the places of a
// piece in 16 consecutive rows cover the 64 banks once, and so do those of 64 bytes of values in four.
template <int DIM>
__device__ __forceinline__ int spread(int r) {
    return DIM == 64 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : (r & 3) << 2 | ((r >> 2) & 3);
}

// Which rows a work-group has: `rows` query rows (tokens times the heads of key head kvh, a token's heads together) of sequence
// s from row0 on, and the keys k0 .. k1 - 1 of its split.
struct Work {
    Sequence s;
    int row0, rows, kvh, split, k0, k1;
};
// Tile `tile` of M rows: the sequences' tiles lie one behind the other.
template <int M>
__device__ __forceinline__ bool find_tile(const AttendArgs& a, int tile, int lane, Work& w) {
    const int g = a.group;
    int before = 0;
    for (int at = 0; at < a.n_seqs; at += 64) {
        const int b = at + lane;
        int t0 = 0, t1 = 0;
        if (b < a.n_seqs) {
            t0 = min(max(a.q_start[b], 0), a.n_tokens);
            t1 = min(max(a.q_start[b + 1], t0), a.n_tokens);
        }
        const int tiles = ((t1 - t0) * g + M - 1) / M;
        int sum = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(sum, d);
            sum += lane >= d ? v : 0;
        }
        const uint64_t past = __ballot(tile < before + sum);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int first = before + __shfl(sum - tiles, l);
            const int s0 = __builtin_amdgcn_readfirstlane(__shfl(t0, l)), s1 = __builtin_amdgcn_readfirstlane(__shfl(t1, l));
            w.s = sequence_at(a, __builtin_amdgcn_readfirstlane(at + l), s0, s1);
            w.s.len = __builtin_amdgcn_readfirstlane(w.s.len);
            w.row0 = __builtin_amdgcn_readfirstlane((tile - first) * M);
            w.rows = min(M, w.s.n * g - w.row0);
            return true;
        }
        before += __shfl(sum, 63);
    }
    return false;
}
// Work-group i: the key heads of a tile and split lie side by side, so that with eight of them each has an XCD (and its L2) to
// itself; the sequences' last tiles, which see the most keys, come first.
template <int M>
__device__ __forceinline__ bool find_work(const AttendArgs& a, const AttendPlan& p, int lane, Work& w) {
    const int i = blockIdx.x;
    w.kvh = i % a.n_kv;
    const int j = i / a.n_kv;
    w.split = j / p.tiles;
    if (!find_tile<M>(a, p.tiles - 1 - j % p.tiles, lane, w)) return false;
    // the keys that some row of the tile sees
    const int first = w.s.len - w.s.n + w.row0 / a.group, last = w.s.len - w.s.n + (w.row0 + w.rows - 1) / a.group;
    w.k0 = a.window ? max(0, first - a.window + 1) : 0;
    w.k1 = a.causal ? min(w.s.len, last + 1) : w.s.len;
    w.k0 = max(w.k0, 0), w.k1 = max(w.k1, w.k0);
    if (p.splits > 1) {
        // equal pieces of at most p.chunk keys, counted from the first one seen
        const int64_t from = (int64_t)w.k0 + (int64_t)w.split * p.chunk;
        w.k1 = (int)min((int64_t)w.k1, from + p.chunk);
        w.k0 = (int)min(from, (int64_t)w.k1);
    }
    return true;
}

__device__ __forceinline__ int divide(uint32_t n, const Divisor& d) {  // n < 2^31
    return (int)((__umulhi(n, d.mul) + n) >> d.shift);
}

// A row's place in the partial sums, its top and sum, and its output.
__device__ __forceinline__ float* part_row(const AttendArgs& a, const AttendPlan& p, int64_t row, int split) {
    return a.part + p.part_floats + (row * p.splits + split) * a.head_dim;
}
__device__ __forceinline__ void put_stats(const AttendArgs& a, const AttendPlan& p, int64_t row, int split, float top, float sum) {
    if (p.splits > 1) *reinterpret_cast<float2*>(a.part + 2 * (row * p.splits + split)) = make_float2(top, sum);
    else if (a.lse) a.lse[row] = lse_of(top, sum);
}

// Row r of the work-group's (a token and a head) by row_alone, written as the tiles write theirs.
__device__ __forceinline__ void redo_row(const AttendArgs& a, const AttendPlan& p, const Work& w, int r, float* q_s, int lane) {
    const int t = w.s.t0 + (w.row0 + r) / a.group, head = w.kvh * a.group + (w.row0 + r) % a.group;
    const int64_t row = (int64_t)t * a.n_heads + head;
    float out[kMaxDim / 64], top, sum;
    row_alone(a, w.s, t, head, w.k0, w.k1, q_s, out, top, sum, lane);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i) {
        const int d = lane + 64 * i;
        if (d >= a.head_dim) continue;
        if (p.splits > 1) part_row(a, p, row, w.split)[d] = out[i];
        else static_cast<uint16_t*>(a.out)[(int64_t)t * a.out_ld + (int64_t)head * a.head_dim + d] = f32_to_half_bits(out[i] * inv, a.f16 ? kF16 : kBf16);
    }
    if (lane == 0) put_stats(a, p, row, w.split, top, sum);
}
// (a work-group without keys: its rows' tops say so)
__device__ __forceinline__ bool no_keys(const AttendArgs& a, const AttendPlan& p, const Work& w, int threads) {
    if (w.k0 < w.k1) return false;
    if (p.splits > 1) {
        for (int r = threadIdx.x; r < w.rows; r += threads) {
            const int t = w.s.t0 + (w.row0 + r) / a.group, head = w.kvh * a.group + (w.row0 + r) % a.group;
            put_stats(a, p, (int64_t)t * a.n_heads + head, w.split, -__builtin_inff(), 0.0f);
        }
        return true;
    }
    for (int i = threadIdx.x; i < w.rows * a.head_dim; i += threads) {
        const int r = i / a.head_dim, d = i - r * a.head_dim;
        const int t = w.s.t0 + (w.row0 + r) / a.group, head = w.kvh * a.group + (w.row0 + r) % a.group;
        static_cast<uint16_t*>(a.out)[(int64_t)t * a.out_ld + (int64_t)head * a.head_dim + d] = 0;
        if (d == 0) put_stats(a, p, (int64_t)t * a.n_heads + head, w.split, -__builtin_inff(), 0.0f);
    }
    return true;
}

// A query row's fragment of the second operand: pieces h, h + STEP, ... of 8 values of its head, zeros past the head, the
// scale's sign taken in (its size multiplies the scores).
template <int N, int STEP>
__device__ __forceinline__ void load_query(const AttendArgs& a, int t, int head, int h, u32x4 (&f)[N]) {
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)t * a.q_ld + (int64_t)head * a.head_dim;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u, keep = a.scale == 0.0f ? 0u : ~0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = i * STEP + h;
        u32x4 v = *reinterpret_cast<const u32x4*>(q + 8 * min(c, a.head_dim / 8 - 1));
#pragma unroll
        for (int j = 0; j < 4; ++j) f[i][j] = 8 * c < a.head_dim ? (v[j] ^ flip) & keep : 0u;
    }
}

// A new key's weight may be up to 2^kLag times the top's before the sums are scaled to a new top.
constexpr float kLag = 8.0f;

}  // namespace

// Tiles of 128 query rows by KEYS keys, four waves of 32 rows.  A wave forms the transposed scores, keys by queries, with
// v_mfma_f32_32x32x16: a lane then holds half of a query's scores, so the maximum, the exponentials and the sum are its own,
// and its weights, in the order in which it holds them, are the second product's right operand as they are (out transposed,
// values of the head by queries); the keys' order in that product is matched by how the values are read (read_columns).  The
// running top moves only when a score passes it by kLag, so the sums are scaled seldom.  Keys and values of the next tile
// travel to LDS while a tile is worked on, the page numbers of the one after with them.
template <int DIM, bool F16>
__global__ __launch_bounds__(256, 2) void k_attend_tile(const AttendArgs a, const AttendPlan p) {
    constexpr int M = kAttendRows, KEYS = DIM == 256 ? 32 : 64;
    constexpr int LPR = DIM / 8, RPI = 64 / LPR, LOADS = KEYS / RPI / 4;  // lanes to a row, rows of a load, a wave's loads of a tile
    constexpr int PLANE = KEYS * DIM * 2;
    __shared__ __align__(1024) uint8_t lds[4 * PLANE];  // two tiles of keys, then values
    __shared__ int ids[2][64];
    __shared__ int bad_page;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Work w;
    if (!find_work<M>(a, p, lane, w)) return;
    if (no_keys(a, p, w, 256)) return;
    if (threadIdx.x == 0) bad_page = 0;
    const int32_t* table = a.pages + w.s.b * a.pages_ld;
    const int n_tiles = (w.k1 - w.k0 + KEYS - 1) / KEYS;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds)), ids0 = __builtin_amdgcn_readfirstlane(lds_addr(ids));
    const auto load_ids = [&](int j) {  // a key's page number to a lane
        const int key = min(w.k0 + j * KEYS + (lane & (KEYS - 1)), w.k1 - 1);
        to_lds4(ids0 + (j & 1) * 256, table + divide(key, p.page));
    };
    const int r_lane = lane / LPR;
    bool bad = false;
    const auto load_tile = [&](int j) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r = (i * 4 + wave) * RPI + r_lane;
            const int place = min(w.k0 + j * KEYS + r, w.k1 - 1);
            const int off = place - divide(place, p.page) * a.page_size;
            int page = ids[j & 1][r];
            bad |= page < 0 || page >= a.n_pages;
            page = page < 0 || page >= a.n_pages ? 0 : page;
            const int c = min((lane % LPR) ^ spread<DIM>(r), a.head_dim / 8 - 1);
            const int64_t from = ((int64_t)((page * a.n_kv + w.kvh) * a.page_size + off) * a.head_dim + 8 * c) * 2;
            const uint32_t to = lds0 + (j & 1) * 2 * PLANE + (i * 4 + wave) * 1024;
            to_lds16(to, a.k + from);
            to_lds16(to + PLANE, a.v + from);
        }
    };
    if (wave == 0) {
        load_ids(0);
        if (n_tiles > 1) load_ids(1);
    }
    // this lane's query
    const int h = lane >> 5, r_q = wave * 32 + (lane & 31);
    const int row_q = w.row0 + min(r_q, w.rows - 1);
    const int t_q = row_q / a.group, head = w.kvh * a.group + row_q % a.group;
    const int pos = w.s.len - w.s.n + t_q;
    const int hi = a.causal ? min(pos + 1, w.k1) : w.k1, lo = a.window ? max(pos - a.window + 1, w.k0) : w.k0;
    // of the wave's queries: keys that all see lie in [lo_all, hi_all), that any sees in [lo_any, hi_any)
    const int lo_any = __builtin_amdgcn_readfirstlane(lo), hi_all = __builtin_amdgcn_readfirstlane(hi);
    const int lo_all = __builtin_amdgcn_readlane(lo, 31), hi_any = __builtin_amdgcn_readlane(hi, 31);
    const bool live = wave * 32 < w.rows;
    u32x4 qf[DIM / 16];
    load_query<DIM / 16, 2>(a, w.s.t0 + t_q, head, h, qf);
    f32x16 acc[DIM / 32];
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;
    float top = -__builtin_inff(), base = 0.0f, sum = 0.0f;
    const float scale = a.scale == 0.0f ? 1.0f : __builtin_fabsf(a.scale);
    // where the lane reads: row lane & 31 of the keys, pieces h, h + 2, ...; rows 4 h + (lane & 15) / 4 of the values
    const uint32_t k_at = (lane & 31) * DIM * 2 + (h ^ spread<DIM>(lane & 31)) * 16;
    const int v_row = 4 * h + ((lane & 15) >> 2), v_piece = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    vmcnt<0>();
    __syncthreads();
    load_tile(0);
    for (int j = 0; j < n_tiles; ++j) {
        vmcnt<0>();
        __syncthreads();
        if (j + 1 < n_tiles) load_tile(j + 1);
        if (wave == 0 && j + 2 < n_tiles) load_ids(j + 2);
        const int key0 = w.k0 + j * KEYS;
        if (!live || key0 >= hi_any || key0 + KEYS <= lo_any) continue;
        const uint8_t* k_s = lds + (j & 1) * 2 * PLANE;
        const uint8_t* v_s = k_s + PLANE;
        f32x16 s[KEYS / 32];
#pragma unroll
        for (int n = 0; n < KEYS / 32; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = 0.0f;
#pragma unroll
        for (int i = 0; i < DIM / 16; ++i)
#pragma unroll
            for (int n = 0; n < KEYS / 32; ++n) {
                const u32x4 kf = *reinterpret_cast<const u32x4*>(k_s + ((k_at ^ (32 * i)) + n * 32 * DIM * 2));
                s[n] = mfma32<F16>(kf, qf[i], s[n]);
            }
        if (key0 < lo_all || key0 + KEYS > hi_all) {
            const int top_key = hi - key0 - 4 * h, low_key = lo - key0 - 4 * h;
#pragma unroll
            for (int n = 0; n < KEYS / 32; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = n * 32 + 8 * (i / 4) + i % 4;
                    s[n][i] = key < top_key && key >= low_key ? s[n][i] : -__builtin_inff();
                }
        }
        float m = s[0][0];
#pragma unroll
        for (int n = 0; n < KEYS / 32; ++n)
#pragma unroll
            for (int i = n ? 0 : 1; i < 16; ++i) m = __builtin_fmaxf(m, s[n][i]);
        if (__ballot(m * scale > top + kLag)) {
            const float next = __builtin_fmaxf(top, max_halves(m) * scale);
            const float keep = next == top ? 1.0f : __builtin_amdgcn_exp2f(top - next);
            top = next;
            base = top == -__builtin_inff() ? 0.0f : top;
            sum *= keep;
#pragma unroll
            for (int i = 0; i < DIM / 32; ++i)
#pragma unroll
                for (int k = 0; k < 16; ++k) acc[i][k] *= keep;
        }
        u32x4 wt[KEYS / 16];
#pragma unroll
        for (int n = 0; n < KEYS / 32; ++n) {
            float e[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i], scale, -base));
                sum += e[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) wt[2 * n + i / 4][i % 4] = pack2<F16>(e[2 * i], e[2 * i + 1]);
        }
#pragma unroll
        for (int n = 0; n < KEYS / 16; ++n)
#pragma unroll
            for (int i = 0; i < DIM / 32; ++i) {
                u32x4 vf;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int r = 8 * x + v_row;
                    const u32x2 half = read_columns(v_s + (16 * n + r) * DIM * 2 + (((4 * i + v_piece) ^ spread<DIM>(r)) * 16) + 8 * (lane & 1));
                    vf[2 * x] = half[0], vf[2 * x + 1] = half[1];
                }
                acc[i] = mfma32<F16>(vf, wt[n], acc[i]);
            }
    }
    sum = add_halves(sum);
    if (bad) bad_page = 1;
    __syncthreads();
    if (!live) return;
    const float inv = p.splits > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
    // what is not finite may come of a value that the query does not see (0 times it): such rows are done anew
    bool odd = !(__builtin_fabsf(sum) < __builtin_inff());
    const int t = w.s.t0 + t_q;
    const int64_t row = (int64_t)t * a.n_heads + head;
    const bool mine = r_q < w.rows;
    uint16_t* out = static_cast<uint16_t*>(a.out) + (int64_t)t * a.out_ld + (int64_t)head * a.head_dim;
    const bool vec = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.out_ld * 2)) & 7) == 0;
    float* part = p.splits > 1 ? part_row(a, p, row, w.split) : nullptr;
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i)
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
            const int d = 32 * i + 2 * k + 4 * h;
            float v[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                v[x] = acc[i][k + x] * inv;
                odd |= d < a.head_dim && !(__builtin_fabsf(v[x]) < __builtin_inff());
            }
            if (!mine || d >= a.head_dim) continue;
            if (part) *reinterpret_cast<f32x4*>(part + d) = f32x4{v[0], v[1], v[2], v[3]};
            else if (vec) store4(out + d, v, F16 ? kF16 : kBf16);
            else
#pragma unroll
                for (int x = 0; x < 4; ++x) out[d + x] = f32_to_half_bits(v[x], F16 ? kF16 : kBf16);
        }
    if (mine && h == 0) put_stats(a, p, row, w.split, top, sum);
    uint64_t again = __ballot(mine && (odd || bad_page));
    again = (again | again >> 32) & 0xFFFFFFFFull;
    for (; again; again &= again - 1)
        redo_row(a, p, w, wave * 32 + __builtin_ctzll(again), reinterpret_cast<float*>(lds) + wave * kMaxDim, lane);
}

// The splits' sums of a query row: out = sum_s 2^(top_s - top) out_s / sum_s 2^(top_s - top) sum_s.  head_dim / 4 threads to a
// split's values; a row has as many such groups as it has splits, at most a whole work-group's, and they meet in LDS (one wave
// to a row and its splits one by one: 170 us of 202 for 32 rows of 256 splits).
__global__ __launch_bounds__(256) void k_attend_join(const AttendArgs a, const AttendPlan p, int per_row) {
    __shared__ f32x4 out_s[256];
    __shared__ float2 stats_s[256];
    const int per = a.head_dim / 4, groups = 256 / per;  // threads of a group, groups
    const int rows = groups / per_row, g = threadIdx.x / per, d = threadIdx.x % per;
    const int mine = g / per_row, first = g % per_row;
    const int64_t row = (int64_t)blockIdx.x * rows + mine;
    const int t = (int)(row / a.n_heads), head = (int)(row % a.n_heads);
    const bool live = mine < rows && t >= a.q_start[0] && t < min(a.q_start[a.n_seqs], a.n_tokens);
    float top = -__builtin_inff(), sum = 0.0f;
    f32x4 out = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
        const float2* stats = reinterpret_cast<const float2*>(a.part) + row * p.splits;
        const float* part = part_row(a, p, row, 0) + 4 * d;
        constexpr int AHEAD = 4;
        for (int s = first; s < p.splits; s += AHEAD * per_row) {
            f32x4 v[AHEAD];
            float2 m[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int at = min(s + i * per_row, p.splits - 1);
                m[i] = stats[at];
                v[i] = *reinterpret_cast<const f32x4*>(part + (int64_t)at * a.head_dim);
            }
            float next = top;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) next = __builtin_fmaxf(next, m[i].x);
            const float base = next == -__builtin_inff() ? 0.0f : next, keep = __builtin_amdgcn_exp2f(top - base);
            top = next;
            sum *= keep;
            out *= keep;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                // (a split without keys has written no values)
                const bool some = s + i * per_row < p.splits && m[i].x != -__builtin_inff();
                const float w = some ? __builtin_amdgcn_exp2f(m[i].x - base) : 0.0f;
                sum = some ? __builtin_fmaf(w, m[i].y, sum) : sum;
#pragma unroll
                for (int k = 0; k < 4; ++k) out[k] = some ? __builtin_fmaf(w, v[i][k], out[k]) : out[k];
            }
        }
    }
    if (per_row > 1) {
        out_s[threadIdx.x] = out, stats_s[threadIdx.x] = make_float2(top, sum);
        __syncthreads();
        if (first == 0) {
            for (int i = 1; i < per_row; ++i) top = __builtin_fmaxf(top, stats_s[threadIdx.x + i * per].x);
            const float base = top == -__builtin_inff() ? 0.0f : top;
            sum = 0.0f, out = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            for (int i = 0; i < per_row; ++i) {
                const float2 m = stats_s[threadIdx.x + i * per];
                const float w = __builtin_amdgcn_exp2f(m.x - base);
                sum = __builtin_fmaf(w, m.y, sum);
                out += w * out_s[threadIdx.x + i * per];
            }
        }
    }
    if (!live || first != 0) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t* o = static_cast<uint16_t*>(a.out) + (int64_t)t * a.out_ld + (int64_t)head * a.head_dim + 4 * d;
    const float v[4] = {out[0] * inv, out[1] * inv, out[2] * inv, out[3] * inv};
    const int type = a.f16 ? kF16 : kBf16;
    if (((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.out_ld * 2)) & 7) == 0) store4(o, v, type);
    else
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = f32_to_half_bits(v[k], type);
    if (a.lse && d == 0) a.lse[row] = lse_of(top, sum);
}

size_t attend_part_bytes(int64_t n_tokens, int n_seqs, int n_heads, int n_kv, int head_dim, int64_t max_len, int window) {
    const AttendPlan p = attend_plan(n_tokens, n_seqs, n_heads, n_kv, head_dim, max_len, window);
    return p.splits > 1 ? (size_t)(p.part_floats + n_tokens * n_heads * p.splits * head_dim) * 4 : 0;
}

namespace {
template <bool F16>
hipError_t launch_attend_as(const AttendArgs& a, const AttendPlan& p, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)p.tiles * a.n_kv * p.splits));
    if (a.head_dim <= 64) hipLaunchKernelGGL((k_attend_tile<64, F16>), grid, dim3(256), 0, s, a, p);
    else if (a.head_dim <= 128) hipLaunchKernelGGL((k_attend_tile<128, F16>), grid, dim3(256), 0, s, a, p);
    else hipLaunchKernelGGL((k_attend_tile<256, F16>), grid, dim3(256), 0, s, a, p);
    return hipGetLastError();
}
}  // namespace

hipError_t launch_attend(const AttendArgs& a, hipStream_t s) {
    AttendPlan p = attend_plan(a.n_tokens, a.n_seqs, a.n_heads, a.n_kv, a.head_dim, a.max_len, a.window);
    p.page = divisor(a.page_size);
    hipError_t e = a.f16 ? launch_attend_as<true>(a, p, s) : launch_attend_as<false>(a, p, s);
    if (e != hipSuccess || p.splits == 1) return e;
    const int groups = 256 / (a.head_dim / 4);
    int per_row = 1;
    while (per_row < p.splits && 2 * per_row <= groups) per_row *= 2;
    const int64_t rows = (int64_t)a.n_tokens * a.n_heads, each = groups / per_row;
    hipLaunchKernelGGL(k_attend_join, dim3((unsigned)((rows + each - 1) / each)), dim3(256), 0, s, a, p, per_row);
    return hipGetLastError();
}

}  // namespace smoe
