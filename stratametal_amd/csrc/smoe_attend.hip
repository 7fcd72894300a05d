// stratametal_amd/csrc/smoe_attend.hip - attention of each sequence's new tokens over its pages of the cache (gfx950, wave64):
// out = sum_j w_j v_j, w = softmax of scale q k_j over the keys that the query sees.
#include "smoe_dma.hpp"
#include "smoe_gemv.hpp"
#include "smoe_launch.hpp"
#include "smoe_rules.hpp"
#include "smoe_types.hpp"

#include <type_traits>

namespace smoe {

namespace {

// Scores travel in units of ln 2 (scale times log2 e), so that weights are 2^(score - top).
constexpr float kLn2 = 0.693147181f;
constexpr int kMaxDim = 256;

// Sequence b: its first query row, rows, length, and how many of its keys are there (no more than max_len).  Its query of row t
// has position len - n + (t - t0).
struct Sequence {
    int b, t0, n, len, keys;
};
// The first key that a query at position p (below 0: before the first key) sees: p - window + 1, where that is not below 0 (and so
// never past 32 bits), window 0: all.
__device__ __forceinline__ int first_seen(int p, int window) { return window && p >= window ? p - window + 1 : 0; }
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
    k1 = min(k1, s.keys);
    k0 = max(k0, first_seen(p, a.window));
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
    // (sums are up to 2^15 times those of weights of at most 1: the powers of two meet `top` by themselves)
    return sum == 0.0f ? -__builtin_inff() : (top + (float)__builtin_amdgcn_frexp_expf(sum) + __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(sum))) * kLn2;
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
// c += a b in accumulation registers: left to itself the compiler keeps the sums elsewhere and moves half of them at every step.
// The hardware does not wait by itself for a matrix instruction's result where another kind of instruction reads it, nor for
// the operands' last writes, and the compiler does not see that this is one: high_wait stands before a run of them, with all the
// sums and the weights as its operands, and one behind it, so that copies of the sums lie outside both and keep their distance.
template <bool F16>
__device__ __forceinline__ void mfma32_high(f32x16& c, const u32x4& a, const u32x4& b) {
    if constexpr (F16) asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
template <int STATES>  // 8 for operands just written, 20 for the results of 16 passes
__device__ __forceinline__ void high_wait(f32x16 (&c)[8], u32x4 (&w)[2]) {
    if constexpr (STATES > 8) asm volatile("s_nop 11" : "+a"(c[7]));
    asm volatile("s_nop 7"
                 : "+a"(c[0]), "+a"(c[1]), "+a"(c[2]), "+a"(c[3]), "+a"(c[4]), "+a"(c[5]), "+a"(c[6]), "+a"(c[7]), "+v"(w[0]), "+v"(w[1]));
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
// Work-group i: the key heads of a tile and split lie side by side, so that with eight of them each has an XCD (and its L2) to
// itself; the sequences' tiles of M rows lie one behind the other, and the last, which see the most keys, come first.
//
// The plan's splits are made for the longest sequence that the call allows; how many keys a piece has is settled here, from
// the lengths that are there: with sequences of about one length whose tiles are fewer than the PLACES of work-groups on the
// card, as many pieces as fill these once; else pieces of a quarter of a place's share, at least the longest over the plan's splits.
// (8 sequences of 4000 keys, 8 key heads: 8 pieces 32 us, 32 35; 64 sequences of up to 8192 keys: 1 piece 214 us, 4 188, 32 199.)
template <int M, int PLACES, int KEYS>
__device__ __forceinline__ bool find_work(const AttendArgs& a, const AttendPlan& p, int lane, Work& w) {
    const int i = blockIdx.x, g = a.group, j = i / a.n_kv, tile = p.tiles - 1 - j % p.tiles;
    w.kvh = i % a.n_kv;
    w.split = j / p.tiles;
    const int seen = a.window ? min(a.window, a.max_len) + (M + g - 1) / g : a.max_len;
    bool found = false;
    int before = 0, most = 0;
    float total = 0.0f;
    int3 next = {0, 0, 0};
    if (lane < a.n_seqs) next = {a.q_start[lane], a.q_start[lane + 1], a.kv_len[lane]};
    for (int at = 0; at < a.n_seqs; at += 64) {
        const int t0 = min(max(next.x, 0), a.n_tokens), t1 = min(max(next.y, t0), a.n_tokens), len = max(next.z, 0);
        next = {0, 0, 0};
        if (const int b = at + 64 + lane; b < a.n_seqs) next = {a.q_start[b], a.q_start[b + 1], a.kv_len[b]};
        const int tiles = ((t1 - t0) * g + M - 1) / M, sum = wave_inclusive_scan(tiles);
        const uint64_t past = found ? 0 : __ballot(tile < before + sum);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int s0 = __builtin_amdgcn_readlane(t0, l), s1 = __builtin_amdgcn_readlane(t1, l);
            const int s_len = __builtin_amdgcn_readlane(len, l);
            w.s = {__builtin_amdgcn_readfirstlane(at + l), s0, s1 - s0, s_len, min(s_len, a.max_len)};
            w.row0 = (tile - before - __builtin_amdgcn_readlane(sum - tiles, l)) * M;
            w.rows = min(M, w.s.n * g - w.row0);
            found = true;
            if (p.splits == 1) break;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
        const int keys = tiles ? min(min(len, a.max_len), seen) : 0;
        most = max(most, keys);
        total += (float)tiles * (float)keys;
    }
    // (starts out of order can count more tiles than 32 bits hold)
    if (!found || w.row0 < 0 || w.rows <= 0) return false;
    // the keys that some row of the tile sees
    const int first = w.s.len - w.s.n + w.row0 / g, last = w.s.len - w.s.n + (w.row0 + w.rows - 1) / g;
    w.k0 = first_seen(first, a.window);
    w.k1 = a.causal ? min(w.s.keys, last + 1) : w.s.keys;
    w.k1 = max(w.k1, w.k0);
    if (p.splits > 1) {
        total = wave_sum_xor_fast(total), most = (int)wave_max_u32_fast((uint32_t)most);
        const float groups = (float)before * (float)a.n_kv, all = total * (float)a.n_kv;
        const bool one = groups <= PLACES && (float)most * groups <= 1.25f * all;
        const float share = one ? (float)(most - 1) / __builtin_floorf(PLACES / groups) : all * (0.25f / PLACES);
        int chunk = max((int)__builtin_fminf(share, (float)most), (most - 1) / p.splits);
        chunk = (chunk / KEYS + 1) * KEYS;
        chunk = __builtin_amdgcn_readfirstlane(chunk);
        const int64_t from = (int64_t)w.k0 + (int64_t)w.split * chunk;
        w.k1 = (int)min((int64_t)w.k1, from + chunk);
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
// Values that are not finite and that a row's sums may hold 0 times: those of keys that some row of the work-group does not see,
// the last and the first such key, and of the last key, which fills up the last block of 32.
struct Broken {
    int last, first;
    bool filling;
    // whether a row that sees the keys lo .. hi - 1 is touched
    __device__ __forceinline__ bool touches(int lo, int hi) const { return last >= hi || first < lo || filling; }
};
__device__ __forceinline__ Broken broken_values(const AttendArgs& a, const Work& w, int lane) {
    const int first_p = w.s.len - w.s.n + w.row0 / a.group, last_p = w.s.len - w.s.n + (w.row0 + w.rows - 1) / a.group;
    const int hi = a.causal ? max(first_p + 1, w.k0) : w.k1, lo = min(first_seen(last_p, a.window), w.k1);
    const int32_t* pages = a.pages + w.s.b * a.pages_ld;
    const uint32_t top_bits = a.f16 ? 0x7C00u : 0x7F80u;  // an exponent of ones
    const auto broken = [&](int key) {
        const int page = pages[key / a.page_size];
        if (page < 0 || page >= a.n_pages) return false;
        const int64_t row = ((int64_t)page * a.n_kv + w.kvh) * a.page_size + key % a.page_size;
        const u32x4* v = reinterpret_cast<const u32x4*>(a.v + row * (a.head_dim * 2));
        bool some = false;
        for (int i = 0; i < a.head_dim / 8; ++i) {
            const u32x4 q = v[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) some |= (q[j] & top_bits) == top_bits || (q[j] >> 16 & top_bits) == top_bits;
        }
        return some;
    };
    Broken b = {-1, 0x7FFFFFFF, (w.k1 - w.k0) % 32 != 0 && broken(w.k1 - 1)};
    const auto look = [&](int from, int to) {
        for (int key = from + lane; key < to; key += 64)
            if (broken(key)) b.last = max(b.last, key), b.first = min(b.first, key);
    };
    look(w.k0, lo), look(hi, w.k1);
    for (int x = 32; x > 0; x >>= 1) b.last = max(b.last, __shfl_xor(b.last, x)), b.first = min(b.first, __shfl_xor(b.first, x));
    return b;
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
// What weights are relative to: the top less LIFT, a weight 2^LIFT times up.  fp16 ones would lose a weight below 2^-25 of the top's
// whole, and half a step of 2^-24 of others, from the values' sums but not from their own, and with many equal keys behind one large
// score these losses add up: so as far up as the type allows (2^15 with the lag), while a step of f32 in the scores is at most a
// quarter.  bf16 ones lose nothing, but beside values near the type's largest must not pass 1.
template <bool F16, bool LAG>
__device__ __forceinline__ float base_of(float top) {
    constexpr float LIFT = (F16 ? 15.0f : 0.0f) - (LAG ? kLag : 0.0f);
    return top == -__builtin_inff() ? 0.0f : F16 && !(__builtin_fabsf(top) < 4194304.0f) ? top : top - LIFT;
}

}  // namespace

// Tiles of 128 query rows by 64 keys, four waves of 32 rows, in steps of 32 keys.  A wave forms the transposed scores, keys by
// queries, with v_mfma_f32_32x32x16: a lane then holds half of a query's scores, so the maximum, the exponentials and the sum
// are its own, and its weights, in the order in which it holds them, are the second product's right operand as they are (out
// transposed, values of the head by queries); the keys' order in that product is matched by how the values are read
// (read_columns).  The running top moves only when a score passes it by kLag, so the sums are scaled seldom.
// The scores run a step ahead: while the next step's keys are multiplied, this step's weights are formed between the matrix
// instructions, and while its values are, the next top; what each instruction needs of LDS is read two or three before.  A
// tile of keys starts a step before the tile of values of the same number, so that two steps work on one tile of each while
// the keys of the tile after next and the values of the next travel to LDS, page numbers a tile before them.
// A weight is rounded to the cache's type for the second product (its sum is not), off by half a step: the error against 64 bits grows
// from 1.6 to 2.1 parts in 1000, where the output's own rounding is 1.6.  With what the rounding leaves as a second operand, as in
// k_attend_few, the prompt below took 803 us for 586, 1024 tokens over 33792 keys 880 for 609.
// 8192 tokens, 32 heads of 128, 8 key heads: 575 to 588 us, 935 to 955 TFLOP/s; bound by its parts together: without exponentials 35
// us less of 640, without weights 62, without the reads of LDS 103, without the second product 116, without loads 95.  Tiles of 256
// rows took 645 to 706 for 587 (one work-group to a CU).
template <int DIM, bool F16>
__global__ __launch_bounds__(256, DIM > 128 ? 1 : 2) void k_attend_tile(const AttendArgs a, const AttendPlan p) {
    constexpr int M = kAttendRows, KEYS = kAttendKeys, ND = DIM / 32, NQ = DIM / 16;
    constexpr int LPR = DIM / 8, RPI = 64 / LPR, LOADS = KEYS / RPI / 4;  // lanes to a row, rows of a load, a wave's loads of a tile
    constexpr int PLANE = KEYS * DIM * 2, HALF = PLANE / 2;
    constexpr bool HIGH = DIM > 128;  // the sums of values in accumulation registers
    __shared__ __align__(1024) uint8_t lds[4 * PLANE];  // two tiles of keys, two of values
    __shared__ int ids[4][64], rows_s[4][64];  // of a tile's keys: page numbers, then rows of the cache
    __shared__ int bad_page;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Work w;
    if (!find_work<M, (DIM > 128 ? 256 : 512), KEYS>(a, p, lane, w)) return;
    if (no_keys(a, p, w, 256)) return;
    if (threadIdx.x == 0) bad_page = 0;
    const int32_t* table = a.pages + w.s.b * a.pages_ld;
    const int n_steps = (w.k1 - w.k0 + 31) / 32;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds)), ids0 = __builtin_amdgcn_readfirstlane(lds_addr(ids));
    // row r of key tile j: its key (before the first: the first, past the last: the last)
    const auto key_of = [&](int j, int r) { return max(w.k0, min(w.k0 + j * KEYS - 32 + r, w.k1 - 1)); };
    const auto load_ids = [&](int j) {  // a key's page number to a lane (every wave: the same numbers)
        to_lds4(ids0 + (j & 3) * 256, table + divide(key_of(j, lane), p.page));
    };
    // a lane's key of tile j: its row in the cache
    bool bad = false;
    const auto find_rows = [&](int j) {
        const int page = ids[j & 3][lane], key = key_of(j, lane), off = key - divide(key, p.page) * a.page_size;
        const bool there = (uint32_t)page < (uint32_t)a.n_pages;
        bad |= !there;
        rows_s[j & 3][lane] = ((there ? page : 0) * a.n_kv + w.kvh) * a.page_size + off;
    };
    // the lane's pieces of a tile's rows, from the half of key tile j on
    const int r_lane = wave * RPI + lane / LPR, piece_lane = lane % LPR, last_piece = a.head_dim / 8 - 1;
    const auto load_plane = [&](const uint8_t* plane, uint32_t at, int j, int half) {
        int rows[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r = i * 4 * RPI + r_lane + 32 * half;
            rows[i] = rows_s[(j + (i * 4 * RPI + 32 * half) / 64) & 3][r & 63];
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int c = min(piece_lane ^ spread<DIM>(i * 4 * RPI + r_lane), last_piece);
            to_lds16(lds0 + at + (i * 4 + wave) * 1024, plane + ((int64_t)rows[i] * (a.head_dim * 2) + 16 * c));
        }
    };
    load_ids(0), load_ids(1), load_ids(2), load_ids(3);
    // this lane's query
    const int h = lane >> 5, r_q = wave * 32 + (lane & 31);
    const int row_q = w.row0 + min(r_q, w.rows - 1);
    const int t_q = row_q / a.group, head = w.kvh * a.group + row_q % a.group;
    const int pos = w.s.len - w.s.n + t_q;
    const int hi = a.causal ? min(pos + 1, w.k1) : w.k1, lo = max(first_seen(pos, a.window), w.k0);
    // keys that all of the wave's queries see: [lo_all, hi_all)
    const int hi_all = __builtin_amdgcn_readfirstlane(hi), lo_all = __builtin_amdgcn_readlane(lo, 31);
    const bool live = wave * 32 < w.rows;
    u32x4 qf[NQ];
    load_query<NQ, 2>(a, w.s.t0 + t_q, head, h, qf);
    f32x16 acc[ND], even, odd;  // the sums of values, the scores of even and odd steps
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;
    float top = -__builtin_inff(), base = 0.0f, sum = 0.0f, odd_sum = 0.0f;
    const float scale = a.scale == 0.0f ? 1.0f : __builtin_fabsf(a.scale);
    // where the lane reads: row lane & 31 of the keys, pieces h, h + 2, ... (piece i: bits 5 on); rows 4 h + (lane & 15) / 4 and
    // 8 on of the values, the 16 bytes of its quarter's two lanes (32 values on: bits 6 on)
    const uint32_t k_at = (lane & 31) * DIM * 2 + (h ^ spread<DIM>(lane & 31)) * 16;
    const int v_row = 4 * h + ((lane & 15) >> 2), v_piece = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    const auto value_at = [&](int x) {
        return (uint32_t)((8 * x + v_row) * DIM * 2 + (v_piece ^ spread<DIM>(8 * x + v_row)) * 16 + 8 * (lane & 1));
    };
    const uint32_t v_at[2] = {value_at(0), value_at(1)};
    const auto all_seen = [&](int key0) { return key0 >= lo_all && key0 + 32 <= hi_all; };
    const auto mask = [&](f32x16& t, int key0) {
        const int top_key = hi - key0 - 4 * h, low_key = lo - key0 - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int key = 8 * (i / 4) + i % 4;
            t[i] = key < top_key && key >= low_key ? t[i] : -__builtin_inff();
        }
    };
    // the top, when a score has passed it: then the sums of values are to be scaled by `keep`
    float keep = 1.0f;
    const auto raise = [&](float m) {
        const float next = __builtin_fmaxf(top, max_halves(m) * scale), old = base;
        base = base_of<F16, true>(next);
        keep = next == top ? 1.0f : top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(old - base);
        top = next;
        sum *= keep, odd_sum *= keep;
    };
    const auto passed = [&](float m) { return __ballot(m * scale > top + kLag) != 0; };
    const auto max_of = [](const f32x16& t, int from, int to, float m) {
#pragma unroll
        for (int e = from; e < to; ++e) m = __builtin_fmaxf(m, t[e]);
        return m;
    };
    // the scores of 32 keys at `place` in LDS into t, `slice(i)` behind matrix instruction i; the longest heads in two chains,
    // as one wave to a SIMD would wait for each instruction's end
    const auto scores = [&](uint32_t place, f32x16& t, auto&& slice) {
        constexpr int AHEAD = 2;
        constexpr bool TWO = DIM > 128;
        uint32_t at = k_at + place;
        asm("" : "+v"(at));  // (the places are formed here, and hold no registers through the products of the values)
        const auto key_part = [&](int i) { return *reinterpret_cast<const u32x4*>(lds + (at ^ (32 * i))); };
        u32x4 kf[AHEAD + 1];
        f32x16 zero, other;
#pragma unroll
        for (int k = 0; k < 16; ++k) zero[k] = 0.0f;
        each_of<AHEAD>([&](auto i) { kf[decltype(i)::value] = key_part(decltype(i)::value); });
        each_of<NQ>([&](auto idx) {
            constexpr int I = decltype(idx)::value;
            if constexpr (I + AHEAD < NQ) kf[(I + AHEAD) % (AHEAD + 1)] = key_part(I + AHEAD);
            f32x16& sums = TWO && I % 2 ? other : t;
            sums = mfma32<F16>(kf[I % (AHEAD + 1)], qf[I], I < (TWO ? 2 : 1) ? zero : sums);
            slice(idx);
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (TWO) t = t + other;
    };
    constexpr int EACH = 16 / NQ < 2 ? 2 : 16 / NQ;  // weights between two of its matrix instructions
    u32x4 wt[2];
    // weight e of the step (of 16 in a lane) in place of its score; two of them, e even, into the sum and the operand
    const auto weigh = [&](f32x16& t, int e) { t[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(t[e], scale, -base)); };
    const auto take = [&](const f32x16& t, int e) {
        sum += t[e], odd_sum += t[e + 1];
        uint32_t both = pack2<F16>(t[e], t[e + 1]);
        asm volatile("" : "+v"(both), "+v"(sum), "+v"(odd_sum));  // here: the compiler would move them behind the mask's branch
        wt[e / 8][e % 8 / 2] = both;
    };
    // the values at `place` times the weights onto the sums, which are scaled first or not, `slice(i)` behind matrix
    // instruction i
    const auto values = [&](auto scaled, uint32_t place, auto&& slice) {
        constexpr int AHEAD = 3, N = 2 * ND;
        constexpr bool SCALED = decltype(scaled)::value;
        uint32_t at[2] = {v_at[0] + place, v_at[1] + place};
        asm("" : "+v"(at[0]), "+v"(at[1]));
        const auto value_part = [&](int i) {
            u32x4 f;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const u32x2 half = read_columns(lds + 16 * (i / ND) * DIM * 2 + (at[x] ^ (64 * (i % ND))));
                f[2 * x] = half[0], f[2 * x + 1] = half[1];
            }
            return f;
        };
        const auto scale_sums = [&](int i) {
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[i][k] *= keep;
        };
        if constexpr (SCALED && HIGH) {
#pragma unroll
            for (int i = 0; i < ND; ++i) scale_sums(i);
        }
        u32x4 vf[AHEAD + 1];
        each_of<AHEAD>([&](auto i) { vf[decltype(i)::value] = value_part(decltype(i)::value); });
        if constexpr (SCALED && !HIGH) scale_sums(0);
        if constexpr (HIGH) high_wait<8>(acc, wt);
        each_of<N>([&](auto idx) {
            constexpr int I = decltype(idx)::value;
            if constexpr (I + AHEAD < N) vf[(I + AHEAD) % (AHEAD + 1)] = value_part(I + AHEAD);
            if constexpr (HIGH) mfma32_high<F16>(acc[I % ND], vf[I % (AHEAD + 1)], wt[I / ND]);
            else acc[I % ND] = mfma32<F16>(vf[I % (AHEAD + 1)], wt[I / ND], acc[I % ND]);
            if constexpr (SCALED && !HIGH && I + 1 < ND) scale_sums(I + 1);
            slice(idx);
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (HIGH) high_wait<20>(acc, wt);
    };
    float m = 0.0f;
    // a step, whose scores are `t`, and the scores of the next; RARE: the next is not all seen, or the sums are to be scaled
    const auto step = [&](auto rare, f32x16& t, f32x16& next, uint32_t keys_at, uint32_t values_at, int next_key) {
        constexpr int N = 2 * ND;
        scores(keys_at, next, [&](auto idx) {
            constexpr int I = decltype(idx)::value;
#pragma unroll
            for (int e = I * EACH; e < (I + 1) * EACH && e < 16; ++e) weigh(t, e);
#pragma unroll
            for (int e = (I - 1) * EACH; e < I * EACH && e < 16; e += 2)
                if (e >= 0) take(t, e);
        });
#pragma unroll
        for (int e = (NQ - 1) * EACH; e < 16; e += 2) take(t, e);
        if constexpr (decltype(rare)::value) mask(next, next_key);
        m = next[0];
        values(rare, values_at, [&](auto idx) { m = max_of(next, decltype(idx)::value * 16 / N, (decltype(idx)::value + 1) * 16 / N, m); });
    };
    vmcnt<0>();
    __syncthreads();
    if (wave < 3) find_rows(wave);
    __syncthreads();
    load_plane(a.k, 0, 0, 0);
    // the values of tile j and the keys of tile j + 1
    const auto load_tiles = [&](int j) {
        const uint32_t plane = (j & 1) * PLANE;
        load_plane(a.k, PLANE - plane, j + 1, 0);
        load_plane(a.v, 2 * PLANE + plane, j, 1);
    };
    load_tiles(0);
    // what tile j's steps read is there, and every wave is past the steps before
    const auto turn = [&](int j) {
        vmcnt<0>();
        __syncthreads();
        load_tiles(j + 1);
        if (wave == (j & 3)) find_rows(j + 3);
        load_ids(j + 4);
    };
    vmcnt<0>();
    __syncthreads();
    if (live) {
        scores(HALF, even, [](auto) {});
        mask(even, w.k0);
        raise(max_of(even, 0, 16, -__builtin_inff()));
        // (no branch within the plain steps that their sums would have to pass: the compiler would copy them each time)
        int u = 0;
        bool rare = true;
        while (u + 1 < n_steps) {
            if (!rare && (u & 1) == 0) {
                for (;;) {
                    const uint32_t plane = (u >> 1 & 1) * PLANE;
                    turn(u >> 1);
                    step(std::false_type{}, even, odd, PLANE - plane, 2 * PLANE + plane, 0);
                    ++u;
                    if (u + 1 >= n_steps || passed(m) || !all_seen(w.k0 + (u + 1) * 32)) {
                        even = odd;
                        break;
                    }
                    step(std::false_type{}, odd, even, PLANE - plane + HALF, 2 * PLANE + plane + HALF, 0);
                    ++u;
                    if (u + 1 >= n_steps || passed(m) || !all_seen(w.k0 + (u + 1) * 32)) break;
                }
            } else {
                const uint32_t plane = (u >> 1 & 1) * PLANE, half = (u & 1) * HALF;
                if ((u & 1) == 0) turn(u >> 1);
                step(std::true_type{}, even, odd, PLANE - plane + half, 2 * PLANE + plane + half, w.k0 + (u + 1) * 32);
                even = odd;
                ++u;
            }
            keep = 1.0f;
            rare = passed(m);
            if (rare) raise(m);
            rare = rare || !all_seen(w.k0 + (u + 1) * 32);
        }
        vmcnt<0>();
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 16; ++e) weigh(even, e);
#pragma unroll
        for (int e = 0; e < 16; e += 2) take(even, e);
        values(std::true_type{}, 2 * PLANE + (u >> 1 & 1) * PLANE + (u & 1) * HALF, [](auto) {});
    } else {
        for (int j = 0; j < n_steps / 2; ++j) turn(j);
        vmcnt<0>();
        __syncthreads();
    }
    sum += odd_sum;
    sum = add_halves(sum);
    if (bad) bad_page = 1;
    __syncthreads();
    if (!live) return;
    const float inv = p.splits > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
    // What is not finite may come of a value that the query does not see (0 times it): rows that one touches are done anew (all of
    // 2048 tokens, 32 heads: 25 ms).  Where a score is NaN, which only one that it sees can be, all values are NaN as they stand, if
    // the head fills the tile: behind a shorter one the key's last values stand again, and 0 times an infinite one is NaN as well.
    const bool odd_score = sum != sum, settled = odd_score && a.head_dim == DIM;
    bool lost = false;
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
                lost |= !settled && d < a.head_dim && !(__builtin_fabsf(v[x]) < __builtin_inff());
            }
            if (!mine || d >= a.head_dim) continue;
            if (part) *reinterpret_cast<f32x4*>(part + d) = f32x4{v[0], v[1], v[2], v[3]};
            else if (vec) store4(out + d, v, F16 ? kF16 : kBf16);
            else
#pragma unroll
                for (int x = 0; x < 4; ++x) out[d + x] = f32_to_half_bits(v[x], F16 ? kF16 : kBf16);
        }
    if (mine && h == 0) put_stats(a, p, row, w.split, top == -__builtin_inff() ? top : base, sum);
    uint64_t again = __ballot(mine && (lost || bad_page));
    if (again && !bad_page) {
        const Broken b = broken_values(a, w, lane);
        again = __ballot(mine && lost && (odd_score || b.touches(lo, hi)));
    }
    again = (again | again >> 32) & 0xFFFFFFFFull;
    for (; again; again &= again - 1)
        redo_row(a, p, w, wave * 32 + __builtin_ctzll(again), reinterpret_cast<float*>(lds) + wave * kMaxDim, lane);
}

// Sequences of few query rows: tiles of 16 rows, four waves each on every fourth block of 32 keys, by itself until the waves' sums
// meet in LDS.  A block's keys and values travel to the wave's own LDS, the next block's as soon as this one's have been
// read, page numbers two blocks ahead.  The transposed scores (v_mfma_f32_16x16x32: keys by queries) leave a lane with 8 keys of
// one query, which are the second product's right operand as they are, with the keys in that order (read_columns), in two numbers of
// the cache's type: the matrix instructions have the time (single tokens took as long with one; 796 with a window 10.2 us for 10.7).
// Bound by the cache's bytes where there are many (56 tokens of 64 sequences of up to 8193 keys, 8 key heads of 128: 179 us, 5.3 TB/s,
// part of it from the Infinity Cache; one token over 131072 keys, 4 key heads 52 us), else by the trips to memory before them (one token
// over 1001 keys, 2 key heads of 256: 10 us).  Waves that share blocks, in tiles of 128 rows, took 201, 57 and 15.
template <int DIM, bool F16>
__global__ __launch_bounds__(256, DIM > 128 ? 1 : 2) void k_attend_few(const AttendArgs a, const AttendPlan p) {
    constexpr int M = kAttendFewRows, NQ = DIM / 32, ND = DIM / 16, PLANE = 32 * DIM * 2;
    constexpr int LPR = DIM / 8, RPI = 64 / LPR, LOADS = 32 / RPI;  // lanes to a row, rows of a load, loads of a block
    static_assert(4 * ND * 1024 <= 8 * PLANE, "the waves' sums");
    __shared__ __align__(1024) uint8_t lds[8 * PLANE];
    __shared__ int32_t ids[4][2][64];
    __shared__ float2 stats_s[4][M];
    __shared__ uint32_t again_s;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Work w;
    if (!find_work<M, (DIM > 128 ? 256 : DIM > 64 ? 512 : 1024), kAttendFewKeys>(a, p, lane, w)) return;
    if (no_keys(a, p, w, 256)) return;
    if (threadIdx.x == 0) again_s = 0;
    const int32_t* table = a.pages + (int64_t)w.s.b * a.pages_ld;
    const int blocks = (w.k1 - w.k0 + 31) / 32;
    uint8_t *const keys = lds + wave * 2 * PLANE, *const values = keys + PLANE;
    const uint32_t keys_at = __builtin_amdgcn_readfirstlane(lds_addr(keys)), values_at = keys_at + PLANE;
    const uint32_t ids_at = __builtin_amdgcn_readfirstlane(lds_addr(ids[wave]));
    const auto key_of = [&](int j) { return min(w.k0 + 32 * j + (lane & 31), w.k1 - 1); };  // (past the last: the last)
    const auto load_ids = [&](int j, int slot) { to_lds4(ids_at + slot * 256, table + divide(key_of(j), p.page)); };
    bool bad = false;
    const auto find_row = [&](int j, int slot) {  // a lane's key of block j: its row in the cache
        const int page = ids[wave][slot][lane], key = key_of(j), off = key - divide(key, p.page) * a.page_size;
        const bool there = (uint32_t)page < (uint32_t)a.n_pages;
        bad |= !there;
        return ((there ? page : 0) * a.n_kv + w.kvh) * a.page_size + off;
    };
    const int r_lane = lane / LPR, piece_lane = lane % LPR, last_piece = a.head_dim / 8 - 1;
    const auto load_plane = [&](const uint8_t* plane, uint32_t at, int row) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r = i * RPI + r_lane, c = min(piece_lane ^ spread<DIM>(r), last_piece);
            to_lds16(at + i * 1024, plane + ((int64_t)__shfl(row, r) * (a.head_dim * 2) + 16 * c));
        }
    };
    // this lane's query, and its quarter of the keys (of the values)
    const int h = lane >> 4, r_q = lane & 15, row_q = w.row0 + min(r_q, w.rows - 1);
    const int t_q = row_q / a.group, head = w.kvh * a.group + row_q % a.group;
    const int pos = w.s.len - w.s.n + t_q;
    const int hi = a.causal ? min(pos + 1, w.k1) : w.k1, lo = max(first_seen(pos, a.window), w.k0);
    if (wave < blocks) load_ids(wave, 0), load_ids(wave + 4, 1);
    u32x4 qf[NQ];
    load_query<NQ, 4>(a, w.s.t0 + t_q, head, h, qf);
    f32x4 acc[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float top = -__builtin_inff(), base = 0.0f, sum = 0.0f;
    const float scale = a.scale == 0.0f ? 1.0f : __builtin_fabsf(a.scale);
    // rows 4 h + (lane & 15) / 4 and 16 on of the values, the 8 bytes of the lane's quarter of 16 values
    const int v_row = 4 * h + (r_q >> 2), v_piece = (lane & 3) >> 1;
    int row = 0;
    if (wave < blocks) {
        vmcnt<0>();
        row = find_row(wave, 0);
        load_plane(a.k, keys_at, row), load_plane(a.v, values_at, row);
    }
    int slot = 1;
    for (int j = wave; j < blocks; j += 4) {
        const bool more = j + 4 < blocks;
        vmcnt<LOADS>();  // the keys, and the next block's page numbers
        f32x4 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            s[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            const int r = 16 * b + r_q;
#pragma unroll
            for (int i = 0; i < NQ; ++i)
                s[b] = mfma16<F16>(*reinterpret_cast<const u32x4*>(keys + r * DIM * 2 + ((4 * i + h) ^ spread<DIM>(r)) * 16), qf[i], s[b]);
        }
        if (more) {
            row = find_row(j + 4, slot);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the keys and these numbers have been read)
            slot ^= 1;
            load_ids(j + 8, slot);
            load_plane(a.k, keys_at, row);
        }
        float t[8], m = -__builtin_inff();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int key = w.k0 + 32 * j + 16 * (e / 4) + 4 * h + e % 4;
            t[e] = key < hi && key >= lo ? s[e / 4][e % 4] : -__builtin_inff();
            m = __builtin_fmaxf(m, t[e]);
        }
        m = max_halves(max_quarters(m));
        const float next = __builtin_fmaxf(top, m * scale);
        if (__ballot(next != top)) {
            const float old = base;
            base = base_of<F16, false>(next);
            const float keep = next == top ? 1.0f : top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(old - base);
            top = next;
            sum *= keep;
#pragma unroll
            for (int i = 0; i < ND; ++i) acc[i] *= keep;
        }
        u32x4 wt, rest;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            t[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(t[e], scale, -base));
            sum += t[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            wt[e] = pack2<F16>(t[2 * e], t[2 * e + 1]);
            rest[e] = pack2<F16>(t[2 * e] - half_value(wt[e] & 0xFFFFu, F16), t[2 * e + 1] - half_value(wt[e] >> 16, F16));
        }
        if (more) vmcnt<LOADS + 1>();  // the values
        else vmcnt<0>();
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            u32x4 f;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int r = 16 * x + v_row;
                const u32x2 half = read_columns(values + r * DIM * 2 + ((2 * i + v_piece) ^ spread<DIM>(r)) * 16 + 8 * (lane & 1));
                f[2 * x] = half[0], f[2 * x + 1] = half[1];
            }
            acc[i] = mfma16<F16>(f, wt, acc[i]);
            acc[i] = mfma16<F16>(f, rest, acc[i]);
        }
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            load_plane(a.v, values_at, row);
        }
    }
    vmcnt<0>();
    sum += __shfl_xor(sum, 16);
    sum = add_halves(sum);
    __syncthreads();  // (again_s is set, and every wave has read its blocks)
    if (bad) atomicOr(&again_s, 0x1FFFFu);  // (bit 16: a page outside the cache)
    if (h == 0) stats_s[wave][r_q] = make_float2(top == -__builtin_inff() ? top : base, sum);
    f32x4* const sums = reinterpret_cast<f32x4*>(lds);  // [wave][16 values][lane]
#pragma unroll
    for (int i = 0; i < ND; ++i) sums[(wave * ND + i) * 64 + lane] = acc[i];
    __syncthreads();
    float part_of[4];
    top = -__builtin_inff();
#pragma unroll
    for (int v = 0; v < 4; ++v) top = __builtin_fmaxf(top, stats_s[v][r_q].x);
    base = top == -__builtin_inff() ? 0.0f : top;
    sum = 0.0f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        part_of[v] = __builtin_amdgcn_exp2f(stats_s[v][r_q].x - base);
        sum = __builtin_fmaf(part_of[v], stats_s[v][r_q].y, sum);
    }
    const float inv = p.splits > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
    // What is not finite may come of a value that the query does not see (0 times it): rows that one touches are done anew (all of
    // 2048 tokens, 32 heads: 25 ms).  Where a score is NaN, which only one that it sees can be, all values are NaN as they stand, if
    // the head fills the tile: behind a shorter one the key's last values stand again, and 0 times an infinite one is NaN as well.
    const bool odd_score = sum != sum, settled = odd_score && a.head_dim == DIM;
    bool lost = false;
    const int tok = w.s.t0 + t_q;
    const int64_t out_row = (int64_t)tok * a.n_heads + head;
    const bool mine = r_q < w.rows;
    uint16_t* out = static_cast<uint16_t*>(a.out) + (int64_t)tok * a.out_ld + (int64_t)head * a.head_dim;
    const bool vec = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.out_ld * 2)) & 7) == 0;
    float* part = p.splits > 1 ? part_row(a, p, out_row, w.split) : nullptr;
#pragma unroll
    for (int i = 0; i < ND / 4; ++i) {
        const int n = 4 * i + wave, d = 16 * n + 4 * h;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < 4; ++v) o += part_of[v] * sums[(v * ND + n) * 64 + lane];
        float y[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            y[x] = o[x] * inv;
            lost |= !settled && d < a.head_dim && !(__builtin_fabsf(y[x]) < __builtin_inff());
        }
        if (!mine || d >= a.head_dim) continue;
        if (part) *reinterpret_cast<f32x4*>(part + d) = f32x4{y[0], y[1], y[2], y[3]};
        else if (vec) store4(out + d, y, F16 ? kF16 : kBf16);
        else
#pragma unroll
            for (int x = 0; x < 4; ++x) out[d + x] = f32_to_half_bits(y[x], F16 ? kF16 : kBf16);
    }
    if (wave == 0 && mine && h == 0) put_stats(a, p, out_row, w.split, top, sum);
    if (mine && lost) atomicOr(&again_s, 1u << r_q);
    __syncthreads();
    uint32_t again = again_s & ((1u << w.rows) - 1);
    if (again && !(again_s >> 16)) {
        const Broken b = broken_values(a, w, lane);
        again &= (uint32_t)__ballot(odd_score || b.touches(lo, hi));  // (lanes 0 .. 15 have rows 0 .. 15)
    }
    for (; again; again &= again - 1) {
        const int r = __builtin_ctz(again);
        if (r % 4 == wave) redo_row(a, p, w, r, reinterpret_cast<float*>(lds) + wave * kMaxDim, lane);
    }
}

// The splits' sums of a query row: out = sum_s 2^(top_s - top) out_s / sum_s 2^(top_s - top) sum_s.  head_dim / 4 threads to a
// split's values; a row has as many such groups as it has splits, at most a whole work-group's, and they meet in LDS (one wave
// to a row and its splits one by one: 170 us of 202 for 32 rows of 256 splits).
__global__ __launch_bounds__(256) void k_attend_join(const AttendArgs a, const AttendPlan p, int per_row) {
    __shared__ f32x4 out_s[256];
    __shared__ float2 stats_s[256];
    const int per = a.head_dim / 4, d = threadIdx.x % per;  // threads of a group
    const JoinPlace place = attend_join_place(threadIdx.x, per, per_row);
    const int first = place.group;
    const int64_t row = (int64_t)blockIdx.x * (256 / per / per_row) + place.row;
    const int t = (int)(row / a.n_heads), head = (int)(row % a.n_heads);
    const bool live = place.row >= 0 && t >= a.q_start[0] && t < min(a.q_start[a.n_seqs], a.n_tokens);
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
                // (a split without keys has a sum of 0 and has written no values; one whose scores are all NaN has a top of -inf and a
                // sum of NaN, which 0 times it keeps)
                const bool some = s + i * per_row < p.splits && m[i].y != 0.0f;
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
        if (live && first == 0) {  // (of a thread past the last row the other groups' places lie past the arrays)
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
    if (p.few) {
        if (a.head_dim <= 64) hipLaunchKernelGGL((k_attend_few<64, F16>), grid, dim3(256), 0, s, a, p);
        else if (a.head_dim <= 128) hipLaunchKernelGGL((k_attend_few<128, F16>), grid, dim3(256), 0, s, a, p);
        else hipLaunchKernelGGL((k_attend_few<256, F16>), grid, dim3(256), 0, s, a, p);
    } else if (a.head_dim <= 64) hipLaunchKernelGGL((k_attend_tile<64, F16>), grid, dim3(256), 0, s, a, p);
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
