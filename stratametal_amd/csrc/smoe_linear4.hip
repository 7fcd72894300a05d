// stratametal_amd/csrc/smoe_linear4.hip - the product with 4-bit weights and group scales (gfx950, wave64): as the dense
// product, W[o][i] = scale[g][o] (code[o][i] - zero[g][o]), g = i / group.
//
// A group's part of a sum is scale (sum code x - zero sum x): the codes enter the matrix instructions as whole numbers of x's
// type, so that every product is exact and a weight is never rounded, and sum x comes from the same instructions with a
// matrix of ones.
#include "smoe_linear.hpp"

namespace smoe {

namespace {

// The codes of a dword (k = 0 .. 7, k's at bits 4 k) as eight whole numbers of bf16 or fp16.  bf16: a code in a byte is the
// e4m3 number code 2^-9 (its subnormals and first binade are one linear range), converted with a scale of 2^9; fp16: 1024 +
// code by its bits, less 1024.
template <bool F16>
__device__ __forceinline__ u32x4 expand8(uint32_t w) {
    const uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
    const uint32_t a = __builtin_amdgcn_perm(hi, lo, 0x05010400u), b = __builtin_amdgcn_perm(hi, lo, 0x07030602u);
    u32x4 r;
    if constexpr (F16) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const auto two = [](uint32_t c) {
            const f16x2 v = __builtin_bit_cast(f16x2, c | 0x64006400u) - f16x2{(_Float16)1024.0f, (_Float16)1024.0f};
            return __builtin_bit_cast(uint32_t, v);
        };
        r[0] = two(__builtin_amdgcn_perm(0u, a, 0x0C010C00u)), r[1] = two(__builtin_amdgcn_perm(0u, a, 0x0C030C02u));
        r[2] = two(__builtin_amdgcn_perm(0u, b, 0x0C010C00u)), r[3] = two(__builtin_amdgcn_perm(0u, b, 0x0C030C02u));
    } else {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 512.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 512.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 512.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 512.0f, true));
    }
    return r;
}

// The same less the row's zero, exact as well: fp16 from 1024 + code less 1024 + zero; bf16 through f32, which holds 2^23 + code.
// `less`: minus 1024 - zero twice in fp16, or minus 2^23 - zero in f32.
template <bool F16>
__device__ __forceinline__ uint32_t zero_term(uint32_t z) {
    if constexpr (F16) {
        const uint32_t h = __builtin_bit_cast(uint16_t, (_Float16)(-1024.0f - (float)z));
        return h | h << 16;
    } else {
        return f2u(-8388608.0f - (float)z);
    }
}
template <bool F16>
__device__ __forceinline__ u32x4 expand8_less(uint32_t w, uint32_t less) {
    const uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
    u32x4 r;
    if constexpr (F16) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const uint32_t a = __builtin_amdgcn_perm(hi, lo, 0x05010400u), b = __builtin_amdgcn_perm(hi, lo, 0x07030602u);
        const auto two = [&](uint32_t c) {
            return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, c) + __builtin_bit_cast(f16x2, less));
        };
        r[0] = two(__builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)), r[1] = two(__builtin_amdgcn_perm(0x64646464u, a, 0x04030402u));
        r[2] = two(__builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)), r[3] = two(__builtin_amdgcn_perm(0x64646464u, b, 0x04030402u));
    } else {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // 0x4B0000cc: 2^23 + code
            const uint32_t sel = 0x070C0C00u + i;
            const f32x2 v = {u2f(__builtin_amdgcn_perm(0x4B4B4B4Bu, lo, sel)) + u2f(less),
                             u2f(__builtin_amdgcn_perm(0x4B4B4B4Bu, hi, sel)) + u2f(less)};
            r[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
        }
    }
    return r;
}

// The 16-bit or 32-bit values and bytes of a lane, as dwords in LDS (at lds + 4 lane); asynchronous, counted by vmcnt.
__device__ __forceinline__ void scale_to_lds(uint32_t lds, const void* p, bool wide) {
    if (wide) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
    else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ushort %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
__device__ __forceinline__ void byte_to_lds(uint32_t lds, const void* p) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
__device__ __forceinline__ void codes_to_lds(uint32_t lds, const void* p) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
// One or four of them to f32, by selects: a branch for each value's type took two thirds of a step.
__device__ __forceinline__ float one_scale(uint32_t v, int type) {
    const float f16 = (float)__builtin_bit_cast(_Float16, (uint16_t)v);
    return type == kF16 ? f16 : u2f(v << (type == kF32 ? 0 : 16));
}
__device__ __forceinline__ f32x4 four_scales(const uint32_t* p, int type) {
    const u32x4 v = *reinterpret_cast<const u32x4*>(p);
    return f32x4{one_scale(v[0], type), one_scale(v[1], type), one_scale(v[2], type), one_scale(v[3], type)};
}

}  // namespace

// Up to 16 tokens: 16 outputs (of both matrices) to a work-group of eight waves, each every eighth stage of 128 of K.  A stage
// travels to the wave's own LDS whole and asynchronously, RING stages on their way: 64 bytes of each row, so that four lanes
// load one line's half (piece p of row r at place p ^ (r >> 2), and the dwords that a matrix instruction takes of 16 rows
// cover the 64 banks once), the tokens' values, and the scales and zeros of its up to four groups.  Lanes past the last token
// hold its values, and their results are dropped; the waves' sums meet in LDS, in wave order.  Bound by the latency of a wave's few
// stages: one token, 2 x 8192 rows of 2048, groups of 128, 8.2 us; 16 tokens, 2048 rows of 8192, groups of 64, 10.6 us (14.9 with
// stages of more than one group in a loop).
template <bool PAIR, bool F16, int TOKENS>
__global__ __launch_bounds__(512, 4) void k_linear4_few(const Linear4Args a) {
    constexpr int SETS = PAIR ? 2 : 1, WAVES = 8, RING = kLinear4Ring<PAIR, TOKENS>;
    constexpr int XS = TOKENS > 4 ? TOKENS / 4 : 1, LOADS = 3 * SETS + XS;  // a stage's loads of the tokens, and all
    constexpr int STAGE = kLinear4Stage<PAIR, TOKENS>, X0 = SETS * 1536;
    __shared__ __align__(1024) uint8_t lds4[WAVES * RING * STAGE];
    static_assert(WAVES * SETS * 1024 <= WAVES * RING * STAGE, "the waves' sums");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o0 = blockIdx.x * 16, q = lane >> 4;
    const int groups = (a.n_in + a.group - 1) / a.group, stages = (a.n_in + 127) / 128, half_row = a.n_in / 2;
    const uint8_t* w[2] = {static_cast<const uint8_t*>(a.w), static_cast<const uint8_t*>(a.w2)};
    const uint8_t* sc[2] = {static_cast<const uint8_t*>(a.scales), static_cast<const uint8_t*>(a.scales2)};
    const uint8_t* zr[2] = {a.zeros, a.zeros2};
    const bool wide = a.s_type == kF32;
    uint8_t* const mine = lds4 + wave * (RING * STAGE);
    const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(mine));
    const int row = min(o0 + (lane >> 2), a.n_out - 1), piece = (lane & 3) ^ ((lane >> 4) & 3);
    const int out = min(o0 + (lane & 15), a.n_out - 1);
    // (a load past the row's end, or of a stage past the last, brings the row's last values: no step reads them)
    const auto load = [&](int u, uint32_t at) {
        u = min(u, stages - 1);
        const int k = u * 128, g0 = k / a.group;
#pragma unroll
        for (int i = 0; i < SETS; ++i) {
            codes_to_lds(at + i * 1536, w[i] + (int64_t)row * half_row + min(k / 2 + 16 * piece, half_row - 16));
            const int64_t g = (int64_t)min(g0 + q, groups - 1) * a.n_out + out;
            scale_to_lds(at + i * 1536 + 1024, sc[i] + g * (wide ? 4 : 2), wide);
            byte_to_lds(at + i * 1536 + 1280, zr[i] ? zr[i] + g : sc[i]);
        }
#pragma unroll
        for (int j = 0; j < XS; ++j) {
            const int t = min(4 * j + (lane >> 4), TOKENS - 1), c = (lane & 15) ^ t;
            codes_to_lds(at + X0 + j * 1024, static_cast<const uint16_t*>(a.x) + (int64_t)min(t, a.n_tokens - 1) * a.x_ld + min(k + 8 * c, a.n_in - 8));
        }
    };
    const uint32_t one = F16 ? 0x3C003C00u : 0x3F803F80u;
    const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 acc[SETS];
#pragma unroll
    for (int i = 0; i < SETS; ++i) acc[i] = none;
#pragma unroll
    for (int r = 0; r < RING; ++r) load(wave + r * WAVES, base + r * STAGE);
    const int tok = min(lane & 15, TOKENS - 1);
    const uint32_t w_at = (lane & 15) * 64 + 4 * q, w_sw = (lane >> 2) & 3;
    const bool whole = a.group % 128 == 0, halves = a.group % 64 == 0;
    uint32_t at = 0;
    for (int u = wave; u < stages; u += WAVES) {
        vmcnt<(RING - 1) * LOADS>();
        const uint8_t* st = mine + at;
        const auto scaled = [&](int g, f32x4 (&sum)[SETS], f32x4 sx) {  // the sums of the stage's group g
#pragma unroll
            for (int i = 0; i < SETS; ++i) {
                const f32x4 scale = four_scales(reinterpret_cast<const uint32_t*>(st + i * 1536 + 1024) + g * 16 + 4 * q, a.s_type);
                const u32x4 z = *reinterpret_cast<const u32x4*>(st + i * 1536 + 1280 + g * 64 + 16 * q);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = __builtin_fmaf(scale[j], __builtin_fmaf(zr[i] ? -(float)z[j] : -8.0f, sx[j], sum[i][j]), acc[i][j]);
            }
        };
        const auto product = [&](int s, f32x4 (&sum)[SETS], f32x4& sx) {
            const uint4 xv = *reinterpret_cast<const uint4*>(st + X0 + tok * 256 + ((4 * s + q) ^ tok) * 16);
            sx = mfma16<F16>(make_uint4(one, one, one, one), xv, sx);
#pragma unroll
            for (int i = 0; i < SETS; ++i) {
                const uint32_t c = *reinterpret_cast<const uint32_t*>(st + i * 1536 + w_at + (s ^ w_sw) * 16);
                sum[i] = mfma16<F16>(__builtin_bit_cast(uint4, expand8<F16>(c)), xv, sum[i]);
            }
        };
        int g = 0, left = a.group - u * 128 % a.group;  // of the stage's groups, and what is left of it
        const bool full = u * 128 + 128 <= a.n_in;
        if (whole && full) {  // one group, straight on
            f32x4 sum[SETS] = {}, sx = none;
#pragma unroll
            for (int s = 0; s < 4; ++s) product(s, sum, sx);
            scaled(0, sum, sx);
        } else if (halves && full) {  // each half in one group
            const int second = left == 64;
#pragma unroll(PAIR ? 1 : 2)
            for (int i = 0; i < 2; ++i) {
                f32x4 sum[SETS] = {}, sx = none;
                product(2 * i, sum, sx), product(2 * i + 1, sum, sx);
                scaled(i ? second : 0, sum, sx);
            }
        } else if (!PAIR && full) {  // (of two matrices the registers would not hold it)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                f32x4 sum[SETS] = {}, sx = none;
                product(s, sum, sx);
                scaled(g, sum, sx);
                left -= 32;
                if (left == 0) left = a.group, ++g;
            }
        } else {
#pragma unroll 1
            for (int s = 0; s < 4 && u * 128 + s * 32 < a.n_in; ++s) {
                f32x4 sum[SETS] = {}, sx = none;
                product(s, sum, sx);
                scaled(g, sum, sx);
                left -= 32;
                if (left == 0) left = a.group, ++g;
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        load(u + RING * WAVES, base + at);
        at = at + STAGE == RING * STAGE ? 0 : at + STAGE;
    }
    vmcnt<0>();
    // An infinite x makes sum code x and zero sum x infinite both, and so does one past 2^128 / 15: what is not finite is summed anew
    // from codes less their zeros, as the tiles do it, so that the answer is the formula's and goes by no number of tokens.
    bool lost = false;
#pragma unroll
    for (int i = 0; i < SETS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) lost |= !(__builtin_fabsf(acc[i][j]) < __builtin_inff());
    if (__ballot(lost)) {
        f32x4 again[SETS];
#pragma unroll
        for (int i = 0; i < SETS; ++i) again[i] = none;
        const uint16_t* x = static_cast<const uint16_t*>(a.x) + (int64_t)min(lane & 15, a.n_tokens - 1) * a.x_ld + 8 * q;
#pragma unroll 1
        for (int u = wave; u < stages; u += WAVES)
#pragma unroll 1
            for (int k = u * 128; k < min(u * 128 + 128, a.n_in); k += 32) {
                const int64_t g = (int64_t)(k / a.group) * a.n_out;
                const uint4 xv = *reinterpret_cast<const uint4*>(x + k);
#pragma unroll
                for (int i = 0; i < SETS; ++i) {
                    const uint32_t c = *reinterpret_cast<const uint32_t*>(w[i] + (int64_t)out * half_row + k / 2 + 4 * q);
                    const u32x4 wv = expand8_less<F16>(c, zero_term<F16>(zr[i] ? zr[i][g + out] : 8u));
                    const f32x4 sum = mfma16<F16>(__builtin_bit_cast(uint4, wv), xv, none);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int64_t at = g + min(o0 + 4 * q + j, a.n_out - 1);
                        const float scale = wide ? static_cast<const float*>(static_cast<const void*>(sc[i]))[at]
                                                 : one_scale(static_cast<const uint16_t*>(static_cast<const void*>(sc[i]))[at], a.s_type);
                        again[i][j] = __builtin_fmaf(scale, sum[j], again[i][j]);
                    }
                }
            }
#pragma unroll
        for (int i = 0; i < SETS; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_fabsf(acc[i][j]) < __builtin_inff() ? acc[i][j] : again[i][j];
    }
    __syncthreads();
    f32x4* sum_s = reinterpret_cast<f32x4*>(lds4);  // [wave][set][lane]
#pragma unroll
    for (int i = 0; i < SETS; ++i) sum_s[(wave * SETS + i) * 64 + lane] = acc[i];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 0; i < SETS; ++i)
#pragma unroll
        for (int v = 1; v < WAVES; ++v) acc[i] = acc[i] + sum_s[(v * SETS + i) * 64 + lane];
    const int t = lane & 15, o = o0 + 4 * q;
    if (t >= a.n_tokens || o >= a.n_out) return;
    const f32x4 g = acc[0], u = acc[SETS - 1];
    finish4<PAIR>(a, rows_vec(a), t, o, {g[0], g[1], g[2], g[3]}, {u[0], u[1], u[2], u[3]});
}

// More tokens: 128 weight rows (PAIR: 64 of each matrix, 16 of each in turn) by 16 NT tokens, 32 rows to each of four waves; up to
// 64 tokens a work-group has eight, four for each half of its slice of K, whose sums meet in LDS, half the tokens with each (301
// tokens, 2560 x 5003: 31.5 us where one half wrote them all, 29.0).  A step is 64 of K: the wave's codes (half p of row r at place p ^ (r >> 3)), its scales and zeros of the two 32-value steps, and its share of the
// tokens (as in k_linear_tile), through a ring of RING stages in LDS.  A wave expands the codes of its rows in registers, less
// their zeros, for all of the tile's tokens; a group's sums are scaled into the outputs' where it ends (SMALL, groups that do
// not hold whole steps: after every 32 values).  blockIdx.y: a slice of K, whose sums go to `part` for k_linear_join.
// A step is bound by the instructions that expand and scale (180 to 290 beside 32 matrix instructions at 128 tokens) and by the
// reads and the barrier before them: 2048 tokens, 4096 x 4096, groups of 128: 100 us, 686 TFLOP/s (groups of 32: 110); of
// 115 to 120 of a form with the conversions a step ahead, 90 without the loads, 61 without expansion and scales as well.
template <int NT, bool PAIR, bool F16, bool SMALL>
__global__ __launch_bounds__(256 * kLinear4Parts<NT>, 2 / kLinear4Parts<NT>) void k_linear4_tile(const Linear4Args a, int tiles_o, int tiles_t) {
    constexpr int MT = 2, WAVES = 4, BN = 16 * NT, OUTS = PAIR ? 64 : 128, PARTS = kLinear4Parts<NT>, RING = NT == 2 ? 7 : NT == 4 ? 5 : 3;
    constexpr int XS = BN / 8 / WAVES;                                  // a wave's loads of the tokens, 8 rows each
    constexpr int LOADS = 3 + XS, X0 = WAVES * 1536, STAGE = X0 + BN * 128, SLOT = PARTS * STAGE;
    constexpr int NG = NT < 4 ? NT : 4;
    static_assert(WAVES * (kStoreBytes<MT, NG> * PARTS + (PARTS - 1) * MT * NT * 1024) <= RING * SLOT, "the waves' pieces of the epilogue, a part's sums");
    __shared__ __align__(1024) uint8_t lds[RING * SLOT];
    const int lane = threadIdx.x & 63, q = lane >> 4;
    const int part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6 & 3);
    int to, tt;
    tile_of(blockIdx.x, gridDim.x, tiles_o, tiles_t, to, tt);
    const int o0 = to * OUTS, t0 = tt * BN;
    const int n_t = min(BN, a.n_tokens - t0);
    const int half_row = a.n_in / 2, groups = (a.n_in + a.group - 1) / a.group;
    const int all = (a.n_in + 63) / 64;
    const int s0 = (int)((int64_t)all * blockIdx.y / gridDim.y), s1 = (int)((int64_t)all * (blockIdx.y + 1) / gridDim.y);
    const int steps = (s1 - s0 + PARTS - 1) / PARTS, u0 = s0 + part * steps, u1 = min(u0 + steps, s1);
    const bool wide = a.s_type == kF32;
    // row i (0 .. 31) of the wave: its matrix and output
    const auto matrix = [&](int i) { return PAIR && i >= 16; };
    const auto output = [&](int i) { return min(o0 + (PAIR ? wave * 16 + (i & 15) : wave * 32 + i), a.n_out - 1); };
    const uint8_t* codes = static_cast<const uint8_t*>(matrix(lane >> 1) ? a.w2 : a.w) + (int64_t)output(lane >> 1) * half_row;
    const int half = (lane & 1) ^ ((lane >> 4) & 1);
    const bool second = matrix(lane & 31);
    const uint8_t* scales = static_cast<const uint8_t*>(second ? a.scales2 : a.scales) + (int64_t)output(lane & 31) * (wide ? 4 : 2);
    const uint8_t* zeros = second ? a.zeros2 : a.zeros;
    const uint8_t* zeros_at = zeros ? zeros + output(lane & 31) : scales;
    const int64_t zero_ld = zeros ? a.n_out : 0, scale_ld = (int64_t)a.n_out * (wide ? 4 : 2);
    const i32x4 rx = uniform_rsrc(static_cast<const uint8_t*>(a.x) + (size_t)t0 * a.x_ld * 2, (uint32_t)((n_t - 1) * a.x_ld * 2) + 2u * a.n_in);
    uint32_t x_off[XS];
#pragma unroll
    for (int i = 0; i < XS; ++i) {
        const int r = 8 * (i * WAVES + wave) + (lane >> 3);
        x_off[i] = r < n_t ? (uint32_t)(r * a.x_ld * 2) + 16u * ((lane & 7) ^ (lane >> 3)) : kOob;
    }
    const int x_lane = 8 * ((lane & 7) ^ (lane >> 3));
    const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + part * STAGE;
    int next_g = u0 * 64 / a.group, next_left = a.group - u0 * 64 % a.group;  // the group of the next load's first value
    // (codes, scales and zeros past the row's end: its last; the tokens' values there are zeros)
    const auto load = [&](int u, uint32_t at) {
        const int k = u * 64;
        codes_to_lds(at + wave * 1536, codes + min(k / 2 + 16 * half, half_row - 16));
        const int64_t first = min(next_g, groups - 1);
        next_left -= 32;
        if (next_left == 0) next_left = a.group, ++next_g;
        const int64_t second = min(next_g, groups - 1);
        next_left -= 32;
        if (next_left == 0) next_left = a.group, ++next_g;
        scale_to_lds(at + wave * 1536 + 1024, scales + (lane < 32 ? first * scale_ld : second * scale_ld), wide);
        byte_to_lds(at + wave * 1536 + 1280, zeros_at + (lane < 32 ? first * zero_ld : second * zero_ld));
#pragma unroll
        for (int i = 0; i < XS; ++i)
            dma16(at + X0 + (i * WAVES + wave) * 1024, k + x_lane < a.n_in ? x_off[i] + 2u * k : kOob, rx, 0);
    };
    const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 acc[MT][NT], sum[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = sum[m][n] = none;
#pragma unroll
    for (int r = 0; r < RING - 1; ++r) load(u0 + r, base + r * SLOT);
    const int fr = lane & 15;
    int left = a.group - u0 * 64 % a.group;  // of the group
    const bool has_zeros = a.zeros != nullptr, has_zeros2 = PAIR ? a.zeros2 != nullptr : has_zeros;
    uint32_t at = 0;
    for (int u = u0; u < u0 + steps; ++u) {
        // every wave has read the step before, and this one is there
        vmcnt<(RING - 2) * LOADS>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        {
            const uint32_t next = at + (RING - 1) * SLOT;
            load(u + RING - 1, base + (next >= RING * SLOT ? next - RING * SLOT : next));
        }
        uint8_t* const st = lds + at + part * STAGE;
        uint8_t* const ws = st + wave * 1536;
        at = at + SLOT == RING * SLOT ? 0 : at + SLOT;
        if (PARTS > 1 && u >= u1) continue;  // (the second part's last step, of an odd number)
        {  // the step's scales to f32 where they lie, one by each lane
            uint32_t* const own = reinterpret_cast<uint32_t*>(ws + 1024) + lane;
            *own = f2u(one_scale(*own, a.s_type));
        }
        u32x4 av[2][MT];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const uint32_t c = *reinterpret_cast<const uint32_t*>(ws + (16 * m + fr) * 32 + (s ^ (fr >> 3)) * 16 + 4 * q);
                const uint32_t z = *reinterpret_cast<const uint32_t*>(ws + 1280 + (32 * s + 16 * m + fr) * 4);
                av[s][m] = expand8_less<F16>(c, zero_term<F16>((m ? has_zeros2 : has_zeros) ? z : 8u));
            }
        const auto products = [&](int s, auto first) {  // (SMALL: a step's first starts its sums)
#pragma unroll
            for (int n0 = 0; n0 < NT; n0 += NG) {
                u32x4 bv[NG];
#pragma unroll
                for (int n = 0; n < NG; ++n)
                    bv[n] = *reinterpret_cast<const u32x4*>(st + X0 + (16 * (n0 + n) + fr) * 128 + ((4 * s + q) ^ (fr & 7)) * 16);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n = 0; n < NG; ++n)
                        sum[m][n0 + n] = mfma16<F16>(__builtin_bit_cast(uint4, av[s][m]), __builtin_bit_cast(uint4, bv[n]),
                                                     decltype(first)::value ? none : sum[m][n0 + n]);
            }
        };
        const auto scaled = [&](int s) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const f32x4 scale = *reinterpret_cast<const f32x4*>(ws + 1024 + (32 * s + 16 * m + 4 * q) * 4);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[m][n][j] = __builtin_fmaf(scale[j], sum[m][n][j], acc[m][n][j]);
            }
        };
        if constexpr (SMALL) {
            products(0, std::true_type{});
            scaled(0);
            if (u * 64 + 32 < a.n_in) {
                products(1, std::true_type{});
                scaled(1);
            }
        } else {  // a step lies in one group
            products(0, std::false_type{});
            products(1, std::false_type{});
            left -= 64;
            if (left == 0 || u + 1 == u1) {
                scaled(0);
                left = a.group;
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n) sum[m][n] = none;
            }
        }
    }
    vmcnt<0>();
    __syncthreads();
    if constexpr (PARTS == 2) {  // each part has the other's sums of half the tokens, and writes those tokens
        constexpr int HALF = NT / 2, STORE = kStoreBytes<MT, HALF>;
        f32x4* const sums = reinterpret_cast<f32x4*>(lds + 2 * WAVES * STORE) + wave * (MT * NT * 64) + lane;  // [m][n]
        f32x4 mine[MT][HALF];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < HALF; ++n) {
                mine[m][n] = part ? acc[m][n + HALF] : acc[m][n];
                sums[(m * NT + n + (part ? 0 : HALF)) * 64] = part ? acc[m][n] : acc[m][n + HALF];
            }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < HALF; ++n) mine[m][n] = mine[m][n] + sums[(m * NT + n + (part ? HALF : 0)) * 64];
        tile_store<MT, HALF, HALF, PAIR>(a, mine, lds + (part * WAVES + wave) * STORE, o0 + wave * (PAIR ? 16 : 32), t0 + part * 16 * HALF, t0 + n_t, lane);
    } else {
        tile_store<MT, NT, NG, PAIR>(a, acc, lds + wave * kStoreBytes<MT, NG>, o0 + wave * (PAIR ? 16 : 32), t0, t0 + n_t, lane);
    }
}

size_t linear4_part_bytes(int64_t T, int K, int N, bool pair, int) {
    const int slices = linear4_plan(T, K, N, pair).slices;
    return slices > 1 ? (size_t)slices * (pair ? 2 : 1) * T * ((N + 3) / 4) * 16 : 0;
}

namespace {
template <bool PAIR, bool F16, int TOKENS>
hipError_t launch_few(const Linear4Args& a, hipStream_t s) {
    hipLaunchKernelGGL((k_linear4_few<PAIR, F16, TOKENS>), dim3((a.n_out + 15) / 16), dim3(512), 0, s, a);
    return hipGetLastError();
}
template <int NT, bool PAIR, bool F16, bool SMALL>
hipError_t launch_tile4(const Linear4Args& a, int slices, hipStream_t s) {
    constexpr int OUTS = PAIR ? 64 : 128, BN = 16 * NT;
    const int tiles_o = (a.n_out + OUTS - 1) / OUTS, tiles_t = (a.n_tokens + BN - 1) / BN;
    hipLaunchKernelGGL((k_linear4_tile<NT, PAIR, F16, SMALL>), dim3(tiles_o * tiles_t, slices), dim3(256 * kLinear4Parts<NT>), 0, s, a, tiles_o, tiles_t);
    return hipGetLastError();
}
template <bool PAIR, bool F16>
hipError_t launch_linear4_as(const Linear4Args& a, hipStream_t s) {
    const Linear4Plan p = linear4_plan(a.n_tokens, a.n_in, a.n_out, PAIR);
    if (p.tokens == 1) return launch_few<PAIR, F16, 1>(a, s);
    if (p.tokens == 4) return launch_few<PAIR, F16, 4>(a, s);
    if (p.tokens == 16) return launch_few<PAIR, F16, 16>(a, s);
    const auto tile = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        return a.group % 64 ? launch_tile4<NT, PAIR, F16, true>(a, p.slices, s) : launch_tile4<NT, PAIR, F16, false>(a, p.slices, s);
    };
    const hipError_t e = p.tokens == 32   ? tile(std::integral_constant<int, 2>{})
                         : p.tokens == 64 ? tile(std::integral_constant<int, 4>{})
                                          : tile(std::integral_constant<int, 8>{});
    return e != hipSuccess || p.slices == 1 ? e : launch_linear_join(a, p.slices, s);
}
}  // namespace

hipError_t launch_linear4(const Linear4Args& a, hipStream_t s) {
    const bool f16 = a.w_type == kF16;
    if (a.w2) return f16 ? launch_linear4_as<true, true>(a, s) : launch_linear4_as<true, false>(a, s);
    return f16 ? launch_linear4_as<false, true>(a, s) : launch_linear4_as<false, false>(a, s);
}

}  // namespace smoe
