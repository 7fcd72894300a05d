// stratametal_amd/csrc/smoe_linear.hip - the dense product with bias, activation and residual in its epilogue (gfx950,
// wave64): y[t][o] = act(sum_i x[t][i] w[o][i] + bias[o]) [* (sum_i x[t][i] w2[o][i] + bias2[o])] [+ residual[t][o]],
// x and w bf16 or fp16, sums in f32 on the matrix cores, one rounding to y's type.
#include "smoe_linear.hpp"

namespace smoe {

// A tile of BM = 16 MT WM weight rows by BN = 16 NT WN tokens per work-group of WM WN waves, MT x NT fragments of 16 x 16
// to a wave; K in steps of 64 through a ring of RING LDS buffers, filled by loads that write LDS directly.  A row's step is
// eight 16-byte pieces, piece c of row r at place c ^ (r & 7), so that the 16 rows of a fragment's read spread over the
// banks.  A step is two halves: while a half's products run, the fragments of the next half are read and half of the loads
// of the step RING (weights: past the middle) or RING - 1 (tokens) later are issued; one barrier, in the middle.  (A step's
// fragments read after its barrier: 0.67 us a step of 128 x 128 whatever the ring.)  Steps past the end load nothing: their
// offsets lie past the buffers, zeros go to LDS, and the count of loads under way stays the same.
// blockIdx.y: a slice of K, whose sums go to `part` ([slice][w, w2][token][n_out]) for k_linear_join.
// Some ten tokens are bound by the weights' bytes, some hundred by how few work-groups there are (301 tokens, 5003 x 2568,
// tiles of 128 x 128 in two slices of K: 17 us and 6 to join them, 0.45 PFLOP/s).
template <int MT, int NT, int WM, int WN, int RING, bool PAIR, bool F16>
__global__ __launch_bounds__(64 * WM * WN) void k_linear_tile(const LinearArgs a, int tiles_o, int tiles_t) {
    constexpr int WAVES = WM * WN, BM = 16 * MT * WM, BN = 16 * NT * WN;
    constexpr int OUTS = PAIR ? BM / 2 : BM;           // outputs of the tile
    constexpr int WS = BM / 8 / WAVES, XS = BN / 8 / WAVES, SLOTS = WS + XS;  // a wave's loads of a step, 8 rows each
    constexpr int STEP = (BM + BN) * 128;              // bytes of a step
    static_assert((RING - 1) * SLOTS <= 63, "vmcnt");
    __shared__ __align__(1024) uint8_t lds[RING * STEP];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    int to, tt;
    tile_of(blockIdx.x, gridDim.x, tiles_o, tiles_t, to, tt);
    const int o0 = to * OUTS, t0 = tt * BN;
    const int n_o = min(OUTS, a.n_out - o0), n_t = min(BN, a.n_tokens - t0);
    i32x4 rw, rx;
    uint32_t off[SLOTS];
    tile_loads<BM, BN, WAVES, PAIR>(a, o0, t0, n_o, n_t, wave, lane, rw, rx, off);
    const int all = (a.n_in + 63) / 64;
    const int u0 = (int)((int64_t)all * blockIdx.y / gridDim.y), u1 = (int)((int64_t)all * (blockIdx.y + 1) / gridDim.y);
    const int k_end = min(a.n_in, u1 * 64), k_lane = 8 * ((lane & 7) ^ (lane >> 3));
    const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(lds) + wave * 1024);
    const auto load = [&](int u, int i, uint32_t at) {  // load i of step u into the ring's step `at` (a byte offset)
        dma16(base + at + (i < WS ? i * WAVES * 1024 : BM * 128 + (i - WS) * WAVES * 1024),
              u * 64 + k_lane < k_end ? off[i] + 128u * u : kOob, i < WS ? rw : rx, 0);
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < RING; ++r)
#pragma unroll
        for (int i = 0; i < (r < RING - 1 ? SLOTS : WS); ++i) load(u0 + r, i, r * STEP);
    vmcnt<(RING - 2) * SLOTS + WS>();
    __syncthreads();
    const int fr = lane & 15;
    const uint8_t* wb = lds + (wm * MT * 16 + fr) * 128;
    const uint8_t* xb = lds + (BM + wn * NT * 16 + fr) * 128;
    uint4 av[2][MT], bv[2][NT];
    const auto read = [&](uint32_t at, int h, int i) {  // fragment i of half h: the tokens, then the weights
        const int k = ((4 * h + (lane >> 4)) ^ (fr & 7)) * 16;
        if (i < NT) bv[h][i] = *reinterpret_cast<const uint4*>(xb + at + k + i * 2048);
        else av[h][i - NT] = *reinterpret_cast<const uint4*>(wb + at + k + (i - NT) * 2048);
    };
#pragma unroll
    for (int i = 0; i < MT + NT; ++i) read(0, 0, i);
    uint32_t at = 0, before = (RING - 1) * STEP;  // of this step and the one before
    for (int u = u0; u < u1; ++u) {
        const uint32_t next = at + STEP == RING * STEP ? 0 : at + STEP;
        const auto half = [&](auto which) {
            constexpr int H = decltype(which)::value, L = H ? WS : XS, F = MT * NT, FR = MT + NT;
            each_of<F>([&](auto idx) {
                constexpr int I = decltype(idx)::value;
                // what goes before product I: the I-th shares of the loads and of the next half's fragments
                each_of<(I + 1) * L / F - I * L / F>([&](auto j) {
                    constexpr int l = I * L / F + decltype(j)::value;
                    if constexpr (H) load(u + RING, l, at);
                    else load(u + RING - 1, WS + l, before);
                });
                each_of<(I + 1) * FR / F - I * FR / F>([&](auto j) { read(H ? next : at, 1 - H, I * FR / F + decltype(j)::value); });
                acc[I / NT][I % NT] = mfma16<F16>(av[H][I / NT], bv[H][I % NT], acc[I / NT][I % NT]);
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        half(std::integral_constant<int, 0>{});
        // every wave has read this step, and the next one is there
        vmcnt<(RING - 2) * SLOTS>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        half(std::integral_constant<int, 1>{});
        before = at;
        at = next;
    }
    vmcnt<0>();
    constexpr int NG = WAVES * kStoreBytes<MT, NT> <= RING * STEP ? NT : NT / 2;
    static_assert(WAVES * kStoreBytes<MT, NG> <= RING * STEP, "the waves' pieces");
    __syncthreads();
    tile_store<MT, NT, NG, PAIR>(a, acc, lds + wave * kStoreBytes<MT, NG>, o0 + wm * (16 * MT / (PAIR ? 2 : 1)), t0 + wn * NT * 16, t0 + n_t,
                             lane);
}

// c += a b, in place in accumulation registers: left to itself the compiler rotates k_linear_big's 256 of them through copies
// and their wait states, a third of the loop.  Nothing but LDS reads may write a and b shortly before, and settle() comes
// between the last of these and a read of a sum: the hardware does not wait for either by itself.
template <bool F16>
__device__ __forceinline__ void mfma16_in_place(f32x4& c, const u32x4& a, const u32x4& b) {
    if constexpr (F16) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
// The same with a load into LDS (dma16, to `lds` + AT) round it: the matrix instruction is the wait state between m0's write
// and its use.
template <bool F16, int AT>
__device__ __forceinline__ void mfma16_dma(f32x4& c, const u32x4& a, const u32x4& b, uint32_t lds, uint32_t voff, i32x4 rsrc) {
#define SMOE_MFMA_DMA(OP)                                                                                          \
    asm volatile("s_add_u32 m0, %3, %4\n\t" OP " %0, %1, %2, %0\n\tbuffer_load_dwordx4 %5, %6, 0 offen lds"         \
                 : "+a"(c)                                                                                          \
                 : "v"(a), "v"(b), "s"(lds), "n"(AT), "v"(voff), "s"(rsrc)                                         \
                 : "memory", "m0", "scc")
    if constexpr (F16) SMOE_MFMA_DMA("v_mfma_f32_16x16x32_f16");
    else SMOE_MFMA_DMA("v_mfma_f32_16x16x32_bf16");
#undef SMOE_MFMA_DMA
}
__device__ __forceinline__ void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// The same product in tiles of 256 weight rows by 256 tokens, four waves (one to a SIMD) of 128 by 128: 64 fragments of
// sums in 256 accumulation registers, so that 128 matrix instructions share 32 fragment reads of LDS (eight waves of 128 by
// 64 need 48, which with the loads' writes keeps the LDS as long busy as the matrix cores).  A step of 64 of K is two
// halves; while a half's 64 instructions run, the fragments of the next half are read.  LDS is a ring of five tiles of 256
// rows, of w and of x in turn: in a step's first half the weights of the step after the next go where the step before had
// its tokens, in its second half, past the one barrier, the tokens where this step had its weights, so that the loads are
// spread evenly: a wave issues in order, and waits where they back up (all of them in the second half: 7 % slower).
// Bound by the matrix cores and, with one work-group to a CU, by the epilogue, under which nothing runs: 4096 tokens by
// 8192 x 8192 with an f32 residual 406 us, 1.35 PFLOP/s, by two of 8192 x 2048 220 us, 1.25.
template <bool PAIR, bool F16>
__global__ __launch_bounds__(256, 1) void k_linear_big(const LinearArgs a, int tiles_o, int tiles_t) {
    constexpr int MT = 8, NT = 8, WAVES = 4, BM = 256, BN = 256, OUTS = PAIR ? 128 : 256;
    constexpr int WS = 8, SLOTS = 16, TILE = 256 * 128, RING = 5;
    static_assert(WAVES * kStoreBytes<MT, 4> <= RING * TILE, "the waves' pieces of the epilogue");
    __shared__ __align__(1024) uint8_t lds[RING * TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    int to, tt;
    tile_of(blockIdx.x, gridDim.x, tiles_o, tiles_t, to, tt);
    const int o0 = to * OUTS, t0 = tt * BN;
    const int n_o = min(OUTS, a.n_out - o0), n_t = min(BN, a.n_tokens - t0);
    uint32_t off[SLOTS];
    i32x4 rw, rx;
    tile_loads<BM, BN, WAVES, PAIR>(a, o0, t0, n_o, n_t, wave, lane, rw, rx, off);
    const int all = (a.n_in + 63) / 64;
    const int u0 = (int)((int64_t)all * blockIdx.y / gridDim.y), u1 = (int)((int64_t)all * (blockIdx.y + 1) / gridDim.y);
    const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(lds) + wave * 1024);
    // values of K that are left from the lane's first one on; the buffers' bases move on by a step's 128 bytes, their sizes
    // stay (less 128 a step, that of a tile of one row would fall below 0 past the end, and kOob be in range): which lanes
    // load rests on w_left, x_left and off alone
    int w_left = min(a.n_in, u1 * 64) - 8 * ((lane & 7) ^ (lane >> 3)), x_left = w_left;
    const auto move_on = [](i32x4& r, int& left, int steps) {
        const uint64_t p = ((uint64_t)(uint32_t)r[1] << 32 | (uint32_t)r[0]) + 128u * steps;
        r[0] = (int)(uint32_t)p;
        r[1] = (int)(uint32_t)(p >> 32);
        left -= 64 * steps;
    };
    move_on(rw, w_left, u0);
    move_on(rx, x_left, u0);
    const auto later = [](uint32_t at, int tiles) {  // the ring's tile `tiles` (1 .. 4) after
        at += tiles * TILE;
        return at >= RING * TILE ? at - RING * TILE : at;
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int fr = lane & 15;
    u32x4 av[2][MT], bv[2][NT];
    // fragment i of half h of the step whose weights are the ring's tile `at`: the tokens, which the half's first
    // instructions all need, then the weights' rows
    const uint8_t* wb = lds + (wm * MT * 16 + fr) * 128;
    const uint8_t* xb = lds + (wn * NT * 16 + fr) * 128;
    const auto read = [&](uint32_t at, int h, int i) {
        const int k = ((4 * h + (lane >> 4)) ^ (fr & 7)) * 16;
        if (i < NT) bv[h][i] = *reinterpret_cast<const u32x4*>(xb + later(at, 1) + k + i * 2048);
        else av[h][i - NT] = *reinterpret_cast<const u32x4*>(wb + at + k + (i - NT) * 2048);
    };
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
            dma16(base + (i < WS ? 2 * r : 2 * r + 1) * TILE + i % WS * WAVES * 1024, w_left > 0 ? off[i] : kOob, i < WS ? rw : rx, 0);
        move_on(rw, w_left, 1);
        move_on(rx, x_left, 1);
    }
    vmcnt<SLOTS>();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT + NT; ++i) read(0, 0, i);
    // A wave issues in order and a matrix instruction takes 16 cycles, time for three others: what else there is goes in
    // between, one by one.  (One loop for all steps, whose loads past the end are of zeros from past the buffers: between
    // versions of it the compiler would copy the sums.)
    uint32_t at = 0;
    for (int u = u0; u < u1; ++u) {
        const uint32_t next = later(at, 2);
        const auto half = [&](auto which) {
            constexpr int H = decltype(which)::value;
            const uint32_t dst = __builtin_amdgcn_readfirstlane(base + (H ? at : later(at, 4)));
            each_of<MT * NT>([&](auto idx) {
                constexpr int I = decltype(idx)::value, M = I / NT, N = I % NT;
                if constexpr (I % 3 == 0 && I / 3 < MT + NT) read(H ? next : at, 1 - H, I / 3);
                if constexpr (I % 8 == 2)
                    mfma16_dma<F16, I / 8 * WAVES * 1024>(acc[M][N], av[H][M], bv[H][N], dst,
                                                          (H ? x_left : w_left) > 0 ? off[H * WS + I / 8] : kOob, H ? rx : rw);
                else
                    mfma16_in_place<F16>(acc[M][N], av[H][M], bv[H][N]);
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr (H) move_on(rx, x_left, 1);
            else move_on(rw, w_left, 1);
        };
        half(std::integral_constant<int, 0>{});
        // every wave has read this step, and the next one is there (of the one after, its weights may be on their way)
        asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        half(std::integral_constant<int, 1>{});
        at = next;
    }
    vmcnt<0>();
    settle();
    __syncthreads();
    tile_store<MT, NT, 4, PAIR>(a, acc, lds + wave * kStoreBytes<MT, 4>, o0 + wm * (16 * MT / (PAIR ? 2 : 1)), t0 + wn * NT * 16, t0 + n_t,
                             lane);
}

// v[j] of lane p of a quad becomes its lane j's v[p].
__device__ __forceinline__ void turn_quads(u32x4 (&v)[4], int lane) {
    const bool odd = lane & 1, high = lane & 2;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const auto pair = [&](int i, int j, bool second, auto ctrl) {
            constexpr int CTRL = decltype(ctrl)::value;
            const uint32_t a = v[i][d], b = v[j][d];
            const uint32_t pa = __builtin_amdgcn_mov_dpp((int)a, CTRL, 0xF, 0xF, true);
            const uint32_t pb = __builtin_amdgcn_mov_dpp((int)b, CTRL, 0xF, 0xF, true);
            v[i][d] = second ? pb : a;
            v[j][d] = second ? b : pa;
        };
        pair(0, 1, odd, std::integral_constant<int, 0xB1>{});  // lanes 1, 0, 3, 2
        pair(2, 3, odd, std::integral_constant<int, 0xB1>{});
        pair(0, 2, high, std::integral_constant<int, 0x4E>{});  // lanes 2, 3, 0, 1
        pair(1, 3, high, std::integral_constant<int, 0x4E>{});
    }
}

// Up to 16 tokens: 16 outputs to a work-group of eight waves, each every eighth 128 of K, straight from memory to the matrix
// instruction's layout: lane l holds row (or token) l & 15, 8 values of each 32-value quarter l >> 4 of a block at a time.
// That layout's own loads would have neighbouring lanes on different rows, four lines to a quad, and the L1 serve 15 bytes a
// cycle; so the quads load 64 bytes of one row, of four rows in turn, and exchange them (turn_quads): 16 tokens by 2048 x
// 8192 11.3 us for 16.9, by 2048 x 2048 4.9 for 6.3.  BLOCKS blocks of a wave are on their way together (linear_few_blocks).
// Lanes past the last token hold its values, and their results are dropped; the waves' sums meet in LDS, in wave order.
// Bound by the weights' bytes (one token by two matrices of 8192 x 2048, 67 MB, 14.5 us from HBM in turn, 4.6 TB/s; 12 where the
// caches hold part of them, 25 behind a fill that leaves the caches dirty), in few work-groups by what a CU takes in.
template <int BLOCKS, bool PAIR, bool F16>
__global__ __launch_bounds__(512) void k_linear_few(const LinearArgs a) {
    constexpr int SETS = PAIR ? 2 : 1, WAVES = 8;
    __shared__ f32x4 sum_s[WAVES][SETS][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int o0 = blockIdx.x * 16, row = lane & 12, kl = 8 * (4 * (lane >> 4) + (lane & 3)), kq = 32 * (lane >> 4);
    const size_t first = (size_t)o0 * a.n_in;
    const uint16_t* wp[SETS];
    wp[0] = static_cast<const uint16_t*>(a.w) + first;
    if constexpr (PAIR) wp[1] = static_cast<const uint16_t*>(a.w2) + first;
    const uint16_t* xp = static_cast<const uint16_t*>(a.x);
    uint32_t w_at[4], x_at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        w_at[j] = (uint32_t)(min(row + j, a.n_out - 1 - o0) * a.n_in);
        x_at[j] = (uint32_t)(min(row + j, a.n_tokens - 1) * (int)a.x_ld);
    }
    f32x4 acc[SETS];
#pragma unroll
    for (int i = 0; i < SETS; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const u32x4 zero = {0, 0, 0, 0};
    const int blocks = (a.n_in + 127) / 128;
    for (int u = wave; u < blocks; u += BLOCKS * WAVES) {
        u32x4 wv[BLOCKS][SETS][4], xv[BLOCKS][4];
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            const uint32_t k = min((u + b * WAVES) * 128 + kl, a.n_in - 8);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int i = 0; i < SETS; ++i) wv[b][i][j] = *reinterpret_cast<const u32x4*>(wp[i] + (w_at[j] + k));
                xv[b][j] = *reinterpret_cast<const u32x4*>(xp + (x_at[j] + k));
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
            for (int i = 0; i < SETS; ++i) turn_quads(wv[b][i], lane);
            turn_quads(xv[b], lane);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // (past the row: zeros of both, whatever the last values are)
                const bool in = (u + b * WAVES) * 128 + kq + 8 * j < a.n_in;
                const u32x4 x = in ? xv[b][j] : zero;
#pragma unroll
                for (int i = 0; i < SETS; ++i)
                    acc[i] = mfma16<F16>(__builtin_bit_cast(uint4, in ? wv[b][i][j] : zero), __builtin_bit_cast(uint4, x), acc[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < SETS; ++i) sum_s[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 0; i < SETS; ++i)
#pragma unroll
        for (int w = 1; w < WAVES; ++w) acc[i] = acc[i] + sum_s[w][i][lane];
    const int t = lane & 15, o = o0 + 4 * (lane >> 4);
    if (t >= a.n_tokens || o >= a.n_out) return;
    const f32x4 g = acc[0], u = acc[SETS - 1];
    finish4<PAIR>(a, rows_vec(a), t, o, {g[0], g[1], g[2], g[3]}, {u[0], u[1], u[2], u[3]});
}

// The slices' sums added in order, and the epilogue: four outputs of a token to a thread, or one where rows take no vectors.
template <bool PAIR, bool VEC>
__global__ __launch_bounds__(256) void k_linear_join(const LinearArgs a, int slices) {
    const int per = VEC ? (a.n_out + 3) / 4 : a.n_out;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.n_tokens * per) return;
    const int64_t t = i / per;
    const int o = (int)(i % per) * (VEC ? 4 : 1);
    if constexpr (VEC) {
        f32x4 g = *part_at<PAIR>(a, 0, 0, t, o), u = *part_at<PAIR>(a, 0, PAIR, t, o);
        for (int s = 1; s < slices; ++s) {
            g = g + *part_at<PAIR>(a, s, 0, t, o);
            if constexpr (PAIR) u = u + *part_at<PAIR>(a, s, 1, t, o);
        }
        finish4<PAIR>(a, true, t, o, {g[0], g[1], g[2], g[3]}, {u[0], u[1], u[2], u[3]});
    } else {
        const auto one = [&](int s, int which) { return reinterpret_cast<const float*>(part_at<PAIR>(a, s, which, t, o))[o & 3]; };
        float g = one(0, 0), u = one(0, PAIR);
        for (int s = 1; s < slices; ++s) {
            g += one(s, 0);
            if constexpr (PAIR) u += one(s, 1);
        }
        finish1<PAIR>(a, t, o, g, u);
    }
}

hipError_t launch_linear_join(const LinearArgs& a, int slices, hipStream_t s) {
    const bool vec = rows_vec(a) && a.n_out % 4 == 0;
    const int64_t n = (int64_t)a.n_tokens * (vec ? a.n_out / 4 : a.n_out);
    const dim3 grid((unsigned)((n + 255) / 256));
    if (a.w2 && vec) hipLaunchKernelGGL((k_linear_join<true, true>), grid, dim3(256), 0, s, a, slices);
    else if (a.w2) hipLaunchKernelGGL((k_linear_join<true, false>), grid, dim3(256), 0, s, a, slices);
    else if (vec) hipLaunchKernelGGL((k_linear_join<false, true>), grid, dim3(256), 0, s, a, slices);
    else hipLaunchKernelGGL((k_linear_join<false, false>), grid, dim3(256), 0, s, a, slices);
    return hipGetLastError();
}

size_t linear_part_bytes(int64_t T, int K, int N, bool pair) {
    const int slices = linear_plan(T, K, N, pair).slices;
    return slices > 1 ? (size_t)slices * (pair ? 2 : 1) * T * ((N + 3) / 4) * 16 : 0;
}

namespace {
template <int MT, int NT, int WM, int WN, int STAGES, bool PAIR, bool F16>
hipError_t launch_tile(const LinearArgs& a, int slices, hipStream_t s) {
    constexpr int OUTS = 16 * MT * WM / (PAIR ? 2 : 1), BN = 16 * NT * WN;
    const int tiles_o = (a.n_out + OUTS - 1) / OUTS, tiles_t = (a.n_tokens + BN - 1) / BN;
    hipLaunchKernelGGL((k_linear_tile<MT, NT, WM, WN, STAGES, PAIR, F16>), dim3(tiles_o * tiles_t, slices),
                       dim3(64 * WM * WN), 0, s, a, tiles_o, tiles_t);
    return hipGetLastError();
}
template <bool PAIR, bool F16>
hipError_t launch_linear_as(const LinearArgs& a, const LinearPlan& p, hipStream_t s) {
    if (p.kind == kLinearFew) {
        const dim3 grid((a.n_out + 15) / 16);
        if (linear_few_blocks(a.n_in) == 1) hipLaunchKernelGGL((k_linear_few<1, PAIR, F16>), grid, dim3(512), 0, s, a);
        else hipLaunchKernelGGL((k_linear_few<2, PAIR, F16>), grid, dim3(512), 0, s, a);
        return hipGetLastError();
    }
    hipError_t e = hipErrorInvalidValue;
    if (p.kind == kLinear256) {
        const int tiles_o = (a.n_out + (PAIR ? 127 : 255)) / (PAIR ? 128 : 256), tiles_t = (a.n_tokens + 255) / 256;
        hipLaunchKernelGGL((k_linear_big<PAIR, F16>), dim3(tiles_o * tiles_t, p.slices), dim3(256), 0, s, a, tiles_o, tiles_t);
        e = hipGetLastError();
    }
    // tiles of 64 x 32, 64 x 64, 128 x 64 and 128 x 128: two work-groups to a CU but for the last
    if (p.kind == kLinear64x32) e = launch_tile<2, 1, 2, 2, 6, PAIR, F16>(a, p.slices, s);
    if (p.kind == kLinear64) e = launch_tile<2, 2, 2, 2, 5, PAIR, F16>(a, p.slices, s);
    if (p.kind == kLinear128x64) e = launch_tile<4, 2, 2, 2, 3, PAIR, F16>(a, p.slices, s);
    if (p.kind == kLinear128) e = launch_tile<4, 4, 2, 2, 3, PAIR, F16>(a, p.slices, s);
    return e != hipSuccess || p.slices == 1 ? e : launch_linear_join(a, p.slices, s);
}
}  // namespace

hipError_t launch_linear(const LinearArgs& a, hipStream_t s) {
    const LinearPlan p = linear_plan(a.n_tokens, a.n_in, a.n_out, a.w2 != nullptr);
    const bool f16 = a.w_type == kF16;
    if (a.w2) return f16 ? launch_linear_as<true, true>(a, p, s) : launch_linear_as<true, false>(a, p, s);
    return f16 ? launch_linear_as<false, true>(a, p, s) : launch_linear_as<false, false>(a, p, s);
}

}  // namespace smoe
