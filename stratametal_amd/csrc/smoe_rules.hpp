// stratametal_amd/csrc/smoe_rules.hpp - which kernel a call runs on, where the choice was measured: plain host
// functions of a call's sizes, so that a CPU test can hold them to the times they come from
// (tests/test_dispatch_rules.py).
#pragma once

#include <cstdint>
#include <initializer_list>

namespace smoe {

// The register slots of a token's streams in k_hc_proj and k_hc_act: HC streams of NM values per thread.  Every slot
// is loaded (the indices clamped into the row), so a spare one is a load too: the least that hold hc streams of n
// values (with 4 and 8 streams of 2, 8 and 16 alone the read of 16 tokens, hc 1, n 1024, hc_lr 320, took 14.0 us,
// with branches around the loads 13.4, so 10.1).
constexpr int kHcStreams[] = {2, 4, 8}, kHcValues[] = {2, 4, 6, 8, 10, 12, 16};
constexpr int hc_streams(int hc) {
    for (const int s : kHcStreams)
        if (hc <= s) return s;
    return 8;
}
constexpr int hc_values(int n) {
    for (const int v : kHcValues)
        if (n <= 256 * v) return v;
    return 16;
}
// 16-byte pieces of a weight row per lane: hc n / 512 rounded up to a multiple of eight.
constexpr int hc_chunks(int n, int hc) { return (hc * n / 8 + 511) / 512 * 8; }

// The same for the pieces of an `up` row per lane of k_hc_mix (hc_lr / 64 rounded up; five for one piece: the read of
// 64 tokens, hc 5, n 512, hc_lr 64, 14.5 us, with branches around the loads 13.7, with one 13.0).
constexpr int kHcPieces[] = {1, 2, 3, 4, 5, 8, 16, 32};
constexpr int hc_pieces(int hc_lr) {
    for (const int p : kHcPieces)
        if (hc_lr <= 64 * p) return p;
    return 32;
}

// The norm's slots are loaded with the streams' (one memory round trip less: 2 us of 13 at one token, n 2560, hc 4)
// where both fit 256 registers beside the weight row's `more`, two waves per SIMD.
constexpr bool hc_norm_fits(int slots, int more) { return 2 * slots + more <= 192; }
// Where they don't, the norm is loaded with the streams by one wave per SIMD or, where the streams and the weight row
// alone fit, after the scales are formed by two: by two where that halves the rounds of work-groups over the 256 CUs
// and an XCD's L2 holds the weights (n 2048, hc 6, hc_lr 64: 16 tokens, 288 work-groups, 26.7 us in two rounds of one
// wave, 21.7 in one of two waves; 14 tokens, 252, 17.6 against 20.2; hc 8, hc_lr 320: 4 tokens, 328, 32.3 against
// 34.3).
constexpr bool hc_norm_ahead(int slots, int more, int64_t groups, int64_t weight_bytes) {
    return hc_norm_fits(slots, more) || slots + more > 192 || (groups + 255) / 256 % 2 == 1 ||
           weight_bytes > (int64_t)5 << 20;
}

// Whether the read of a batch runs on the matrix cores: from 17 tokens (a second 16-token tile) and 2^23 products of
// the projection, where the row-per-wave kernels' time, which grows with the tokens, has passed the four launches',
// which hardly does but grows with the streams and hc_lr.  Fitted to 60 shapes of 8 to 400 tokens; rows and matrix
// cores, us: hc 4, hc_lr 320, n 2048 30 and 28 at 17 tokens, 82 and 31 at 64, 1965 and 66 at 1000; n 512 11 and 24 at
// 17, 24 and 26 at 64, 38 and 28 at 128; hc 8, n 256 45 and 36 at 128; hc 4, hc_lr 64, n 2048 17 and 20 at 24, 32 and
// 21 at 64; hc 1, hc_lr 960, n 4096 114 and 35 at 17.
constexpr bool hc_mm_gains(int64_t T, int n, int hc, int hc_lr) {
    return T >= 17 && T * hc * n * hc_lr >= (int64_t)1 << 23 &&
           120 * T * n * (hc * (hc_lr + 80) + hc_lr + 160) >= (int64_t)92 * 32768 * (960 + 360 * hc + hc_lr);
}

// The write of T tokens: kHcWriteValues a value per thread; else 16-byte vectors (n % 4 == 0 and aligned buffers), a
// work-group's piece of y through one stream (kHcWriteStream) or through all (kHcWriteStreams: y read once, from
// where the launch is long; rows of few values leave lanes idle in every piece, and one or two streams re-read
// little, so earlier).  us by value, by stream and through all: hc 8, n 64, 200 tokens 2.5, 2.6, 3.5, 4000 tokens
// 7.3, 13.0, 6.5; hc 8, n 512, 64 tokens 2.7, 2.5, 3.4; hc 4, n 2048, 64 tokens 3.3, 2.6, 2.9, 1000 tokens 21.5,
// 10.6, 11.6, 4000 tokens 98, 56, 44.
enum HcWrite { kHcWriteValues, kHcWriteStream, kHcWriteStreams };
constexpr HcWrite hc_write_kind(int64_t T, int n, int hc) {
    const int64_t limit = n < 512 ? 15 << 16 : n < 768 ? 15 << 17 : hc <= 2 ? 6 << 20 : 11 << 20;
    const bool all = T * hc * n >= limit;
    return n < 64 || (n < 256 && !all) ? kHcWriteValues : all ? kHcWriteStreams : kHcWriteStream;
}

// Whether an IQ2_S layer's products of P routed pairs run on the matrix cores (tiles of 16 columns; the row kernels'
// cost grows with the columns).  An item's tiles go one after the other, so few experts leave the chip idle: from
// seven or eight pairs per expert on where the products' work-groups, each as long as its rows, fill it; else from
// 64, or 128 with fewer than 32 experts, where an expert's pairs are several items.  Rows against matrix cores, the
// whole call: 512 experts of 2048 x 512 389 and 408 us at 5.9 pairs, 648 and 472 at 11.7; 128 experts of 2048 x 512,
// most pairs in 16 of them, 150 and 189 at 6.3, 1.05 times as fast at 8; 16 experts 70 and 102 at 12.5, 137 and 188
// at 38, 1.3 times as fast at 100; 32 experts of 1024 x 2048 0.84 times at 11, 1.34 at 64; of 2048 x 2048 187 and 161
// at 12.5.
constexpr bool iq2_mm_gains(int64_t P, int E, int H, int F) {
    const bool fills = (E >= 64 || (E >= 32 && H * F >= 2048 * 2048)) && (int64_t)E * F * 8 / H >= 128 &&
                       (int64_t)E * H * 4 / F >= 128;
    return P >= (int64_t)E * (fills ? E >= 128 ? 7 : 8 : E >= 32 ? 64 : 128);
}

// The native types' GEMV of n_col columns (nz matrices by one launch): columns per work-group of the column tiles, or
// 1 for a work-group per column and eight rows.  The most of 16, 8 and 4 that is not half empty and leaves the chip
// two work-groups per CU, else 4; a tile's chain of columns is the longer one, so few work-groups of 4 columns go by
// columns (512 x 2048 at 16 columns 3.9 to 6.6 us by type against 5.0 to 8.5 in tiles, at 32 5.8 to 10.9 against 4.1
// to 8.4).  Q4_K, Q5_K and Q6_K, whose decode the tiles save little of, from six or eight columns and more
// work-groups, long rows more yet (by columns and in tiles: Q4_K 256 x 20000 at 4 columns 8.3 and 12.4, Q5_K 512 x
// 2048 at 5 3.2 and 3.7, Q6_K 8192 x 1000 at 24 40 and 49, at 48 1.4 times as fast in tiles).
constexpr int kNativeTileRows = 16;
constexpr int native_cols(int type, int n_in, int n_out, int n_col, int nz) {
    const int64_t rg = ((int64_t)n_out + kNativeTileRows - 1) / kNativeTileRows * nz;
    const bool k = type == 12 || type == 13 || type == 14;
    const int64_t least = !k || n_col >= 128 ? 224 : n_in <= 4096 ? 336 : 480;
    if (n_col < (!k ? 4 : rg >= 256 ? 6 : 8) || n_col / 4 >= 65535 || rg * ((n_col + 3) / 4) < least) return 1;
    for (const int c : {16, 8})
        if (2 * n_col > c && rg * ((n_col + c - 1) / c) >= 512) return c;
    return 4;
}

// A native shared expert of T tokens in two launches (k_native_gu, k_native_down): every work-group quantises its
// token's whole row again and takes eight rows of it, so the stage kernels, whose tokens share a row's decode and one
// quantised row, win where tokens times weights are many (the layer's call with the two launches against it, Q8_0: 4
// tokens 2048 x 512 1.16 times as fast, 1 token 4096 x 4096 1.00, 2 tokens 3072 x 1536 1.05, 2048 x 2048 1.14, 4
// tokens 0.97, 4096 x 4096 0.63; Q4_K 3 tokens 3072 x 1536 0.93).
constexpr bool native_few_gains(int T, int H, int F) { return T <= 4 && (int64_t)T * H * F <= (int64_t)10 << 20; }

// The native shared expert's products of a prompt on the matrix cores (nz matrices of n_out rows by one launch): a
// chunk of K after the other is a chain of latencies, so from 128 columns, and 128 tiles of 32 rows by 32 columns
// (the layer's call on the matrix cores against the row kernels: Q8_0 2048 x 512 0.81 at 5 columns, 0.88 at 64, 0.98
// at 128, 1.05 at 200; gate and up apart 0.70 at 8, 0.89 at 128; Q3_K 1.07 at 128, 1.42 at 400).
constexpr bool native_mm_gains(int n_out, int n_col, int nz) {
    return n_col >= 128 && (int64_t)((n_out + 31) / 32) * ((n_col + 31) / 32) * nz >= 128;
}

// Whether the router of T tokens without the fused junction runs k_router_tile: from five tokens on, but for long
// bf16 rows of few experts, whose waves walk K in stages while most of the chip is idle.  512 rows of 2048, k_router
// and the tiles, us: bf16 6.3 and 6.3 at 5 tokens, 8.4 and 6.4 at 16, 19.8 and 7.7 at 64, 126 and 38 at 600; f32 7.8
// and 5.9 at 5, 27 and 7.1 at 64.  bf16 rows of 4096, the tiles' gain: 8 experts -1.0 at 8 tokens, +1.6 at 64; 32
// experts -1.8 at 5; 128 experts -0.4 at 8, +0.3 at 16; 512 experts 0.0 at 5, +2.4 at 16.
constexpr bool router_tiles(int64_t T, int E, int H, bool f32) {
    return T >= 5 && (f32 || H <= 2560 || T * (E > 64 ? E : 64) >= 2048);
}

// The tile: few tokens or experts need the work-groups (bf16 4 rows by 4 tokens, f32 2 by 8), many of both re-read
// less in tiles of 4 by 8 (512 rows of 2048, bf16 9.6 against 10.4 us at 100 tokens, 11.4 against 10.7 at 127; rows
// of 4096 at 127 tokens in tiles of 4 by 8 the same with 400 and 512 experts, 4.6 us longer with 256 and 4.8 with 64;
// f32 64 experts 3.1 us longer at 300 tokens, 128 experts 0.3 at 448).
constexpr bool router_tile_wide(int64_t T, int E) { return T >= 112 && T * E >= 112 * 512; }

// The tiled router's one-dimensional grid: the tiles of tt tokens by 4 rr rows, those of a row group, or by_tok of a
// token tile, on one XCD (whole groups of 8).  A launch holds kGridGroups work-groups of 256 threads in a dimension and
// takes a larger grid modulo that, with no error: a larger product, of some 2^31 outputs and more, is refused.
constexpr int64_t kGridGroups = 0xFFFFFFFFll / 256;
constexpr bool router_by_tok(int64_t T, int64_t E, bool f32) { return T * 4 > E * (f32 ? 4 : 2); }  // x, not W, on every XCD
constexpr int64_t router_tile_grid(int64_t T, int64_t E, bool f32, int rr, int tt) {
    const int64_t rb = (E + 4 * rr - 1) / (4 * rr), tb = (T + tt - 1) / tt;
    return router_by_tok(T, E, f32) ? (tb + 7) / 8 * 8 * rb : (rb + 7) / 8 * 8 * tb;
}
constexpr bool router_tile_fits(int64_t T, int E, int H, bool f32) {
    const bool wide = router_tile_wide(T, E);
    return router_tile_grid(T, E, f32, f32 && !wide ? 2 : 4, !f32 && !wide ? 4 : 8) + T + T * (H / 32) / 8 < kGridGroups;
}

// Whether the decode path runs the junction of T tokens as a kernel of its own: fused into the router kernel it saves
// the launch, and repeats the norm in every work-group of the router.  Apart from 12 tokens on where the tiled
// router's gain passes the launch, us: bf16, 512 experts of 2048 +0.4 at 10 tokens, +0.8 at 12, +3.6 at 16, 28.8 to
// 12.0 at 48; 64 experts of 2048 -0.6 at 12, -1.3 at 16, +0.3 at 32; of 4096 -1.4 at 12, +4.4 at 32; 256 experts of
// 512 +0.4 at 12, +1.1 at 32; 8 experts of 512 -0.6 at 32, +7 at 127; f32 rows longer than 2048 +4 and more at any
// number of experts.
constexpr bool junction_apart(int64_t T, int E, int H, bool f32) {
    return T >= 12 && ((f32 && H > 2048) || T >= (H >= 2048 ? 32 : 80) ||
                       T * E >= (H >= 2560 ? 2048 : H >= 2048 ? 4096 : 8192));
}

// The ends of a block: lanes to a row, and slots of four values to a lane.
struct EndsShape {
    int lanes, slots;
};
constexpr int kEndsMaxRow = 16384;
constexpr EndsShape ends_shape(int n) {
    return n <= 64 ? EndsShape{16, 1} : n <= 128 ? EndsShape{32, 1} : n <= 256 ? EndsShape{64, 1} : n <= 512 ? EndsShape{64, 2}
           : n <= 1024 ? EndsShape{256, 1} : n <= 2048 ? EndsShape{256, 2} : n <= 4096 ? EndsShape{512, 2}
           : n <= 8192 ? EndsShape{1024, 2} : EndsShape{1024, 4};
}
// Work-groups: as many as the chip holds at a time (16 waves to a CU), each taking rows in turn.
constexpr int64_t ends_groups(int64_t T, int n) {
    const int lanes = ends_shape(n).lanes, rows = lanes < 256 ? 256 / lanes : 1;
    const int64_t sets = (T + rows - 1) / rows, most = 256 * 1024 / (lanes < 256 ? 256 : lanes);
    return sets < most ? sets : most;
}

// The router's balance loss: one work-group for a few tokens (64 tokens of 512 experts 15.7 us with gradients, in two launches
// 18.9; 256 tokens 38 and 19.5).
constexpr bool balance_one(int64_t T, int k) { return T <= 64 && T * k <= 4096; }
// The pairs counted first, by a launch of their own, or by every work-group that needs them: with gradients those of the rows
// (us apart and not: 2560 pairs 18.7 and 19.5 with a mask, 17.6 and 17.0 without, 5120 19.5 and 23.2, 10240 20.5 and
// 28.8), else those of the sums, few and large (10240 pairs 16.4 and 15.5).  One work-group has no other to count for.
constexpr bool balance_counts_apart(int64_t T, int k, bool grad) {
    return !balance_one(T, k) && T * k > (grad ? 3000 : 12000);
}
// Work-groups of four rows at a time, at most 512 (k_balance_sums takes up to 1024): each leaves a row of partial sums (4096
// tokens of 512 experts 27.5 us with 256 or 512 of them, 31.8 with 1024, 30.4 with 128; 32768 of 1024 99, 77.5, 79.8, 151).
constexpr int64_t balance_groups(int64_t T) { return T < 4 ? 1 : (T + 3) / 4 < 512 ? (T + 3) / 4 : 512; }
// Work-groups of the counts, whose rows every reader adds up (4096 tokens 29.8 us with 8, 31.7 with 16; 32768 84 and 80,
// with 64 95).
constexpr int64_t balance_count_groups(int64_t T) { return T < 1024 ? 1 : T / 512 < 16 ? T / 512 : 16; }

// The dense product: a row of x or w, rows of w, and the distance of x's rows (a tile of 256 rows stays within 31-bit
// offsets).
constexpr int kLinearMaxIn = 65536, kLinearMaxOut = 1 << 24;
constexpr int64_t kLinearMaxLd = (int64_t)1 << 21;
// Which kernel, and in how many slices of K.
enum LinearKind { kLinearFew, kLinear64x32, kLinear64, kLinear128x64, kLinear128, kLinear256 };
struct LinearPlan {
    LinearKind kind;
    int slices;
};
struct LinearTile {
    int rows, tokens;    // of w (and w2), of x
    int per_cu;          // work-groups that a CU's LDS holds
    double fixed;        // us of a work-group beside its steps
    double step, shared; // us of a step of 64 of K, alone on a CU and with the others
    double astride;      // as much longer with rows that start inside a 128-byte line: a step's piece of one is of two lines
};
constexpr LinearTile kLinearTiles[] = {{},
                                       {64, 32, 2, 0.8, 0.18, 0.42, 1.0},
                                       {64, 64, 2, 1.5, 0.23, 0.48, 1.3},
                                       {128, 64, 2, 1.8, 0.40, 0.71, 1.4},
                                       {128, 128, 1, 2.4, 0.62, 0.62, 1.1},
                                       {256, 256, 1, 11.3, 1.24, 1.24, 1.0}};
// The rows' kernel: blocks of 128 of K that each of a work-group's eight waves has on its way: one where two would not come
// out even (1 and 2, us, 1 token, n_in x n_out: 512 x 512 2.9 and 3.3, 1024 x 16384 7.9 and 9.9, 2568 x 5003 8.4 and 9.2;
// 2048 x 2048 5.1 and 4.9, 4096 x 4096 8.6 and 8.2, 8192 x 2048 11.4 and 10.3).
constexpr int linear_few_blocks(int64_t K) {
    const int64_t each = (K + 1023) / 1024;  // a wave's blocks
    return each == 1 || each == 3 ? 1 : 2;
}
// A product's time in us, from its sizes (n_in x n_out below): the rounds of work-groups over the 256 CUs times their
// steps, or the bytes of w and x at 6 bytes a ps where those take longer, and where K is sliced the launch and the bytes
// that join the sums; the rows' kernel takes in the weights by each CU's rate.  Fitted to 254 shapes (9 of 256 to 8192 by
// 512 to 16384, 1 to 2500 tokens, one matrix and pairs), each timed by every kernel in 1 to 8 slices: the kernel of the
// least of it takes on average 0.9 % longer than the shape's fastest, at most 25 %; the rows' kernel anew to 36 of 1 and
// 16 tokens, its choice within 5 % but for one matrix 8192 x 512 (tiles in slices 10.6 for 9.6).  us, by few, 64 x 32, 64
// x 64, 128 x 64, 128 x 128 and 256 x 256: 1 token 2048 x 2048 4.9, 8.2, 9.7, -, -, -; 9 tokens 2048 x 8192 8.2, 8.6,
// 10.1, -, -, -; 16 tokens 8192 x 2048 11.3, 24.1, 29.6 and in four slices -, 12.0, 13.9, by two matrices 21.4, 27.9 and
// in four slices 18.6; 128 tokens 2048 x 8192 -, -, 12.9, 18.7, 23.3, -; 301 tokens 2560 x 5004 -, -, 21.2, 20.4, 24.3, -
// and in two slices -, -, -, 24.4, 21.1, 37, the same of 2568 -, -, 30.0, 27.8, 30.9, - and -, -, -, 28.9, 24.1, 40; 4096
// tokens 4096 x 4096 -, -, 232, 191, 157, 102.
inline double linear_time(LinearKind kind, int slices, int64_t T, int64_t K, int64_t N, bool pair) {
    const int64_t rows = pair ? 2 * N : N;
    const double w_bytes = (double)rows * (double)K * 2, x_bytes = (double)T * (double)K * 2;
    if (kind == kLinearFew) {
        const int64_t wg = (N + 15) / 16;
        const double cus = w_bytes / ((double)(wg < 256 ? wg : 256) * (pair ? 31e3 : 36e3));  // what a CU takes in
        return 2.9 + (cus > w_bytes / 6.4e6 ? cus : w_bytes / 6.4e6) * (1 + 0.002 * (double)(T - 1));
    }
    const LinearTile& t = kLinearTiles[kind];
    const int64_t wg = (rows + t.rows - 1) / t.rows * ((T + t.tokens - 1) / t.tokens) * slices;
    const int64_t steps = ((K + 63) / 64 + slices - 1) / slices;
    const int64_t at_once = wg <= 256 ? 1 : t.per_cu, rounds = (wg + 256 * at_once - 1) / (256 * at_once);
    const double step = (at_once == 1 ? t.step : t.shared) * (K % 64 ? t.astride : 1);
    const double work = (double)rounds * (t.fixed + (double)steps * step);
    const double bytes = t.fixed + (w_bytes + x_bytes) / 6.4e6;
    return 2.4 + (work > bytes ? work : bytes) + (slices > 1 ? 2.9 + 0.31e-6 * 4 * (double)(slices * T * rows) : 0);
}
constexpr int64_t kLinearFewTokens = 16;
inline LinearPlan linear_plan(int64_t T, int64_t K, int64_t N, bool pair) {
    LinearPlan best{kLinear64, 1};
    double least = -1;
    for (int kind = T <= kLinearFewTokens ? kLinearFew : kLinear64x32; kind <= kLinear256; ++kind)
        for (const int slices : {1, 2, 4, 8}) {
            // (a slice of two steps and more; slices only where the tiles are few)
            if (slices > 1) {
                if (kind == kLinearFew || K / 64 < 2 * slices) continue;
                const LinearTile& t = kLinearTiles[kind];
                const int64_t rows = pair ? 2 * N : N;
                if ((rows + t.rows - 1) / t.rows * ((T + t.tokens - 1) / t.tokens) * slices > 1100) continue;
            }
            const double us = linear_time((LinearKind)kind, slices, T, K, N, pair);
            if (least < 0 || us < least) least = us, best = LinearPlan{(LinearKind)kind, slices};
        }
    return best;
}
inline int64_t linear_groups(LinearPlan p, int64_t T, int64_t N, bool pair) {
    if (p.kind == kLinearFew) return (N + 15) / 16;
    const LinearTile& t = kLinearTiles[p.kind];
    return ((pair ? 2 * N : N) + t.rows - 1) / t.rows * ((T + t.tokens - 1) / t.tokens);
}

}  // namespace smoe
