// stratametal_amd/csrc/smoe_attention.cpp - the C ABI of the attention in front of the block (include/smoe.h): argument checks
// and launches of smoe_rope.hip and smoe_attend.hip.  As in smoe_api.cpp every refusal happens before the first launch, and
// a zero count returns before launching.
#include "smoe.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "smoe_check.hpp"
#include "smoe_launch.hpp"
#include "smoe_rules.hpp"

using namespace smoe;

namespace {

constexpr int kMaxHeads = 4096;

smoe_status check_rope(const smoe_rope* r, const char* what) {
    if (!r) return fail(SMOE_ENULL, std::string(what) + ": the rotary positions are NULL");
    if (r->head_dim < 2 || r->head_dim > 1024 || r->head_dim % 2)
        return fail(SMOE_EINVAL, std::string(what) + ": head_dim must be even, 2 to 1024");
    if (r->rot_dim < 2 || r->rot_dim > r->head_dim || r->rot_dim % 2)
        return fail(SMOE_EINVAL, std::string(what) + ": rot_dim must be even, 2 to head_dim");
    if (r->layout != SMOE_ROPE_HALF && r->layout != SMOE_ROPE_PAIRS)
        return fail(SMOE_EINVAL, std::string(what) + ": layout is SMOE_ROPE_HALF or SMOE_ROPE_PAIRS");
    if (!finite(r->scale)) return fail(SMOE_EINVAL, std::string(what) + ": scale must be finite");
    return SMOE_OK;
}

smoe_status check_kv(const smoe_kv* kv, const char* what) {
    if (!kv) return fail(SMOE_ENULL, std::string(what) + ": the cache is NULL");
    if (kv->type != SMOE_BF16 && kv->type != SMOE_F16)
        return fail(SMOE_ETYPE, std::string(what) + ": the cache is SMOE_BF16 or SMOE_F16");
    if (kv->head_dim < 8 || kv->head_dim > 256 || kv->head_dim % 8)
        return fail(SMOE_EINVAL, std::string(what) + ": head_dim must be a multiple of 8, 8 to 256");
    if (kv->n_kv_heads < 1 || kv->n_kv_heads > kMaxHeads)
        return fail(SMOE_EINVAL, std::string(what) + ": n_kv_heads must be 1 to " + std::to_string(kMaxHeads));
    if (kv->page_size < 1 || kv->page_size > 65536) return fail(SMOE_EINVAL, std::string(what) + ": page_size must be 1 to 65536");
    if (kv->n_pages < 1 || (int64_t)kv->n_pages * kv->n_kv_heads >= ((int64_t)1 << 31) / kv->page_size)
        return fail(SMOE_EINVAL, std::string(what) + ": pages, heads and tokens together must be 1 to 2^31 - 1");
    return SMOE_OK;
}

Span pages_of(const smoe_kv* kv, const void* p) {
    return bytes_of(p, (int64_t)kv->n_pages * kv->n_kv_heads * kv->page_size * kv->head_dim * 2);
}

// Rows of n_heads heads: a token's values are contiguous.
bool bad_rows(int64_t ld, int64_t n_tokens, int64_t n) { return bad_ld(ld, n_tokens, n); }

}  // namespace

extern "C" {

// ------------------------------------------------------------------------------------------------ rotary positions

smoe_status smoe_rope_table(int32_t rot_dim, double base, int32_t scaling, double factor, double trained_len, double slow,
                            double fast, double* turns, float* scale) {
    if (!turns || !scale) return fail(SMOE_ENULL, "rope_table: turns or scale is NULL");
    if (rot_dim < 2 || rot_dim > 1024 || rot_dim % 2) return fail(SMOE_EINVAL, "rope_table: rot_dim must be even, 2 to 1024");
    if (!(base > 0) || !std::isfinite(base)) return fail(SMOE_EINVAL, "rope_table: base must be positive");
    if (scaling < SMOE_ROPE_NONE || scaling > SMOE_ROPE_PARTS) return fail(SMOE_EINVAL, "rope_table: unknown scaling");
    if (scaling != SMOE_ROPE_NONE && (!(factor > 0) || !std::isfinite(factor)))
        return fail(SMOE_EINVAL, "rope_table: factor must be positive");
    if (scaling == SMOE_ROPE_PARTS && (!(trained_len > 0) || !std::isfinite(trained_len) || !std::isfinite(slow) || !(fast > slow) ||
                                       !std::isfinite(fast)))
        return fail(SMOE_EINVAL, "rope_table: parts need trained_len > 0 and fast > slow");
    constexpr double kTurn = 6.283185307179586476925;
    if (scaling == SMOE_ROPE_BASE && rot_dim > 2) base *= std::pow(factor, (double)rot_dim / (rot_dim - 2));
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (scaling == SMOE_ROPE_LINEAR) f /= factor;
        if (scaling == SMOE_ROPE_PARTS) {
            double g = (trained_len * f / kTurn - slow) / (fast - slow);
            g = g < 0 ? 0 : g > 1 ? 1 : g;
            f *= g + (1 - g) / factor;
        }
        turns[i] = f / kTurn;
        if (!std::isfinite(turns[i])) return fail(SMOE_EINVAL, "rope_table: the frequencies leave 64 bits");
    }
    *scale = scaling == SMOE_ROPE_PARTS ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return ok();
}

smoe_status smoe_rope_run(const smoe_rope* r, const int32_t* positions, int32_t n_tokens, int32_t n_heads, const void* x,
                          int32_t x_type, int64_t x_ld, void* y, int32_t y_type, int64_t y_ld, void* hip_stream) {
    const smoe_status s = check_rope(r, "rope");
    if (s != SMOE_OK) return s;
    if (n_tokens < 0) return fail(SMOE_EINVAL, "rope: negative token count");
    if (!rope_fits(n_tokens)) return fail(SMOE_EINVAL, "rope: the tokens exceed a launch's grid: split them");
    if (n_heads < 1 || n_heads > kMaxHeads) return fail(SMOE_EINVAL, "rope: n_heads must be 1 to " + std::to_string(kMaxHeads));
    if (!elem_type(x_type) || !elem_type(y_type)) return fail(SMOE_ETYPE, "rope: rows are SMOE_F32, SMOE_F16 or SMOE_BF16");
    if (n_tokens == 0) return ok();
    if (!positions || !x || !y || !r->turns) return fail(SMOE_ENULL, "rope: NULL buffer");
    const int64_t n = (int64_t)n_heads * r->head_dim;
    if (bad_rows(x_ld, n_tokens, 0) || bad_rows(y_ld, n_tokens, n))
        return fail(SMOE_EINVAL, "rope: row strides must not be negative, and y's rows not overlap");
    if (!aligned(x, elem_size(x_type)) || !aligned(y, elem_size(y_type)) || !aligned(positions, 4) || !aligned(r->turns, 8))
        return fail(SMOE_EALIGN, "rope: a buffer is not aligned to its values");
    const Span sx = rows_of(x, x_type, n_tokens, x_ld, n), sy = rows_of(y, y_type, n_tokens, y_ld, n);
    if (overlap(sy, sx) && !(same(sy, sx) && x_type == y_type)) return fail(SMOE_EINVAL, "rope: y is x's own rows or shares none with it");
    if (overlap(sy, bytes_of(positions, 4ll * n_tokens)) || overlap(sy, bytes_of(r->turns, 4ll * r->rot_dim)))
        return fail(SMOE_EINVAL, "rope: y overlaps the positions or the table");
    RopeArgs a{};
    a.turns = r->turns, a.positions = positions;
    a.q = x, a.q_out = y, a.q_ld = n_tokens > 1 ? x_ld : 0, a.q_out_ld = n_tokens > 1 ? y_ld : 0;
    a.n_tokens = n_tokens, a.n_heads = n_heads, a.head_dim = r->head_dim, a.rot = r->rot_dim, a.half = r->layout == SMOE_ROPE_HALF;
    a.page_size = 1, a.x_type = x_type, a.q_type = y_type, a.t_type = SMOE_BF16, a.scale = r->scale;
    return launched(launch_rope(a, reinterpret_cast<hipStream_t>(hip_stream)), "rope");
}

// ------------------------------------------------------------------------------------------------ paged cache

smoe_status smoe_kv_append(const smoe_kv* kv, const smoe_rope* r, const int32_t* positions, const int64_t* slots,
                           int32_t n_tokens, int32_t x_type, const void* q, int64_t q_ld, int32_t n_heads, void* q_out,
                           int64_t q_out_ld, const void* k, int64_t k_ld, const void* v, int64_t v_ld, void* hip_stream) {
    smoe_status s = check_kv(kv, "kv_append");
    if (s == SMOE_OK && r) s = check_rope(r, "kv_append");
    if (s != SMOE_OK) return s;
    if (r && r->head_dim != kv->head_dim) return fail(SMOE_EINVAL, "kv_append: the rotary positions' head_dim is not the cache's");
    if (n_tokens < 0) return fail(SMOE_EINVAL, "kv_append: negative token count");
    if (!rope_fits(n_tokens)) return fail(SMOE_EINVAL, "kv_append: the tokens exceed a launch's grid: split them");
    if (!elem_type(x_type)) return fail(SMOE_ETYPE, "kv_append: rows are SMOE_F32, SMOE_F16 or SMOE_BF16");
    if (!q != !q_out) return fail(SMOE_ENULL, "kv_append: q and q_out go together");
    if (q && !r) return fail(SMOE_EINVAL, "kv_append: queries without rotary positions");
    if (q && (n_heads < 1 || n_heads > kMaxHeads))
        return fail(SMOE_EINVAL, "kv_append: n_heads must be 1 to " + std::to_string(kMaxHeads));
    if (n_tokens == 0) return ok();
    if (!kv->k || !kv->v || !k || !v || !slots || (r && (!positions || !r->turns))) return fail(SMOE_ENULL, "kv_append: NULL buffer");
    const int64_t n = (int64_t)kv->n_kv_heads * kv->head_dim, nq = q ? (int64_t)n_heads * kv->head_dim : 1;
    if (bad_rows(k_ld, n_tokens, 0) || bad_rows(v_ld, n_tokens, 0) || (q && (bad_rows(q_ld, n_tokens, 0) || bad_rows(q_out_ld, n_tokens, nq))))
        return fail(SMOE_EINVAL, "kv_append: row strides must not be negative, and q_out's rows not overlap");
    const size_t es = elem_size(x_type);
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return fail(SMOE_EALIGN, "kv_append: the cache must be 16-byte aligned");
    if (!aligned(q, es) || !aligned(k, es) || !aligned(v, es) || !aligned(q_out, 2) || !aligned(slots, 8) ||
        (r && (!aligned(positions, 4) || !aligned(r->turns, 8))))
        return fail(SMOE_EALIGN, "kv_append: a buffer is not aligned to its values");
    const Span sq = rows_of(q, x_type, n_tokens, q_ld, nq), so = rows_of(q_out, kv->type, n_tokens, q_out_ld, nq);
    const Span in[] = {rows_of(k, x_type, n_tokens, k_ld, n), rows_of(v, x_type, n_tokens, v_ld, n), bytes_of(slots, 8ll * n_tokens),
                       bytes_of(r ? positions : nullptr, 4ll * n_tokens), bytes_of(r ? r->turns : nullptr, r ? 4ll * r->rot_dim : 1)};
    const Span out[] = {so, pages_of(kv, kv->k), pages_of(kv, kv->v)};
    for (const Span& o : out) {
        for (const Span& i : in)
            if (overlap(o, i)) return fail(SMOE_EINVAL, "kv_append: the cache or q_out overlaps an input");
        if (overlap(o, sq) && !(&o == &out[0] && same(o, sq) && x_type == kv->type))
            return fail(SMOE_EINVAL, "kv_append: q_out is q's own rows or shares none with it, nor does the cache");
    }
    if (overlap(out[0], out[1]) || overlap(out[0], out[2]) || overlap(out[1], out[2]))
        return fail(SMOE_EINVAL, "kv_append: two outputs overlap");
    RopeArgs a{};
    a.slots = slots, a.q = q, a.k = k, a.v = v;
    a.q_out = q_out, a.k_pages = kv->k, a.v_pages = kv->v;
    a.n_slots = (int64_t)kv->n_pages * kv->page_size;
    if (n_tokens > 1) a.q_ld = q_ld, a.q_out_ld = q_out_ld, a.k_ld = k_ld, a.v_ld = v_ld;
    a.n_tokens = n_tokens, a.n_heads = q ? n_heads : 0, a.n_kv = kv->n_kv_heads, a.head_dim = kv->head_dim, a.page_size = kv->page_size;
    if (r) a.turns = r->turns, a.positions = positions, a.rot = r->rot_dim, a.half = r->layout == SMOE_ROPE_HALF, a.scale = r->scale;
    a.x_type = x_type, a.q_type = kv->type, a.t_type = kv->type;
    return launched(launch_rope(a, reinterpret_cast<hipStream_t>(hip_stream)), "kv_append");
}

// ------------------------------------------------------------------------------------------------ attention

static smoe_status check_attend(const smoe_kv* kv, int32_t n_heads, int32_t n_tokens, int32_t n_seqs, int64_t max_len) {
    const smoe_status s = check_kv(kv, "attend");
    if (s != SMOE_OK) return s;
    if (n_heads < 1 || n_heads > kMaxHeads || n_heads % kv->n_kv_heads)
        return fail(SMOE_EINVAL, "attend: n_heads must be a multiple of n_kv_heads, at most " + std::to_string(kMaxHeads));
    if (n_tokens < 0 || n_seqs < 0) return fail(SMOE_EINVAL, "attend: negative count");
    if ((int64_t)n_tokens * n_heads >= ((int64_t)1 << 31) / 256 || n_seqs > (1 << 20))
        return fail(SMOE_EINVAL, "attend: at most 2^23 query rows (tokens times heads) and 2^20 sequences: split the batch");
    if (max_len < 0 || max_len > ((int64_t)1 << 30)) return fail(SMOE_EINVAL, "attend: max_len must be 0 to 2^30");
    return SMOE_OK;
}

size_t smoe_attend_workspace_bytes(const smoe_kv* kv, int32_t n_heads, int32_t n_tokens, int32_t n_seqs, int64_t max_len,
                                   int32_t window) {
    if (check_attend(kv, n_heads, n_tokens, n_seqs, max_len) != SMOE_OK) return 0;
    if (window < 0) {
        fail(SMOE_EINVAL, "attend: a window must be positive");
        return 0;
    }
    ok();
    return 256 + attend_part_bytes(n_tokens, n_seqs, n_heads, kv->n_kv_heads, kv->head_dim, max_len, window);
}

smoe_status smoe_attend(const smoe_kv* kv, const void* q, int64_t q_ld, int32_t n_tokens, int32_t n_heads,
                        const int32_t* q_start, const int32_t* kv_len, int32_t n_seqs, const int32_t* pages, int64_t pages_ld,
                        int32_t max_pages, int64_t max_len, float scale, int32_t causal, int32_t window, void* out,
                        int64_t out_ld, float* lse, void* workspace, size_t workspace_bytes, void* hip_stream) {
    const smoe_status s = check_attend(kv, n_heads, n_tokens, n_seqs, max_len);
    if (s != SMOE_OK) return s;
    if (max_pages < 0 || max_len > (int64_t)max_pages * kv->page_size)
        return fail(SMOE_EINVAL, "attend: max_len is more than max_pages hold");
    constexpr float kLog2e = 1.44269504f;
    if (!finite(scale * kLog2e)) return fail(SMOE_EINVAL, "attend: scale must be finite, and so must scale times log2 e");
    if (window < 0 || (window && !causal)) return fail(SMOE_EINVAL, "attend: a window must be positive, and causal");
    if (n_tokens == 0 || n_seqs == 0) return ok();
    if (!kv->k || !kv->v || !q || !q_start || !kv_len || !out || (max_len && !pages)) return fail(SMOE_ENULL, "attend: NULL buffer");
    const int64_t n = (int64_t)n_heads * kv->head_dim;
    if (bad_rows(q_ld, n_tokens, 0) || bad_rows(out_ld, n_tokens, n) || bad_rows(pages_ld, n_seqs, 0))
        return fail(SMOE_EINVAL, "attend: row strides must not be negative, and out's rows not overlap");
    if (n_tokens > 1 && q_ld % 8) return fail(SMOE_EINVAL, "attend: q's row stride must be a multiple of 8");
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16) || !aligned(q, 16))
        return fail(SMOE_EALIGN, "attend: q and the cache must be 16-byte aligned");
    if (!aligned(out, 2) || !aligned(lse, 4) || !aligned(q_start, 4) || !aligned(kv_len, 4) || !aligned(pages, 4))
        return fail(SMOE_EALIGN, "attend: a buffer is not aligned to its values");
    const Span in[] = {rows_of(q, kv->type, n_tokens, q_ld, n), pages_of(kv, kv->k), pages_of(kv, kv->v),
                       bytes_of(q_start, 4ll * (n_seqs + 1)), bytes_of(kv_len, 4ll * n_seqs),
                       max_pages ? rows_of(pages, SMOE_F32, n_seqs, pages_ld, max_pages) : bytes_of(nullptr, 1)};
    const size_t need = attend_part_bytes(n_tokens, n_seqs, n_heads, kv->n_kv_heads, kv->head_dim, max_len, window);
    if (need) {
        if (!workspace) return fail(SMOE_ENULL, "attend: the workspace is NULL");
        if (!aligned(workspace, 256)) return fail(SMOE_EALIGN, "attend: the workspace must be 256-byte aligned");
        if (workspace_bytes < need)
            return fail(SMOE_ESIZE, "attend workspace is " + std::to_string(workspace_bytes) + " bytes, needs " + std::to_string(need));
    }
    const Span written[] = {rows_of(out, kv->type, n_tokens, out_ld, n), bytes_of(lse, 4ll * n_tokens * n_heads),
                            bytes_of(need ? workspace : nullptr, (int64_t)need)};
    for (const Span& o : written) {
        for (const Span& i : in)
            if (overlap(o, i)) return fail(SMOE_EINVAL, "attend: an output or the workspace overlaps an input");
        for (const Span& p : written)
            if (&p != &o && overlap(o, p)) return fail(SMOE_EINVAL, "attend: two outputs, or one and the workspace, overlap");
    }
    AttendArgs a{};
    a.k = static_cast<const uint8_t*>(kv->k), a.v = static_cast<const uint8_t*>(kv->v), a.q = q;
    a.q_start = q_start, a.kv_len = kv_len, a.pages = pages;
    a.out = out, a.lse = lse, a.part = static_cast<float*>(workspace);
    a.q_ld = n_tokens > 1 ? q_ld : 0, a.out_ld = n_tokens > 1 ? out_ld : 0, a.pages_ld = n_seqs > 1 ? pages_ld : 0;
    a.n_tokens = n_tokens, a.n_seqs = n_seqs, a.n_heads = n_heads, a.n_kv = kv->n_kv_heads, a.group = n_heads / kv->n_kv_heads;
    a.head_dim = kv->head_dim, a.page_size = kv->page_size, a.n_pages = kv->n_pages, a.max_len = (int)max_len;
    a.causal = causal != 0, a.window = window, a.f16 = kv->type == SMOE_F16;
    a.scale = scale * kLog2e;
    return launched(launch_attend(a, reinterpret_cast<hipStream_t>(hip_stream)), "attend");
}

}  // extern "C"
