// stratametal_amd/csrc/smoe_dense.cpp - the C ABI of the dense operators round the block (include/smoe.h): argument checks
// and launches of smoe_ends.hip, smoe_linear.hip, smoe_linear4.hip and smoe_balance.hip.  As in smoe_api.cpp every refusal happens before
// the first launch, and a zero count returns before launching.
#include "smoe.h"

#include <hip/hip_runtime.h>

#include <iterator>
#include <string>

#include "smoe_check.hpp"
#include "smoe_launch.hpp"
#include "smoe_rules.hpp"

using namespace smoe;

extern "C" {

// ------------------------------------------------------------------------------------------------ block ends

smoe_status smoe_block_ends(const smoe_ends* e, int32_t n_embd, int32_t n_tokens, const void* R, int32_t r_type,
                            int64_t r_ld, const void* y, int32_t y_type, int64_t y_ld, const float* gate, int64_t gate_ld,
                            int64_t gate_step, void* out, int64_t out_ld, void* x, int32_t x_type, int64_t x_ld,
                            void* hip_stream) {
    if (!e) return fail(SMOE_ENULL, "block_ends: the ends are NULL");
    if (n_embd < 1 || n_embd > smoe::kEndsMaxRow)
        return fail(SMOE_EINVAL, "block_ends: rows of 1 to " + std::to_string(smoe::kEndsMaxRow) + " values");
    if (n_tokens < 0) return fail(SMOE_EINVAL, "block_ends: negative token count");
    if (!(e->eps >= 0.0f) || !finite(e->eps)) return fail(SMOE_EINVAL, "block_ends: eps must be finite and non-negative");
    if (!finite(e->res_scale) || !finite(e->y_scale)) return fail(SMOE_EINVAL, "block_ends: the scales must be finite");
    if (e->gate_act != SMOE_GATE_NONE && e->gate_act != SMOE_GATE_SIGMOID)
        return fail(SMOE_EINVAL, "block_ends: gate_act is SMOE_GATE_NONE or SMOE_GATE_SIGMOID");
    if (!elem_type(r_type) || (y && !elem_type(y_type)) || (x && !elem_type(x_type)))
        return fail(SMOE_ETYPE, "block_ends: rows are SMOE_F32, SMOE_F16 or SMOE_BF16");
    if (n_tokens == 0) return ok();
    if (!R) return fail(SMOE_ENULL, "block_ends: R is NULL");
    if (!y != !out) return fail(SMOE_ENULL, "block_ends: y and out go together");
    if (!out && !x) return fail(SMOE_ENULL, "block_ends: nothing to write");
    if (gate && !y) return fail(SMOE_EINVAL, "block_ends: a gate without y");
    if (bad_ld(r_ld, n_tokens, 0) || (y && bad_ld(y_ld, n_tokens, 0)) || (gate && bad_ld(gate_ld, n_tokens, 0)) ||
        (out && bad_ld(out_ld, n_tokens, n_embd)) || (x && bad_ld(x_ld, n_tokens, n_embd)))
        return fail(SMOE_EINVAL, "block_ends: row strides must not be negative, and an output's rows not overlap");
    if (gate && (gate_step < 0 || gate_step > kMaxLd / smoe::kEndsMaxRow))
        return fail(SMOE_EINVAL, "block_ends: the gate's steps must not be negative");
    if (!aligned(R, elem_size(r_type)) || !aligned(out, elem_size(r_type)) || (y && !aligned(y, elem_size(y_type))) ||
        (x && !aligned(x, elem_size(x_type))) || !aligned(gate, 4) || !aligned(e->pre, 4) || !aligned(e->post, 4))
        return fail(SMOE_EALIGN, "block_ends: a buffer is not aligned to its values");
    const Span sr = rows_of(R, r_type, n_tokens, r_ld, n_embd), sy = rows_of(y, y_type, n_tokens, y_ld, n_embd),
               so = rows_of(out, r_type, n_tokens, out_ld, n_embd), sx = rows_of(x, x_type, n_tokens, x_ld, n_embd),
               sg = rows_of(gate, SMOE_F32, n_tokens, gate_ld, gate ? (n_embd - 1) * gate_step + 1 : 1),
               sp = rows_of(e->pre, SMOE_F32, 1, 0, n_embd), sq = rows_of(e->post, SMOE_F32, 1, 0, n_embd);
    for (const Span& o : {so, sx}) {
        for (const Span& in : {sr, sy})
            if (overlap(o, in) && !same(o, in))
                return fail(SMOE_EINVAL, "block_ends: out and x are an input's own rows or share none with it");
        if (overlap(o, sg) || overlap(o, sp) || overlap(o, sq))
            return fail(SMOE_EINVAL, "block_ends: an output overlaps the gate or a norm's weight");
    }
    if (overlap(so, sx)) return fail(SMOE_EINVAL, "block_ends: out and x overlap");
    smoe::EndsArgs a{};
    a.R = R, a.y = y, a.out = out, a.x = x;
    a.gate = gate, a.post = y ? e->post : nullptr, a.pre = x ? e->pre : nullptr;
    a.r_ld = r_ld, a.y_ld = y ? y_ld : 0, a.out_ld = out ? out_ld : 0, a.x_ld = x ? x_ld : 0;
    a.gate_ld = gate_ld, a.gate_step = gate_step;
    if (n_tokens == 1) a.r_ld = a.y_ld = a.out_ld = a.x_ld = a.gate_ld = 0;
    a.r_type = r_type, a.y_type = y ? y_type : SMOE_F32, a.x_type = x ? x_type : SMOE_F32;
    a.gate_sigmoid = e->gate_act == SMOE_GATE_SIGMOID;
    a.n = n_embd, a.n_tokens = n_tokens;
    a.eps = e->eps, a.res_scale = e->res_scale, a.y_scale = e->y_scale;
    return launched(smoe::launch_block_ends(a, reinterpret_cast<hipStream_t>(hip_stream)), "block_ends");
}

// ------------------------------------------------------------------------------------------------ dense product

static smoe_status check_linear(const smoe_linear* L) {
    if (!L) return fail(SMOE_ENULL, "linear: the layer is NULL");
    if (L->n_in < 8 || L->n_in % 8 || L->n_in > smoe::kLinearMaxIn)
        return fail(SMOE_EINVAL, "linear: n_in must be a multiple of 8, at most " + std::to_string(smoe::kLinearMaxIn));
    if (L->n_out < 1 || L->n_out > smoe::kLinearMaxOut)
        return fail(SMOE_EINVAL, "linear: n_out must be 1 to " + std::to_string(smoe::kLinearMaxOut));
    if (L->w_type != SMOE_BF16 && L->w_type != SMOE_F16) return fail(SMOE_ETYPE, "linear: weights are SMOE_BF16 or SMOE_F16");
    if (L->act < SMOE_ACT_NONE || L->act > SMOE_ACT_SIGMOID) return fail(SMOE_EINVAL, "linear: unknown activation");
    return SMOE_OK;
}

size_t smoe_linear_workspace_bytes(const smoe_linear* L, int32_t n_tokens) {
    if (check_linear(L) != SMOE_OK) return 0;
    if (n_tokens < 0) {
        fail(SMOE_EINVAL, "linear: negative token count");
        return 0;
    }
    ok();
    return 256 + (n_tokens ? smoe::linear_part_bytes(n_tokens, L->n_in, L->n_out, L->w2 != nullptr) : 0);
}

smoe_status smoe_linear_run(const smoe_linear* L, const void* x, int64_t x_ld, int32_t n_tokens, const void* residual,
                            int64_t r_ld, void* y, int32_t y_type, int64_t y_ld, void* workspace, size_t workspace_bytes,
                            void* hip_stream) {
    const smoe_status s = check_linear(L);
    if (s != SMOE_OK) return s;
    if (n_tokens < 0) return fail(SMOE_EINVAL, "linear: negative token count");
    if (!elem_type(y_type)) return fail(SMOE_ETYPE, "linear: y is SMOE_F32, SMOE_F16 or SMOE_BF16");
    if (n_tokens == 0) return ok();
    if (!x || !y || !L->w) return fail(SMOE_ENULL, "linear: NULL buffer");
    if (L->bias2 && !L->w2) return fail(SMOE_ENULL, "linear: bias2 without w2");
    if (bad_ld(x_ld, n_tokens, 0) || (residual && bad_ld(r_ld, n_tokens, 0)) || bad_ld(y_ld, n_tokens, L->n_out))
        return fail(SMOE_EINVAL, "linear: row strides must not be negative, and y's rows not overlap");
    if (n_tokens > 1 && (x_ld % 8 || x_ld > smoe::kLinearMaxLd))
        return fail(SMOE_EINVAL, "linear: x's row stride must be a multiple of 8, at most " + std::to_string(smoe::kLinearMaxLd));
    if (!aligned(x, 16) || !aligned(L->w, 16) || !aligned(L->w2, 16))
        return fail(SMOE_EALIGN, "linear: x, w and w2 must be 16-byte aligned");
    if (!aligned(y, elem_size(y_type)) || !aligned(residual, elem_size(y_type)) || !aligned(L->bias, 4) ||
        !aligned(L->bias2, 4))
        return fail(SMOE_EALIGN, "linear: a buffer is not aligned to its values");
    const Span sy = rows_of(y, y_type, n_tokens, y_ld, L->n_out);
    const Span sr = rows_of(residual, y_type, n_tokens, r_ld, L->n_out);
    const int64_t wb = (int64_t)L->n_out * L->n_in;
    if (overlap(sy, sr) && !same(sy, sr)) return fail(SMOE_EINVAL, "linear: y is residual's own rows or shares none with it");
    const Span in[] = {rows_of(x, L->w_type, n_tokens, x_ld, L->n_in), rows_of(L->w, L->w_type, 1, 0, wb),
                       rows_of(L->w2, L->w_type, 1, 0, wb), rows_of(L->bias, SMOE_F32, 1, 0, L->n_out),
                       rows_of(L->bias2, SMOE_F32, 1, 0, L->n_out)};
    for (const Span& i : in)
        if (overlap(sy, i)) return fail(SMOE_EINVAL, "linear: y overlaps x, a weight or a bias");
    const smoe::LinearPlan plan = smoe::linear_plan(n_tokens, L->n_in, L->n_out, L->w2 != nullptr);
    if (smoe::linear_groups(plan, n_tokens, L->n_out, L->w2 != nullptr) >= smoe::kGridGroups)
        return fail(SMOE_EINVAL, "linear: the product exceeds a launch's grid: split it");
    const size_t need = smoe::linear_part_bytes(n_tokens, L->n_in, L->n_out, L->w2 != nullptr);
    if (need) {
        if (!workspace) return fail(SMOE_ENULL, "linear: the workspace is NULL");
        if (!aligned(workspace, 256)) return fail(SMOE_EALIGN, "linear: the workspace must be 256-byte aligned");
        if (workspace_bytes < need)
            return fail(SMOE_ESIZE, "linear workspace is " + std::to_string(workspace_bytes) + " bytes, needs " +
                                        std::to_string(need));
        const Span ws = bytes_of(workspace, (int64_t)need);
        bool shared = overlap(ws, sy) || overlap(ws, sr);
        for (const Span& i : in) shared = shared || overlap(ws, i);
        if (shared) return fail(SMOE_EINVAL, "linear: the workspace overlaps y, residual, x, a weight or a bias");
    }
    smoe::LinearArgs a{};
    a.x = x, a.w = L->w, a.w2 = L->w2, a.residual = residual, a.bias = L->bias, a.bias2 = L->bias2, a.y = y;
    a.part = static_cast<float*>(workspace);
    a.x_ld = n_tokens > 1 ? x_ld : 0, a.r_ld = n_tokens > 1 && residual ? r_ld : 0, a.y_ld = n_tokens > 1 ? y_ld : 0;
    a.n_in = L->n_in, a.n_out = L->n_out, a.n_tokens = n_tokens;
    a.w_type = L->w_type, a.y_type = y_type, a.act = L->act;
    return launched(smoe::launch_linear(a, reinterpret_cast<hipStream_t>(hip_stream)), "linear");
}

// ------------------------------------------------------------------------------------------------ 4-bit weights

static smoe_status check_linear4(const smoe_linear4* L) {
    if (!L) return fail(SMOE_ENULL, "linear4: the layer is NULL");
    if (L->n_in < 32 || L->n_in % 32 || L->n_in > smoe::kLinearMaxIn)
        return fail(SMOE_EINVAL, "linear4: n_in must be a multiple of 32, at most " + std::to_string(smoe::kLinearMaxIn));
    if (L->n_out < 1 || L->n_out > smoe::kLinearMaxOut)
        return fail(SMOE_EINVAL, "linear4: n_out must be 1 to " + std::to_string(smoe::kLinearMaxOut));
    if (L->x_type != SMOE_BF16 && L->x_type != SMOE_F16) return fail(SMOE_ETYPE, "linear4: x is SMOE_BF16 or SMOE_F16");
    if (!elem_type(L->s_type)) return fail(SMOE_ETYPE, "linear4: scales are SMOE_F32, SMOE_F16 or SMOE_BF16");
    if (L->group < 32 || L->group % 32) return fail(SMOE_EINVAL, "linear4: group must be a multiple of 32");
    if (L->act < SMOE_ACT_NONE || L->act > SMOE_ACT_SIGMOID) return fail(SMOE_EINVAL, "linear4: unknown activation");
    return SMOE_OK;
}

size_t smoe_linear4_workspace_bytes(const smoe_linear4* L, int32_t n_tokens) {
    if (check_linear4(L) != SMOE_OK) return 0;
    if (n_tokens < 0) {
        fail(SMOE_EINVAL, "linear4: negative token count");
        return 0;
    }
    ok();
    return 256 + (n_tokens ? smoe::linear4_part_bytes(n_tokens, L->n_in, L->n_out, L->w2 != nullptr, L->group) : 0);
}

smoe_status smoe_linear4_run(const smoe_linear4* L, const void* x, int64_t x_ld, int32_t n_tokens, const void* residual,
                             int64_t r_ld, void* y, int32_t y_type, int64_t y_ld, void* workspace, size_t workspace_bytes,
                             void* hip_stream) {
    const smoe_status s = check_linear4(L);
    if (s != SMOE_OK) return s;
    if (n_tokens < 0) return fail(SMOE_EINVAL, "linear4: negative token count");
    if (!elem_type(y_type)) return fail(SMOE_ETYPE, "linear4: y is SMOE_F32, SMOE_F16 or SMOE_BF16");
    if (n_tokens == 0) return ok();
    if (!x || !y || !L->w || !L->scales || (L->w2 && !L->scales2)) return fail(SMOE_ENULL, "linear4: NULL buffer");
    if ((L->bias2 || L->scales2 || L->zeros2) && !L->w2) return fail(SMOE_ENULL, "linear4: bias2, scales2 or zeros2 without w2");
    if (bad_ld(x_ld, n_tokens, 0) || (residual && bad_ld(r_ld, n_tokens, 0)) || bad_ld(y_ld, n_tokens, L->n_out))
        return fail(SMOE_EINVAL, "linear4: row strides must not be negative, and y's rows not overlap");
    if (n_tokens > 1 && (x_ld % 8 || x_ld > smoe::kLinearMaxLd))
        return fail(SMOE_EINVAL, "linear4: x's row stride must be a multiple of 8, at most " + std::to_string(smoe::kLinearMaxLd));
    if (!aligned(x, 16) || !aligned(L->w, 16) || !aligned(L->w2, 16))
        return fail(SMOE_EALIGN, "linear4: x, w and w2 must be 16-byte aligned");
    if (!aligned(y, elem_size(y_type)) || !aligned(residual, elem_size(y_type)) || !aligned(L->bias, 4) || !aligned(L->bias2, 4) ||
        !aligned(L->scales, elem_size(L->s_type)) || !aligned(L->scales2, elem_size(L->s_type)))
        return fail(SMOE_EALIGN, "linear4: a buffer is not aligned to its values");
    const int64_t codes = (int64_t)L->n_out * (L->n_in / 2), groups = (L->n_in + (int64_t)L->group - 1) / L->group * L->n_out;
    const Span sy = rows_of(y, y_type, n_tokens, y_ld, L->n_out), sr = rows_of(residual, y_type, n_tokens, r_ld, L->n_out);
    if (overlap(sy, sr) && !same(sy, sr)) return fail(SMOE_EINVAL, "linear4: y is residual's own rows or shares none with it");
    const Span in[] = {rows_of(x, L->x_type, n_tokens, x_ld, L->n_in), bytes_of(L->w, codes), bytes_of(L->w2, codes),
                       rows_of(L->scales, L->s_type, 1, 0, groups), rows_of(L->scales2, L->s_type, 1, 0, groups),
                       bytes_of(L->zeros, groups), bytes_of(L->zeros2, groups), rows_of(L->bias, SMOE_F32, 1, 0, L->n_out),
                       rows_of(L->bias2, SMOE_F32, 1, 0, L->n_out)};
    for (const Span& i : in)
        if (overlap(sy, i)) return fail(SMOE_EINVAL, "linear4: y overlaps x, a weight, a scale, a zero or a bias");
    if (!smoe::linear4_fits(n_tokens, L->n_in, L->n_out, L->w2 != nullptr, L->group))
        return fail(SMOE_EINVAL, "linear4: the product exceeds a launch's grid: split it");
    const size_t need = smoe::linear4_part_bytes(n_tokens, L->n_in, L->n_out, L->w2 != nullptr, L->group);
    if (need) {
        if (!workspace) return fail(SMOE_ENULL, "linear4: the workspace is NULL");
        if (!aligned(workspace, 256)) return fail(SMOE_EALIGN, "linear4: the workspace must be 256-byte aligned");
        if (workspace_bytes < need)
            return fail(SMOE_ESIZE, "linear4 workspace is " + std::to_string(workspace_bytes) + " bytes, needs " +
                                        std::to_string(need));
        const Span ws = bytes_of(workspace, (int64_t)need);
        bool shared = overlap(ws, sy) || overlap(ws, sr);
        for (const Span& i : in) shared = shared || overlap(ws, i);
        if (shared) return fail(SMOE_EINVAL, "linear4: the workspace overlaps an operand");
    }
    smoe::Linear4Args a{};
    a.x = x, a.w = L->w, a.w2 = L->w2, a.residual = residual, a.bias = L->bias, a.bias2 = L->bias2, a.y = y;
    a.part = static_cast<float*>(workspace);
    a.x_ld = n_tokens > 1 ? x_ld : 0, a.r_ld = n_tokens > 1 && residual ? r_ld : 0, a.y_ld = n_tokens > 1 ? y_ld : 0;
    a.n_in = L->n_in, a.n_out = L->n_out, a.n_tokens = n_tokens;
    a.w_type = L->x_type, a.y_type = y_type, a.act = L->act;
    a.scales = L->scales, a.scales2 = L->scales2, a.zeros = L->zeros, a.zeros2 = L->zeros2;
    a.group = smoe::linear4_group(L->group), a.s_type = L->s_type;
    return launched(smoe::launch_linear4(a, reinterpret_cast<hipStream_t>(hip_stream)), "linear4");
}

// ------------------------------------------------------------------------------------------------ router balance

static smoe_status check_balance(int32_t n_tokens, int32_t n_expert, int32_t k) {
    if (n_tokens < 0) return fail(SMOE_EINVAL, "router_balance: negative token count");
    if (n_expert < 1 || n_expert > 1024) return fail(SMOE_EINVAL, "router_balance: n_expert must be 1 to 1024");
    if (k < 1 || k > 64 || k > n_expert) return fail(SMOE_EINVAL, "router_balance: k must be 1 to 64, at most n_expert");
    if ((int64_t)n_tokens * k > (1 << 24)) return fail(SMOE_EINVAL, "router_balance: more than 2^24 pairs");
    return SMOE_OK;
}

size_t smoe_router_balance_workspace_bytes(int32_t max_tokens, int32_t n_expert) {
    if (check_balance(max_tokens, n_expert, 1) != SMOE_OK) return 0;
    ok();
    return smoe::balance_work_bytes(max_tokens, n_expert);
}

smoe_status smoe_router_balance(const float* logits, int64_t logits_ld, const int32_t* ids, const uint8_t* mask,
                                int32_t n_tokens, int32_t n_expert, int32_t k, float balance_coef, float z_coef, float* loss,
                                int32_t* counts, float* mean_p, float* dlogits, int64_t dlogits_ld, float* dbias,
                                void* workspace, size_t workspace_bytes, void* hip_stream) {
    const smoe_status s = check_balance(n_tokens, n_expert, k);
    if (s != SMOE_OK) return s;
    if (!finite(balance_coef) || !finite(z_coef)) return fail(SMOE_EINVAL, "router_balance: the coefficients must be finite");
    if (n_tokens == 0) return ok();
    if (!logits || !ids || !loss || !counts || !mean_p || !workspace) return fail(SMOE_ENULL, "router_balance: NULL buffer");
    if (dbias && !dlogits) return fail(SMOE_ENULL, "router_balance: dbias without dlogits");
    if ((logits_ld != 0 && bad_ld(logits_ld, n_tokens, n_expert)) || (dlogits && bad_ld(dlogits_ld, n_tokens, n_expert)))
        return fail(SMOE_EINVAL, "router_balance: rows overlap");
    for (const void* p : {(const void*)logits, (const void*)ids, (const void*)loss, (const void*)counts, (const void*)mean_p,
                          (const void*)dlogits, (const void*)dbias})
        if (!aligned(p, 4)) return fail(SMOE_EALIGN, "router_balance: buffers must be 4-byte aligned");
    if (!aligned(workspace, 256)) return fail(SMOE_EALIGN, "router_balance: the workspace must be 256-byte aligned");
    const size_t need = smoe::balance_work_bytes(n_tokens, n_expert);
    if (workspace_bytes < need)
        return fail(SMOE_ESIZE, "router_balance workspace is " + std::to_string(workspace_bytes) + " bytes, needs " +
                                    std::to_string(need));
    // (one work-group writes while others still read, and the ids and the mask are read by every launch)
    const Span sl = rows_of(logits, SMOE_F32, n_tokens, logits_ld, n_expert),
               sd = rows_of(dlogits, SMOE_F32, n_tokens, dlogits_ld, n_expert), ws = bytes_of(workspace, (int64_t)need);
    const Span in[] = {sl, bytes_of(ids, (int64_t)n_tokens * k * 4), bytes_of(mask, n_tokens)};
    const Span out[] = {sd, bytes_of(loss, 16), bytes_of(counts, 4 * n_expert), bytes_of(mean_p, 4 * n_expert),
                        bytes_of(dbias, 4 * n_expert), ws};
    if (overlap(sd, sl) && !same(sd, sl))
        return fail(SMOE_EINVAL, "router_balance: dlogits overlaps logits and is not their own rows");
    for (const Span& o : out) {
        for (const Span& i : in)
            if (!(&o == &out[0] && &i == &in[0]) && overlap(o, i))
                return fail(SMOE_EINVAL, "router_balance: an output or the workspace overlaps logits, ids or mask");
        for (const Span* q = &o + 1; q < std::end(out); ++q)
            if (overlap(o, *q))
                return fail(SMOE_EINVAL, "router_balance: two outputs, or one and the workspace, overlap");
    }
    smoe::BalanceArgs a{};
    a.logits = logits, a.ids = ids, a.mask = mask;
    a.loss = loss, a.mean_p = mean_p, a.dlogits = dlogits, a.dbias = dbias, a.counts = counts;
    a.ld = n_tokens > 1 ? logits_ld : 0, a.ld_d = n_tokens > 1 ? dlogits_ld : 0;
    a.n_tokens = n_tokens, a.n_expert = n_expert, a.k = k;
    a.balance_coef = balance_coef, a.z_coef = z_coef;
    a.work = workspace;
    return launched(smoe::launch_balance(a, reinterpret_cast<hipStream_t>(hip_stream)), "router_balance");
}

}  // extern "C"
