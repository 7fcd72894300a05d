"""The operators of a layer's other half, the attention in front of the mixture-of-experts block, over the range a program
calls them in.

A case is one call of one operator:

  append   PagedCache.append   rotary positions for a step's queries and keys, keys and values into a paged cache
  attend   PagedCache.attend   attention of each sequence's new tokens over its pages: a prompt, a chunk, single tokens
  linear4  Linear4.run         a product with 4-bit weights and group scales, with the dense product's epilogue

`own` false computes them from elementary torch operations in 32 bits (angles in 64), true calls the package.  `exact`
evaluates the definitions in 64 bits:

  append   a pair (a, b) of a head's first `rot` values at position p becomes s (a cos pf - b sin pf, b cos pf + a sin pf),
           f_i = base^(-2 i / rot) scaled for long contexts; the pairs lie (i, i + rot / 2) or (2 i, 2 i + 1)
  attend   out = sum_j w_j v_j, w = softmax over the visible keys of scale q k_j; the i-th of n new tokens of a sequence of L
           keys has position p = L - n + i and sees j <= p, and j > p - window where there is one; none: zeros
  linear4  y = act(x W' + b) [* (x W2' + b2)] [+ residual], W[o][i] = scale[i / group][o] (code[o][i] - zero[i / group][o])
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _append(name, tokens, heads, kv, dim, rot, layout="half", scaling="none", base=10000.0, at=0, step=False, page=16, x="bf16",
            t="bf16", pad=False):
    return dict(name=name, op="append", tokens=tokens, heads=heads, kv=kv, dim=dim, rot=rot, layout=layout, scaling=scaling,
                base=base, at=at, step=step, page=page, x=x, t=t, pad=pad)


def _attend(name, seqs, new, ctx, heads, kv, dim, page=16, t="bf16", ragged=False, window=0, causal=True, lse=False):
    return dict(name=name, op="attend", seqs=seqs, new=new, ctx=ctx, heads=heads, kv=kv, dim=dim, page=page, t=t, ragged=ragged,
                window=window, causal=causal, lse=lse)


def _linear4(name, tokens, n_in, n_out, group=128, zeros=False, t="bf16", y="f32", bias=False, pair=False, act="none",
             residual=False):
    return dict(name=name, op="linear4", tokens=tokens, n_in=n_in, n_out=n_out, group=group, zeros=zeros, t=t, y=y, bias=bias,
                pair=pair, act=act, residual=residual)


def listed():
    return [
        # one sequence generates, a quarter of each head turned: the smallest call, latency
        _append("append_1", 1, 16, 2, 256, 64, base=1e7, at=30000, step=True),
        # a serving batch of odd heads far out in long contexts, padded, straight from an f32 product
        _append("append_77_far", 77, 21, 7, 80, 80, layout="pairs", scaling="parts", base=5e5, at=1000000, step=True, page=24,
                x="f32", t="fp16", pad=True),
        # a long prompt
        _append("append_8192", 8192, 32, 8, 128, 128, scaling="ntk", page=64),
        # one sequence generates over a short context: latency
        _attend("attend_step_1", 1, 1, 1000, 16, 2, 256),
        # a serving batch generates, sequences of all lengths, some finished
        _attend("attend_step_64", 64, 1, 8192, 32, 8, 128, page=32, ragged=True),
        # one sequence generates at the end of a very long context; its statistics go to a join with another cache's
        _attend("attend_step_long", 1, 1, 131071, 32, 4, 128, lse=True),
        # chunks of prompts of odd lengths between generating sequences, a sliding window, pages that divide nothing
        _attend("attend_mixed_window", 6, 333, 2000, 14, 2, 64, page=24, t="fp16", ragged=True, window=500),
        # a chunk of a prompt over what is cached of it
        _attend("attend_chunk_1024", 1, 1024, 32768, 32, 8, 128, page=64),
        # a whole prompt at once: the largest call
        _attend("attend_prompt_8192", 1, 8192, 0, 32, 8, 128, page=64),
        # one generated token through gate and up
        _linear4("linear4_gated_1", 1, 2048, 8192, y="bf16", pair=True, act="silu"),
        # a serving batch through the product behind it, back onto the stream
        _linear4("linear4_down_16", 16, 8192, 2048, group=64, zeros=True, residual=True),
        # a prompt, ragged sizes, small groups
        _linear4("linear4_gelu_301", 301, 2560, 5003, group=32, zeros=True, t="fp16", y="fp16", bias=True, act="gelu"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "linear4"])
    if op == "append":
        dim = rng.choice([64, 80, 96, 128, 192, 256])
        kv = rng.choice([1, 2, 3, 4, 8])
        tokens = _log_int(rng, 1, 8192 * 48 * 128 // (dim * kv * 8))
        scaling = rng.choice(["none", "linear", "ntk", "parts"])
        c = _append("", min(tokens, 8192), kv * rng.choice([1, 2, 4, 5]), kv, dim, rng.choice([dim, dim, dim // 2, dim // 4]),
                    layout=rng.choice(["half", "pairs"]), scaling=scaling, base=rng.choice([1e4, 5e5, 1e7]),
                    at=_log_int(rng, 1, 1000000), step=rng.random() < 0.5, page=rng.choice([1, 16, 24, 64, 256]),
                    x=rng.choice(["f32", "bf16", "fp16"]), t=rng.choice(["bf16", "fp16"]), pad=rng.random() < 0.3)
    elif op == "attend":
        dim, kv, group = rng.choice([64, 80, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8, 16])
        group = max(1, min(group, 32 // kv))
        new = 1 if rng.random() < 0.5 else _log_int(rng, 2, 2048)
        seqs = _log_int(rng, 1, 64 if new == 1 else 8)
        top = min(131072, 2 ** 20 // seqs, 2 ** 30 // (seqs * new * kv * group), 2 ** 25 * 16 // (seqs * dim * kv))
        c = _attend("", seqs, new, _log_int(rng, 1, max(1, top)) - 1, kv * group, kv, dim, page=rng.choice([1, 16, 24, 64, 256]),
                    t=rng.choice(["bf16", "fp16"]), ragged=rng.random() < 0.6,
                    window=_log_int(rng, 1, 4096) if rng.random() < 0.25 else 0, causal=True, lse=rng.random() < 0.3)
        if rng.random() < 0.15:
            c.update(causal=False, window=0)
    else:
        n_in, n_out, pair = 32 * _log_int(rng, 2, 256), _log_int(rng, 1, 16384), rng.random() < 0.4
        top = 2 ** 35 // (n_in * n_out * (2 if pair else 1))
        acts = ["silu", "gelu", "relu", "relu2", "sigmoid"]
        c = _linear4("", _log_int(rng, 1, max(1, min(4096, top))), n_in, n_out, group=rng.choice([32, 64, 128, 256, n_in]),
                     zeros=rng.random() < 0.5, t=rng.choice(["bf16", "fp16"]), y=rng.choice(list(TYPES)), bias=rng.random() < 0.3,
                     pair=pair, act=rng.choice(acts if pair else ["none", "none"] + acts), residual=rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs

def _normal(gen, *shape, sigma=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * sigma


def _lengths(case):
    """(new tokens, keys) of each sequence.  Ragged: the first one is the longest, the others spread below it, every
    eighth of a generating batch has finished."""
    n, L = [], []
    for i in range(case["seqs"]):
        new, ctx = case["new"], case["ctx"]
        if case["ragged"] and i:
            new = (0 if i % 8 == 7 else 1) if new == 1 else int(new * (i * 0.6180339887 % 1.0) ** 2)
            ctx = int(ctx * (i * 0.7548776662 % 1.0))
        n.append(new)
        L.append(ctx + new)
    return n, L


def _scaling(case):
    """(kind, factor, trained length, slow, fast): frequencies that turn fewer than `slow` times over the trained length
    are divided by the factor, ones that turn more than `fast` times are kept."""
    return {"none": None, "linear": ("linear", 4.0), "ntk": ("ntk", 8.0), "parts": ("parts", 16.0, 8192, 1.0, 32.0)}[case["scaling"]]


def _inputs(case, seed):
    """The call's tensors, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)
    d = {}
    if case["op"] == "append":
        T, H, kv, D, page = (case[k] for k in ("tokens", "heads", "kv", "dim", "page"))
        # one product's rows, split
        rows = _normal(gen, T, (H + 2 * kv) * D).to(TYPES[case["x"]])
        d["q"], d["k"], d["v"] = (p.unflatten(1, (-1, D)) for p in rows.split([H * D, kv * D, kv * D], dim=1))
        if case["step"]:  # a token of each of many sequences
            d["positions"] = torch.randint(case["at"] // 2, case["at"] + 1, (T,), generator=gen, device="cuda", dtype=torch.int32)
        else:
            d["positions"] = torch.arange(case["at"], case["at"] + T, device="cuda", dtype=torch.int32)
        need = -(-T // page)
        n_pages = need + max(2, need // 4)
        order = torch.randperm(n_pages, generator=gen, device="cuda")
        t = torch.arange(T, device="cuda")
        d["slots"] = order[t // page] * page + t % page
        if case["pad"]:
            d["slots"][T - T // 8:] = -1
        # (a page behind the cache's own, for the plain form's padded tokens)
        for name in ("k_pages", "v_pages"):
            d[name] = _normal(gen, n_pages + 1, kv, page, D).to(TYPES[case["t"]])
    elif case["op"] == "attend":
        H, kv, D, page, t = case["heads"], case["kv"], case["dim"], case["page"], TYPES[case["t"]]
        n, L = _lengths(case)
        T = sum(n)
        need = [-(-l // page) for l in L]
        n_pages = sum(need) + 3
        order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((len(n), max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, m in enumerate(need):
            table[i, :m] = order[at:at + m]
            at += m
        d["pages"] = table
        d["k_pages"] = (_normal(gen, n_pages, kv, page, D) + _normal(gen, kv, 1, D, sigma=0.5)).to(t)
        d["v_pages"] = _normal(gen, n_pages, kv, page, D).to(t)
        # the queries are columns of one product's rows, and lean towards some keys
        d["q"] = (_normal(gen, T, (H + 2 * kv) * D) * 1.5).to(t)[:, :H * D].unflatten(1, (H, D))
        d["q_start"] = torch.tensor([0] + n, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
        d["kv_len"] = torch.tensor(L, dtype=torch.int32).cuda()
    else:
        T, K, N, t = case["tokens"], case["n_in"], case["n_out"], TYPES[case["t"]]
        groups = -(-K // case["group"])
        d["x"] = _normal(gen, T, K).to(t)
        for i in ("", "2") if case["pair"] else ("",):
            codes = (_normal(gen, N, K) * 2.6 + 7.5).round().clamp(0, 15).to(torch.uint8)
            d["w" + i] = codes[:, 0::2] | codes[:, 1::2] << 4
            spread = 0.5 + torch.rand((groups, N), generator=gen, device="cuda")
            d["scales" + i] = (spread * (K ** -0.5 / 2.6)).to(t)
            d["zeros" + i] = None
            if case["zeros"]:
                d["zeros" + i] = torch.randint(5, 11, (groups, N), generator=gen, device="cuda", dtype=torch.uint8)
            d["bias" + i] = _normal(gen, N, sigma=0.2) if case["bias"] else None
        d["residual"] = _normal(gen, T, N).to(TYPES[case["y"]]) if case["residual"] else None
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    if own:
        import stratametal_amd as S
        if case["op"] == "append":
            d["cache"] = S.PagedCache(d["k_pages"][:-1], d["v_pages"][:-1])
            d["rotary"] = S.Rotary(case["dim"], rot_dim=case["rot"], base=case["base"], scaling=_scaling(case),
                                   layout=S.ROPE_PAIRS if case["layout"] == "pairs" else S.ROPE_HALF)
        elif case["op"] == "attend":
            d["cache"] = S.PagedCache(d["k_pages"], d["v_pages"])
        else:
            acts = dict(none=S.ACT_NONE, silu=S.ACT_SILU, gelu=S.ACT_GELU, relu=S.ACT_RELU, relu2=S.ACT_RELU2,
                        sigmoid=S.ACT_SIGMOID)
            d["linear"] = S.Linear4(case["n_in"], case["n_out"], d["w"], d["scales"], zeros=d["zeros"], group=case["group"],
                                    bias=d["bias"], w2=d.get("w2"), scales2=d.get("scales2"), zeros2=d.get("zeros2"),
                                    bias2=d.get("bias2"), act=acts[case["act"]])
    return d


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    if own:
        if case["op"] == "append":
            q = state["cache"].append(state["k"], state["v"], state["slots"], rotary=state["rotary"],
                                      positions=state["positions"], q=state["q"])
            return q, state["k_pages"][:-1], state["v_pages"][:-1]
        if case["op"] == "attend":
            return state["cache"].attend(state["q"], state["q_start"], state["kv_len"], state["pages"], causal=case["causal"],
                                         window=case["window"], lse=case["lse"], max_len=case["ctx"] + case["new"])
        return state["linear"].run(state["x"], residual=state["residual"], y_dtype=TYPES[case["y"]])
    return {"append": _plain_append, "attend": _plain_attend, "linear4": _plain_linear4}[case["op"]](state, case)


def _frequencies(case):
    """f_i in 64 bits, and the factor on turned values."""
    rot, base, s = case["rot"], case["base"], _scaling(case)
    if s is not None and s[0] == "ntk" and rot > 2:
        base = base * s[1] ** (rot / (rot - 2))
    f = torch.pow(torch.tensor(base, dtype=torch.float64, device="cuda"),
                  torch.arange(rot // 2, dtype=torch.float64, device="cuda") * (-2.0 / rot))
    if s is not None and s[0] == "linear":
        return f / s[1], 1.0
    if s is not None and s[0] == "parts":
        _, factor, trained, slow, fast = s
        keep = ((f * (trained / (2.0 * math.pi)) - slow) / (fast - slow)).clamp(0.0, 1.0)
        return f * (keep + (1.0 - keep) / factor), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _turn(x, cos, sin, case):
    half = case["rot"] // 2
    x, rest = x.float().split([case["rot"], case["dim"] - case["rot"]], dim=2)
    if case["layout"] == "pairs":
        a, b = x[..., 0::2], x[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=3).flatten(2)
    else:
        a, b = x[..., :half], x[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=2)
    return torch.cat([turned, rest], dim=2)


def _plain_append(s, case):
    f, factor = _frequencies(case)
    angle = s["positions"].double()[:, None] * f
    cos, sin = (torch.cos(angle) * factor).float()[:, None], (torch.sin(angle) * factor).float()[:, None]
    t, page = TYPES[case["t"]], case["page"]
    slots = torch.where(s["slots"] < 0, (s["k_pages"].shape[0] - 1) * page, s["slots"])
    s["k_pages"][slots // page, :, slots % page] = _turn(s["k"], cos, sin, case).to(t)
    s["v_pages"][slots // page, :, slots % page] = s["v"].to(t)
    return _turn(s["q"], cos, sin, case).to(t), s["k_pages"][:-1], s["v_pages"][:-1]


def _plain_attend(s, case):
    H, kv, D, page, new = case["heads"], case["kv"], case["dim"], case["page"], case["new"]
    B, T, g, L = case["seqs"], s["q"].shape[0], H // kv, case["ctx"] + new
    dev = "cuda"
    j = torch.arange(L, device=dev)
    own_pages = s["pages"][:, j // page].long().clamp(min=0)
    inside = j < s["kv_len"][:, None]
    k = s["k_pages"].transpose(1, 2)[own_pages, j % page].permute(0, 2, 3, 1).float().contiguous()  # [B, kv, D, L]
    v = s["v_pages"].transpose(1, 2)[own_pages, j % page].float()
    v = torch.where(inside[:, :, None, None], v, 0.0).transpose(1, 2).contiguous()  # [B, kv, L, D]
    count = s["q_start"][1:] - s["q_start"][:-1]
    i = torch.arange(new, device=dev)
    row = (s["q_start"][:-1, None] + i).clamp(max=T - 1).long()
    q = s["q"][row].float().unflatten(2, (kv, g)).permute(0, 2, 1, 3, 4).flatten(2, 3).contiguous()  # [B, kv, new g, D]
    score = torch.matmul(q, k).mul_(D ** -0.5).unflatten(2, (new, g))
    position = (s["kv_len"] - count)[:, None] + i
    seen = inside[:, None, :]
    if case["causal"]:
        seen = seen & (j <= position[:, :, None])
        if case["window"]:
            seen = seen & (j > position[:, :, None] - case["window"])
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(dim=4, keepdim=True)
    base = torch.where(top == -math.inf, 0.0, top)
    weight = score.sub_(base).exp_()
    total = weight.sum(dim=4, keepdim=True)
    out = torch.matmul(weight.flatten(2, 3), v).unflatten(2, (new, g)) / torch.where(total == 0.0, 1.0, total)
    token = torch.arange(T, device=dev)
    seq = torch.searchsorted(s["q_start"][1:].contiguous(), token.to(torch.int32), right=True)
    at = token - s["q_start"][seq].long()
    out = out.permute(0, 2, 1, 3, 4)[seq, at].flatten(1, 2).to(TYPES[case["t"]])
    if not case["lse"]:
        return out
    lse = (base + torch.log(total)).squeeze(4)
    return out, lse.permute(0, 2, 1, 3)[seq, at].flatten(1, 2)


def _activate(a, act):
    if act == "silu":
        return a * torch.sigmoid(a)
    if act == "gelu":
        return 0.5 * a * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (a + 0.044715 * a * a * a)))
    if act in ("relu", "relu2"):
        r = torch.clamp(a, min=0.0)
        return r if act == "relu" else r * r
    return torch.sigmoid(a) if act == "sigmoid" else a


def _plain_weights(s, case, i):
    w = s["w" + i]
    codes = torch.stack([w & 15, w >> 4], dim=2).flatten(1).float()
    group = torch.arange(case["n_in"], device="cuda") // case["group"]
    zero = 8.0 if s["zeros" + i] is None else s["zeros" + i].float().t()[:, group]
    return (codes - zero) * s["scales" + i].float().t()[:, group]


def _plain_linear4(s, case):
    x = s["x"].float()
    a = x @ _plain_weights(s, case, "").t()
    if s["bias"] is not None:
        a = a + s["bias"]
    y = _activate(a, case["act"])
    if case["pair"]:
        u = x @ _plain_weights(s, case, "2").t()
        y = y * (u + s["bias2"] if s["bias2"] is not None else u)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(TYPES[case["y"]])


# ------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "append":
        rot, D, page = case["rot"], case["dim"], case["page"]
        freq = []
        for i in range(rot // 2):
            f, s = case["base"] ** (-2.0 * i / rot), _scaling(case)
            if s is not None and s[0] == "linear":
                f /= s[1]
            elif s is not None and s[0] == "ntk":  # the base grows until the slowest pair is slower by the factor
                f *= s[1] ** (-2.0 * i / (rot - 2)) if rot > 2 else 1.0
            elif s is not None:
                turns = f * s[2] / (2.0 * math.pi)
                f = f / s[1] if turns <= s[3] else f if turns >= s[4] else \
                    (f * (turns - s[3]) + f / s[1] * (s[4] - turns)) / (s[4] - s[3])
            freq.append(f)
        scale = 1.0 + 0.1 * math.log(16.0) if case["scaling"] == "parts" else 1.0
        angle = torch.outer(d["positions"].double(), torch.tensor(freq, dtype=torch.float64, device="cuda"))
        # as complex numbers: a + bi times s e^(i angle)
        unit = torch.polar(torch.full_like(angle, scale), angle)[:, None, :]
        first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["layout"] == "pairs" else (slice(0, rot // 2), slice(rot // 2, rot))

        def turned(x):
            x = x.double().clone()
            z = torch.complex(x[..., first], x[..., second]) * unit
            x[..., first], x[..., second] = z.real, z.imag
            return x

        kept = d["slots"] >= 0
        slots = d["slots"][kept]
        pages = []
        for name, value in (("k_pages", turned(d["k"])), ("v_pages", d["v"].double())):
            p = d[name][:-1].double()
            p[slots // page, :, slots % page] = value[kept]
            pages.append(p)
        return turned(d["q"]), pages[0], pages[1]
    if case["op"] == "attend":
        n, L = _lengths(case)
        H, kv, D, page = case["heads"], case["kv"], case["dim"], case["page"]
        g = H // kv
        out = torch.zeros((sum(n), H, D), dtype=torch.float64, device="cuda")
        lse = torch.full((sum(n), H), -math.inf, dtype=torch.float64, device="cuda")
        t0 = 0
        for b in range(case["seqs"]):
            ids = d["pages"][b, :-(-L[b] // page)].long()
            for h in range(kv if n[b] else 0):
                keys = d["k_pages"][ids, h].flatten(0, 1)[:L[b]].double()
                values = d["v_pages"][ids, h].flatten(0, 1)[:L[b]].double()
                q = d["q"][t0:t0 + n[b], h * g:(h + 1) * g].double().transpose(0, 1).reshape(g * n[b], D)
                s = (torch.mm(q, keys.t().contiguous()) / math.sqrt(D)).view(g, n[b], L[b])
                if case["causal"]:
                    ahead = torch.arange(L[b], device="cuda")[None, :] - torch.arange(L[b] - n[b], L[b], device="cuda")[:, None]
                    hidden = ahead > 0
                    if case["window"]:
                        hidden |= ahead <= -case["window"]
                    s.masked_fill_(hidden, -math.inf)
                z = torch.logsumexp(s, 2)
                w = torch.exp(s - z[:, :, None]).view(g * n[b], L[b])
                out[t0:t0 + n[b], h * g:(h + 1) * g] = torch.mm(w, values).view(g, n[b], D).transpose(0, 1)
                lse[t0:t0 + n[b], h * g:(h + 1) * g] = z.t()
            t0 += n[b]
        return (out, lse) if case["lse"] else out
    x = d["x"].double()

    def product(i):
        q = d["w" + i].long()
        codes = torch.empty((case["n_out"], case["n_in"]), dtype=torch.float64, device="cuda")
        codes[:, 0::2], codes[:, 1::2] = (q % 16).double(), (q // 16).double()
        rep = lambda v: v.double().repeat_interleave(case["group"], dim=0)[:case["n_in"]].t()  # noqa: E731
        codes -= 8.0 if d["zeros" + i] is None else rep(d["zeros" + i])
        codes *= rep(d["scales" + i])
        a = torch.mm(x, codes.t().contiguous())
        return a if d["bias" + i] is None else a + d["bias" + i].double()

    a = product("")
    sig = lambda v: 1.0 / (1.0 + torch.exp(-v))  # noqa: E731
    y = {"none": lambda: a, "silu": lambda: a * sig(a), "relu": lambda: a * (a > 0), "relu2": lambda: a * a * (a > 0),
         "sigmoid": lambda: sig(a),
         # 0.5 (1 + tanh u) = 1 / (1 + e^-2u)
         "gelu": lambda: a * sig(2.0 * math.sqrt(2.0 / math.pi) * (a + 0.044715 * a ** 3))}[case["act"]]()
    if case["pair"]:
        y = y * product("2")
    return y if d["residual"] is None else y + d["residual"].double()


# ------------------------------------------------------------------------------------------------ work

def work(case):
    size = {"f32": 4, "bf16": 2, "fp16": 2}
    if case["op"] == "append":
        T = case["tokens"]
        turned = (case["heads"] + case["kv"]) * case["rot"]
        stored = T - (T // 8 if case["pad"] else 0)
        kv = 2 * case["kv"] * case["dim"]
        b = T * case["heads"] * case["dim"] * (size[case["x"]] + size[case["t"]]) + stored * kv * (size[case["x"]] + size[case["t"]])
        return {"bytes": b + 12 * T, "flops": T * (3 * turned + 4 * case["rot"])}
    if case["op"] == "attend":
        n, L = _lengths(case)
        H, kv, D, w = case["heads"], case["kv"], case["dim"], case["window"]
        pairs = keys = 0  # visible (query, key) pairs, and keys that some query sees
        for m, l in zip(n, L):
            if m == 0:
                continue
            if not case["causal"]:
                pairs += m * l
                keys += l
                continue
            first, last = l - m + 1, l  # keys up to the first and the last query's position
            pairs += m * (first + last) // 2
            if w:
                over = lambda p: max(0, p - w) * (max(0, p - w) + 1) // 2  # noqa: E731
                pairs -= over(last) - over(first - 1)
            keys += min(l, m + w - 1) if w else l
        T = sum(n)
        b = 2 * keys * kv * D * 2 + 2 * T * H * D * 2 + (4 * T * H if case["lse"] else 0)
        b += 4 * sum(-(-l // case["page"]) for l in L) + 8 * case["seqs"]
        return {"bytes": b, "flops": 4 * pairs * H * D}
    T, K, N, pairs = case["tokens"], case["n_in"], case["n_out"], 2 if case["pair"] else 1
    groups = -(-K // case["group"])
    weights = N * K // 2 + groups * N * (2 + (1 if case["zeros"] else 0)) + (4 * N if case["bias"] else 0)
    b = 2 * T * K + pairs * weights + T * N * size[case["y"]] * (2 if case["residual"] else 1)
    return {"bytes": b, "flops": 2 * T * K * N * pairs}
