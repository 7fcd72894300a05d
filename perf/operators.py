"""The dense operators round the mixture-of-experts block, over the range a program calls them in.

A case is one call of one operator:

  ends     BlockEnds.read / write / join   one residual stream's norms before and after a block, with gate and scales
  linear   Linear.run                      a dense product with bias, activation (gated or not) and residual
  balance  router_balance                  the router's load: counts, balance and z loss, gradients

`own` false computes them from elementary torch operations in 32 bits, true calls the package.  `exact` evaluates the
definitions in 64 bits:

  ends     out = res_scale R + y_scale g z, z = y or y / sqrt(mean y^2 + eps) * post, g = 1, gate or sigmoid(gate);
           x = out / sqrt(mean out^2 + eps) * pre
  linear   y = act(x W' + b) [* (x W2' + b2)] [+ residual]
  balance  p = softmax(logits), f = counts / (n k), P = mean p over the n tokens of the mask:
           cb E sum f P + cz mean lse^2, its gradient to the logits (the counts are constants) and to a bias added to them
"""
import math

import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _ends(name, tokens, n, mode="join", r="f32", y="f32", x="bf16", post=True, pre=True, gate="channel", act="none",
          res_scale=1.0, y_scale=1.0):
    return dict(name=name, op="ends", tokens=tokens, n=n, mode=mode, r=r, y=y, x=x, post=post, pre=pre, gate=gate, act=act,
                res_scale=res_scale, y_scale=y_scale)


def _linear(name, tokens, n_in, n_out, w="bf16", y="f32", bias=True, pair=False, act="none", residual=False):
    return dict(name=name, op="linear", tokens=tokens, n_in=n_in, n_out=n_out, w=w, y=y, bias=bias, pair=pair, act=act,
                residual=residual)


def _balance(name, tokens, experts, k, mask=1.0, grad=True, cb=0.01, cz=0.001):
    return dict(name=name, op="balance", tokens=tokens, experts=experts, k=k, mask=mask, grad=grad, cb=cb, cz=cz)


def listed():
    return [
        # between two blocks while one sequence generates: the smallest call, latency
        _ends("ends_join_1", 1, 2048),
        # a serving batch of odd rows kept in fp16, a gate per token, nothing aligned
        _ends("ends_write_77_odd", 77, 2061, mode="write", r="fp16", y="fp16", gate="token", act="sigmoid"),
        # an ordinary prompt into the block: the norm before it
        _ends("ends_read_512", 512, 2560, mode="read", x="f32"),
        # a long prompt between two blocks, the stream in f32, no gate, scaled residual
        _ends("ends_join_8192", 8192, 4096, y="bf16", gate="none", res_scale=0.5, y_scale=0.25),
        # one generated token through a dense layer's gate and up product
        _linear("linear_gated_1", 1, 2048, 8192, y="bf16", bias=False, pair=True, act="silu"),
        # a serving batch through the product behind it, back onto the stream
        _linear("linear_down_16", 16, 8192, 2048, bias=False, residual=True),
        # a short odd prompt, ragged sizes in fp16
        _linear("linear_gelu_301", 301, 2568, 5003, w="fp16", y="fp16", act="gelu"),
        # a long prompt through gate and up
        _linear("linear_gated_4096", 4096, 2048, 8192, y="bf16", bias=False, pair=True, act="silu"),
        # the largest product: a wide layer on a long prompt, back onto the stream
        _linear("linear_wide_4096", 4096, 8192, 8192, residual=True),
        # a serving batch's load, no gradients
        _balance("balance_64", 64, 512, 10, grad=False),
        # tuning the router on a padded batch
        _balance("balance_grad_4096", 4096, 512, 10, mask=0.9),
        # the largest router and batch
        _balance("balance_grad_32768", 32768, 1024, 8),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ends", "linear", "linear", "balance"])
    t3 = list(TYPES)
    if op == "ends":
        n = _log_int(rng, 16, 8192)
        if rng.random() < 0.6:
            n = max(8, n // 8 * 8)
        tokens = _log_int(rng, 1, max(1, min(16384, 8192 * 4096 // n)))
        c = _ends("", tokens, n, mode=rng.choice(["read", "write", "join", "join"]), r=rng.choice(t3), y=rng.choice(t3),
                  x=rng.choice(t3), post=rng.random() < 0.7, pre=rng.random() < 0.8,
                  gate=rng.choice(["none", "channel", "token", "both"]), act=rng.choice(["none", "sigmoid"]),
                  res_scale=rng.choice([1.0, 0.5]), y_scale=rng.choice([1.0, 0.25]))
    elif op == "linear":
        n_in = _log_int(rng, 2, 1024) * 8
        n_out = _log_int(rng, 1, 16384)
        pair = rng.random() < 0.4
        top = 4096 * 8192 * 8192 // (n_in * n_out * (2 if pair else 1))
        tokens = _log_int(rng, 1, max(1, min(4096, top)))
        act = rng.choice(["silu", "gelu", "relu", "relu2", "sigmoid"] if pair else ["none", "none", "silu", "gelu", "relu", "relu2",
                                                                                  "sigmoid"])
        c = _linear("", tokens, n_in, n_out, w=rng.choice(["bf16", "bf16", "fp16"]), y=rng.choice(t3),
                    bias=rng.random() < 0.5, pair=pair, act=act, residual=rng.random() < 0.5)
    else:
        experts = _log_int(rng, 2, 1024)
        c = _balance("", _log_int(rng, 1, 32768), experts, rng.randint(1, min(experts, 16)), mask=rng.choice([1.0, 0.9, 0.3]),
                     grad=rng.random() < 0.7, cb=rng.choice([0.01, 1.0]), cz=rng.choice([0.0, 0.001]))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs

def _normal(gen, *shape, sigma=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * sigma


def _inputs(case, seed):
    """The call's tensors, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)
    T = case["tokens"]
    d = {}
    if case["op"] == "ends":
        n = case["n"]
        # a residual stream: some channels far larger than the rest
        d["R"] = (_normal(gen, T, n) * (1.0 + 8.0 * (_normal(gen, n) > 2.5).float())).to(TYPES[case["r"]])
        d["pre"] = 1.0 + _normal(gen, n, sigma=0.2) if case["pre"] else None
        d["post"] = 1.0 + _normal(gen, n, sigma=0.2) if case["post"] else None
        if case["mode"] != "read":
            d["y"] = _normal(gen, T, n, sigma=0.3).to(TYPES[case["y"]])
            shape = dict(none=None, channel=(n,), token=(T, 1), both=(T, n))[case["gate"]]
            d["gate"] = None if shape is None else _normal(gen, *shape)
    elif case["op"] == "linear":
        K, N, t = case["n_in"], case["n_out"], TYPES[case["w"]]
        d["x"] = _normal(gen, T, K).to(t)
        for i in ("", "2") if case["pair"] else ("",):
            d["w" + i] = _normal(gen, N, K, sigma=K ** -0.5).to(t)
            d["bias" + i] = _normal(gen, N, sigma=0.2) if case["bias"] else None
        d["residual"] = _normal(gen, T, N).to(TYPES[case["y"]]) if case["residual"] else None
    else:
        E, k = case["experts"], case["k"]
        # popular and unpopular experts
        d["logits"] = _normal(gen, T, E) + _normal(gen, E)
        d["ids"] = torch.topk(d["logits"], k, dim=1).indices.to(torch.int32)
        d["mask"] = torch.rand(T, generator=gen, device="cuda") < case["mask"] if case["mask"] < 1.0 else None
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    if own:
        import stratametal_amd as S
        if case["op"] == "ends":
            d["ends"] = S.BlockEnds(case["n"], pre=d["pre"], post=d["post"], res_scale=case["res_scale"],
                                    y_scale=case["y_scale"], eps=EPS,
                                    gate_act=S.GATE_SIGMOID if case["act"] == "sigmoid" else S.GATE_NONE)
        elif case["op"] == "linear":
            acts = dict(none=S.ACT_NONE, silu=S.ACT_SILU, gelu=S.ACT_GELU, relu=S.ACT_RELU, relu2=S.ACT_RELU2,
                        sigmoid=S.ACT_SIGMOID)
            d["linear"] = S.Linear(case["n_in"], case["n_out"], d["w"], bias=d["bias"], w2=d.get("w2"),
                                   bias2=d.get("bias2"), act=acts[case["act"]])
        else:
            d["balance"] = S.router_balance
    return d


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    if own:
        if case["op"] == "ends":
            if case["mode"] == "read":
                return state["ends"].read(state["R"], x_dtype=TYPES[case["x"]])
            if case["mode"] == "write":
                return state["ends"].write(state["R"], state["y"], gate=state["gate"])
            return state["ends"].join(state["R"], state["y"], gate=state["gate"], x_dtype=TYPES[case["x"]])
        if case["op"] == "linear":
            return state["linear"].run(state["x"], residual=state["residual"], y_dtype=TYPES[case["y"]])
        return state["balance"](state["logits"], state["ids"], mask=state["mask"], balance_coef=case["cb"], z_coef=case["cz"],
                                grad=case["grad"])
    return {"ends": _plain_ends, "linear": _plain_linear, "balance": _plain_balance}[case["op"]](state, case)


def _plain_ends(s, case):
    out = s["R"].float()
    if case["mode"] != "read":
        z = s["y"].float()
        if s["post"] is not None:
            z = z * torch.rsqrt((z * z).mean(1, keepdim=True) + EPS) * s["post"]
        if s["gate"] is not None:
            z = z * (torch.sigmoid(s["gate"]) if case["act"] == "sigmoid" else s["gate"])
        out = case["res_scale"] * out + case["y_scale"] * z
    if case["mode"] == "write":
        return out.to(TYPES[case["r"]])
    x = out * torch.rsqrt((out * out).mean(1, keepdim=True) + EPS)
    if s["pre"] is not None:
        x = x * s["pre"]
    x = x.to(TYPES[case["x"]])
    return x if case["mode"] == "read" else (out.to(TYPES[case["r"]]), x)


def _activate(a, act):
    if act == "silu":
        return a * torch.sigmoid(a)
    if act == "gelu":
        return 0.5 * a * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (a + 0.044715 * a * a * a)))
    if act in ("relu", "relu2"):
        r = torch.clamp(a, min=0.0)
        return r if act == "relu" else r * r
    return torch.sigmoid(a) if act == "sigmoid" else a


def _plain_linear(s, case):
    x = s["x"].float()
    a = x @ s["w"].float().t()
    if s["bias"] is not None:
        a = a + s["bias"]
    y = _activate(a, case["act"])
    if case["pair"]:
        u = x @ s["w2"].float().t()
        y = y * (u + s["bias2"] if s["bias2"] is not None else u)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(TYPES[case["y"]])


def _plain_balance(s, case):
    logits, ids, mask = s["logits"], s["ids"], s["mask"]
    T, E = logits.shape
    k, cb, cz = case["k"], case["cb"], case["cz"]
    m = torch.ones(T, dtype=torch.float32, device="cuda") if mask is None else mask.float()
    counts = torch.zeros(E, dtype=torch.float32, device="cuda")
    counts.index_add_(0, ids.reshape(-1).long(), m.repeat_interleave(k))
    top = logits.max(1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    p = e / total
    lse = (top + torch.log(total)).squeeze(1)
    n = m.sum()
    nn = torch.clamp(n, min=1.0)
    f = counts / (nn * k)
    P = (p * m[:, None]).sum(0) / nn
    balance = E * (f * P).sum()
    z = (lse * lse * m).sum() / nn
    loss = torch.stack([cb * balance + cz * z, balance, z, n])
    out = dict(loss=loss, counts=counts.to(torch.int32), mean_p=P)
    if case["grad"]:
        c = (p * f).sum(1, keepdim=True)
        g = p * (cb * E * (f - c) + 2.0 * cz * lse[:, None]) * (m[:, None] / nn)
        out.update(dlogits=g, dbias=g.sum(0))
    return out


# ------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "ends":
        new = d["R"].double()
        if case["mode"] != "read":
            branch = d["y"].double()
            if case["post"]:
                branch = branch / (branch.square().sum(1, keepdim=True) / case["n"] + EPS).sqrt() * d["post"].double()
            if case["gate"] != "none":
                g = d["gate"].double()
                branch = branch * (1.0 / (1.0 + torch.exp(-g)) if case["act"] == "sigmoid" else g)
            new = new * case["res_scale"] + branch * case["y_scale"]
        if case["mode"] == "write":
            return new
        x = new / (new.square().sum(1, keepdim=True) / case["n"] + EPS).sqrt()
        if case["pre"]:
            x = x * d["pre"].double()
        return x if case["mode"] == "read" else (new, x)
    if case["op"] == "linear":
        x = d["x"].double()

        def product(i):
            a = torch.mm(x, d["w" + i].double().t().contiguous())
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
    l = d["logits"].double()
    T, E = l.shape
    m = torch.ones(T, dtype=torch.float64, device="cuda") if d["mask"] is None else d["mask"].double()
    n = float(m.sum())
    scale = 1.0 / max(n, 1.0)
    hits = d["ids"].long()[m > 0].reshape(-1)
    counts = torch.bincount(hits, minlength=E)
    f = counts.double() * scale / case["k"]
    lse = torch.logsumexp(l, 1)
    p = torch.exp(l - lse[:, None])
    P = torch.mv(p.t(), m) * scale
    balance, z = E * torch.dot(f, P), torch.dot(lse * lse, m) * scale
    loss = torch.stack([case["cb"] * balance + case["cz"] * z, balance, z, m.sum()])
    out = dict(loss=loss, counts=counts.to(torch.int32), mean_p=P)
    if case["grad"]:
        inner = case["cb"] * E * (f[None, :] - torch.mv(p, f)[:, None]) + 2.0 * case["cz"] * lse[:, None]
        g = p * inner * (m * scale)[:, None]
        out.update(dlogits=g, dbias=g.sum(0))
    return out


# ------------------------------------------------------------------------------------------------ work

def work(case):
    T = case["tokens"]
    size = {"f32": 4, "bf16": 2, "fp16": 2}
    if case["op"] == "ends":
        n, mode = case["n"], case["mode"]
        b = T * n * size[case["r"]]
        flops = 0
        if mode != "read":
            b += T * n * (size[case["y"]] + size[case["r"]])
            b += 4 * dict(none=0, channel=n, token=T, both=T * n)[case["gate"]] + (4 * n if case["post"] else 0)
            flops += T * n * (3 + (4 if case["post"] else 0))
        if mode != "write":
            b += T * n * size[case["x"]] + (4 * n if case["pre"] else 0)
            flops += T * n * 4
        return {"bytes": b, "flops": flops}
    if case["op"] == "linear":
        K, N, pairs = case["n_in"], case["n_out"], 2 if case["pair"] else 1
        b = 2 * T * K + pairs * (2 * N * K + (4 * N if case["bias"] else 0)) + T * N * size[case["y"]]
        if case["residual"]:
            b += T * N * size[case["y"]]
        return {"bytes": b, "flops": 2 * T * K * N * pairs}
    E, k = case["experts"], case["k"]
    b = 4 * T * E + 4 * T * k + (T if case["mask"] < 1.0 else 0) + 4 * (2 * E + 4)
    if case["grad"]:
        b += 4 * T * E + 4 * E
    return {"bytes": b, "flops": T * E * (12 if case["grad"] else 5)}
