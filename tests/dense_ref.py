"""Plain 64-bit forms of the dense operators round the block, each with a bound on what its kernel's 32-bit arithmetic may
differ by.  U is half a step of f32; a chain of m roundings is off by at most m U of the values' absolute sum."""
import numpy as np

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}   # half a step of a type, relative
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "fp16": 2.0 ** -24}  # a step of its subnormals


def rounding(v, t):
    return HALF[t] * np.abs(v) + TINY[t]


def rms_scale(v, eps):
    return 1.0 / np.sqrt((v * v).mean(axis=1, keepdims=True) + eps)


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-v))


def ends(R, y, gate, pre, post, res_scale, y_scale, eps, act, r_type, x_type):
    """(out, its bound, x, its bound) in float64; y None: out is R.  A row's sum of squares is a chain of at most 32 fused
    adds in a lane, 6 of the wave's butterfly and 16 over waves: 54 U, half of that in 1 / sqrt, and the mean, eps, root and
    quotient: 32 U on a scale.  A branch value is scaled by rs, post, the gate (a sigmoid: 6 U) and y_scale: 42 U."""
    R = R.astype(np.float64)
    out, err, spread = R, np.zeros_like(R), 0.0
    if y is not None:
        z = y.astype(np.float64)
        if post is not None:
            z = z * rms_scale(z, eps) * post.astype(np.float64)
        if gate is not None:
            g = gate.astype(np.float64)
            z = z * (sigmoid(g) if act else g)
        a, b = res_scale * R, y_scale * z
        out = a + b
        err = 42 * U * np.abs(b) + 2 * U * np.abs(a) + U * np.abs(out)
        rms = lambda v: np.sqrt((v * v).mean(axis=1, keepdims=True))  # noqa: E731
        spread = (42 * U * rms(b) + 3 * U * rms(a)) / np.maximum(rms(out), 1e-300)
    rs = rms_scale(out, eps)
    w = np.ones(out.shape[1]) if pre is None else pre.astype(np.float64)
    x = out * rs * w
    x_err = np.abs(x) * (36 * U + spread) + err * rs * np.abs(w)
    return out, 1.01 * err + rounding(out, r_type), x, 1.01 * x_err + rounding(x, x_type)


def activate(a, act):
    """(value, a bound on its slope)"""
    one = np.ones_like(a)
    if act == "silu":
        return a * sigmoid(a), 1.1 * one
    if act == "gelu":
        return a * sigmoid(2 * np.sqrt(2 / np.pi) * (a + 0.044715 * a ** 3)), 1.14 * one
    if act == "relu":
        return np.maximum(a, 0), one
    if act == "relu2":
        return np.maximum(a, 0) ** 2, 2 * np.maximum(a, 0) + 1e-3
    if act == "sigmoid":
        return sigmoid(a), 0.25 * one
    return a, one


def linear(x, w, bias, w2, bias2, act, residual, y_type):
    """(y, its bound): a sum of K products, exact in f32, is a chain of K / 32 matrix instructions of at most 32 adds each,
    and of at most 32 slices of K; an activation's own arithmetic is below 12 U of its argument and value."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    K = x.shape[1]
    m = (K / 32 + 34 + 32) * U

    def product(w, b):
        a, s = x @ w.T, np.abs(x) @ np.abs(w).T
        if b is not None:
            a, s = a + b, s + np.abs(b)
        return a, m * s + U * np.abs(a)

    a, e = product(w, bias)
    v, slope = activate(a, act)
    e = slope * e + 12 * U * (np.abs(v) + (0 if act == "none" else np.abs(a) * slope))
    if w2 is not None:
        u, eu = product(w2.astype(np.float64), bias2)
        e = e * np.abs(u) + np.abs(v) * eu + e * eu + U * np.abs(v * u)
        v = v * u
    if residual is not None:
        v = v + residual.astype(np.float64)
        e = e + U * np.abs(v)
    return v, 1.01 * e + rounding(v, y_type)


def balance(logits, ids, mask, cb, cz):
    """A dict of the results and one of their bounds.  With d = top - v: v - top is off by U d, its exponential by U d + 3 U
    of itself, a row's sum by 24 U more (16 in a lane, 6 of the butterfly): p by (d + 30) U; log sum exp by 30 U, U of top
    and 4 U of the logarithm.  Sums over the tokens: a wave's chain of T / 4 rows at most, f32."""
    l = logits.astype(np.float64)
    T, E = l.shape
    k = ids.shape[1]
    m = np.ones(T, bool) if mask is None else mask.astype(bool)
    l, idm = l[m], ids[m]
    n = int(m.sum())
    flat = idm[(idm >= 0) & (idm < E)]
    counts = np.bincount(flat, minlength=E).astype(np.int64)
    res, err = dict(counts=counts), {}
    inv = 1.0 / n if n else 0.0
    with np.errstate(invalid="ignore", divide="ignore"):
        top = l.max(axis=1, keepdims=True) if n else np.zeros((0, 1))
        none = np.isneginf(top)
        top = np.where(none, 0.0, top)
        ex = np.exp(l - top)
        s = ex.sum(axis=1, keepdims=True)
        p = np.where(none, 0.0, ex / np.where(none, 1.0, s))
        lse = np.where(none, 0.0, top + np.log(np.where(none, 1.0, s)))
        d = np.where(np.isneginf(l), 0.0, top - l)
    ep = p * (d + 30) * U
    el = (30 + np.abs(top) + 4 * np.abs(lse - top)) * U + U * np.abs(lse)
    f = counts * inv / k
    P = p.sum(axis=0) * inv
    chain = (max(T, 4) / 4 + 8) * U
    err["mean_p"] = ep.sum(axis=0) * inv + chain * P + TINY["f32"]
    bal, z = E * (f * P).sum(), (lse ** 2).sum() * inv
    e_bal = E * (f * err["mean_p"]).sum() + 4 * U * bal
    e_z = (2 * np.abs(lse) * el).sum() * inv + 4 * U * z
    res["mean_p"], res["loss"] = P, np.array([cb * bal + cz * z, bal, z, n])
    err["loss"] = np.array([abs(cb) * e_bal + abs(cz) * e_z + 4 * U * (abs(cb) * bal + abs(cz) * z), e_bal, e_z, 0.0]) + 1e-30
    g, eg = np.zeros((T, E)), np.zeros((T, E))
    fp = (p * f).sum(axis=1, keepdims=True)
    c = cb * E * (f - fp) + 2 * cz * lse
    e_fp = (ep * f).sum(axis=1, keepdims=True) + 26 * U * fp
    e_c = abs(cb) * E * (e_fp + 4 * U * (f + fp)) + 2 * abs(cz) * (el + 3 * U * np.abs(lse)) + U * np.abs(c)
    g[m], eg[m] = p * c * inv, (ep * np.abs(c) + p * e_c + 4 * U * np.abs(p * c)) * inv
    res["dlogits"], err["dlogits"] = g, 1.01 * eg + TINY["f32"]
    res["dbias"] = g.sum(axis=0)
    err["dbias"] = err["dlogits"].sum(axis=0) + chain * np.abs(g).sum(axis=0) + U * np.abs(res["dbias"]) + TINY["f32"]
    return res, err
