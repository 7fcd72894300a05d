"""Plain 64-bit forms of the attention in front of the block and of the product with 4-bit weights, each with a bound on what
its kernel's 32-bit arithmetic may differ by.  U is half a step of f32; a chain of m roundings is off by at most m U of the
values' absolute sum."""
import numpy as np

from dense_ref import TINY, U, HALF, activate, rounding  # noqa: F401


def table(rot, base, scaling=None):
    """(radians per position of each pair, the factor on turned values)"""
    i = np.arange(rot // 2)
    kind, factor = (scaling[0], scaling[1]) if scaling else ("", 1.0)
    if kind == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2.0 * i / rot)
    if kind == "linear":
        return f / factor, 1.0
    if kind == "parts":
        trained, slow, fast = scaling[2:]
        g = np.clip((trained * f / (2 * np.pi) - slow) / (fast - slow), 0, 1)
        return f * (g + (1 - g) / factor), 0.1 * np.log(factor) + 1
    return f, 1.0


def turn(x, positions, f, scale, pairs):
    """(x turned, what the kernel's f32 may be off by before the rounding to a type).  The angle within an eighth of a turn is
    off by 3 U of itself, a polynomial by 4 U and what that moves it: 7 U on a cosine or sine, U more with the scale; a
    product's rounding and the fused sum's: 2 U."""
    x = x.astype(np.float64)
    rot = 2 * len(f)
    w = positions.astype(np.float64)[:, None] * f
    c, s = np.cos(w)[:, None], np.sin(w)[:, None]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., first], x[..., second]
    y, err = x.copy(), np.zeros_like(x)
    y[..., first], y[..., second] = scale * (a * c - b * s), scale * (b * c + a * s)
    # (the angle itself, in 64 bits: 2^-52 of it, once from the table and once from the product)
    err[..., first] = err[..., second] = abs(scale) * (np.abs(a) + np.abs(b)) * (10 * U + np.abs(w)[:, None] * 2.0 ** -51)
    return y, err


def attend(q, keys, values, scale, causal, window, t):
    """One sequence: q [n][H][D], keys and values [L][Hkv][D] -> (out, its bound, lse, its bound).  A score is a chain of D
    products, exact in f32, and U of its scale; a weight 2^(score - top) is off by that difference, its argument's two roundings
    and 2 U of the exponential's, and by half a step of the cache's type (fp16 weights, at most 2^8 of one whose sum is 1 or more,
    by half a subnormal step too); the sums by a chain of L / 16 matrix instructions of at most 16 adds, 64 waves and splits."""
    n, H, D = q.shape
    L, kv, _ = keys.shape
    g = H // kv
    q, keys, values = (v.astype(np.float64) for v in (q, keys, values))
    out, e_out = np.zeros((n, H, D)), np.zeros((n, H, D))
    lse, e_lse = np.full((n, H), -np.inf), np.zeros((n, H))
    for i in range(n):
        p = L - n + i
        hi = max(0, min(L, p + 1)) if causal else L
        lo = max(0, p - window + 1) if window else 0
        if hi <= lo:
            continue
        for h in range(H):
            k, v = keys[lo:hi, h // g], values[lo:hi, h // g]
            s = k @ q[i, h] * scale
            e_s = ((D + 4) * U * (np.abs(k) @ np.abs(q[i, h])) * abs(scale)) + 3 * U * np.abs(s)
            top = s.max()
            w = np.exp(s - top)
            total = w.sum()
            w /= total
            e_w = e_s + e_s[s.argmax()] + 3 * U * np.abs(s - top) + 4 * U
            chain = ((hi - lo) / 16 + 16 + 64) * U
            out[i, h] = w @ v
            e_out[i, h] = ((w * (e_w + HALF[t] + chain)) @ np.abs(v) + np.abs(out[i, h]) * ((w * e_w).sum() + chain)
                           + TINY["fp16"] / 2 * np.abs(v).sum(axis=0) * (t == "fp16"))
            lse[i, h] = top + np.log(total)
            e_lse[i, h] = (w * e_w).sum() + chain + 4 * U * np.abs(lse[i, h]) + 4 * U * (abs(top) + 1)
    return out, 1.01 * e_out + rounding(out, t), lse, 1.01 * e_lse


def codes_of(w):
    c = np.empty((w.shape[0], 2 * w.shape[1]))
    c[:, 0::2], c[:, 1::2] = w & 15, w >> 4
    return c


def linear4(x, layer, group, act, residual, y_type):
    """(y, its bound); layer: dicts of codes w, scales, zeros (or None) and bias, one or two.  A group's sums of code x and of x,
    exact products, are chains of group / 32 matrix instructions of at most 32 adds; the groups' a chain of as many fused adds,
    and of 8 waves and 32 slices."""
    x = x.astype(np.float64)
    K = x.shape[1]

    def product(p):
        at = np.arange(K) // group
        c = codes_of(p["w"])
        z = 8.0 if p["zeros"] is None else p["zeros"].astype(np.float64).T[:, at]
        s = p["scales"].astype(np.float64).T[:, at]
        a = x @ ((c - z) * s).T
        spread = np.abs(x) @ ((c + z) * np.abs(s)).T
        if p["bias"] is not None:
            a, spread = a + p["bias"], spread + np.abs(p["bias"])
        return a, (K / 32 + 34 + 3 + 40) * U * spread + U * np.abs(a)

    a, e = product(layer[0])
    v, slope = activate(a, act)
    e = slope * e + 12 * U * (np.abs(v) + (0 if act == "none" else np.abs(a) * slope))
    if len(layer) > 1:
        u, eu = product(layer[1])
        e = e * np.abs(u) + np.abs(v) * eu + e * eu + U * np.abs(v * u)
        v = v * u
    if residual is not None:
        v = v + residual.astype(np.float64)
        e = e + U * np.abs(v)
    return v, 1.01 * e + rounding(v, y_type)
