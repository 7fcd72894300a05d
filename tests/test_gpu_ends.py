"""GPU tests of the ends of a block on one residual stream (BlockEnds) against their plain form in 64 bits (dense_ref.py)."""
import numpy as np
import pytest
import torch

import dense_ref as D
import stratametal_amd as S

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def say(*a):
    print(*a, flush=True)


def host(t):
    return t.detach().float().cpu().numpy()


def close(got, want, bound):
    got = host(got).astype(np.float64)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


def normal(seed, *shape, sigma=1.0):
    return torch.from_numpy((np.random.default_rng(seed).standard_normal(shape) * sigma).astype(np.float32)).cuda()


def make(seed, T, n, r, y, gate, pre=True, post=True, **kw):
    R, b = normal(seed, T, n).to(TYPES[r]), normal(seed + 1, T, n, sigma=0.3).to(TYPES[y])
    shape = dict(none=None, channel=(n,), token=(T, 1), both=(T, n))[gate]
    g = None if shape is None else normal(seed + 2, *shape)
    w = [1.0 + normal(seed + 3 + i, n, sigma=0.2) if on else None for i, on in enumerate((pre, post))]
    return R, b, g, S.BlockEnds(n, pre=w[0], post=w[1], eps=EPS, **kw)


def check(e, R, y, g, r, x_type, out, x):
    act = e._c.gate_act == S.GATE_SIGMOID
    gate = None if g is None else host(g.expand(R.shape))
    wo, eo, wx, ex = D.ends(host(R), None if y is None else host(y), gate, None if e.pre is None else host(e.pre),
                            None if e.post is None else host(e.post), e._c.res_scale, e._c.y_scale, e._c.eps, act, r, x_type)
    if out is not None:
        close(out, wo, eo)
    if x is not None:
        close(x, wx, ex)


SIZES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 511), (4, 512), (9, 513), (1, 2048), (6, 2049), (3, 4096), (2, 5000), (2, 8192),
         (3, 8200), (1, 16383), (2, 16384)]


@pytest.mark.parametrize("T,n", SIZES)
@pytest.mark.parametrize("types", [("f32", "f32", "bf16"), ("bf16", "fp16", "f32"), ("fp16", "bf16", "fp16")])
def test_join(T, n, types):
    r, y, x = types
    say(f"case: ends join T={T} n={n} {types}")
    R, b, g, e = make(n, T, n, r, y, "channel", res_scale=0.5, y_scale=2.0, gate_act=S.GATE_SIGMOID)
    out, xo = e.join(R, b, gate=g, x_dtype=TYPES[x])
    check(e, R, b, g, r, x, out, xo)
    assert torch.equal(e.write(R, b, gate=g), out)  # the parts give the whole's values


@pytest.mark.parametrize("gate", ["none", "channel", "token", "both"])
@pytest.mark.parametrize("post,pre", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("T,n", [(70, 264), (33, 1001)])
def test_parts(gate, post, pre, T, n):
    say(f"case: ends parts T={T} n={n} gate={gate} post={post} pre={pre}")
    R, b, g, e = make(7, T, n, "f32", "bf16", gate, pre=pre, post=post)
    out = e.write(R, b, gate=g)
    check(e, R, b, g, "f32", "f32", out, None)
    x = e.read(R, x_dtype=torch.float16)
    check(e, R, None, None, "f32", "fp16", None, x)
    out2, x2 = e.join(R, b, gate=g)
    assert torch.equal(out2, out)
    check(e, R, b, g, "f32", "f32", out2, x2)


@pytest.mark.parametrize("n", [256, 1000, 2047])
def test_strides_in_place_and_rows_behind(n):
    """Rows of a wider matrix, a repeated row, out over R and x over y, and the rows past the tokens left as they were."""
    say(f"case: ends strides n={n}")
    T = 11
    R, b, g, e = make(3, T, n, "bf16", "bf16", "both")
    want, wx = e.join(R, b, gate=g)
    wide = torch.full((T + 2, n + 40), 7.0, dtype=torch.bfloat16, device="cuda")
    wide[:T, 8:8 + n] = R
    Rs = wide[:T, 8:8 + n]
    gt = torch.empty((n, T), device="cuda")
    gt.copy_(g.t())
    bx = torch.full((T + 2, n), 5.0, dtype=torch.bfloat16, device="cuda")
    bx[:T] = b
    out, x = e.join(Rs, bx[:T], gate=gt.t(), out=Rs, x=bx[:T])
    assert torch.equal(out, want) and torch.equal(x, wx)
    assert bool((wide[T:] == 7).all()) and bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + n:] == 7).all())
    assert bool((bx[T:] == 5).all())
    one = R[:1].expand(T, n)
    o1 = e.write(one, b, gate=g)
    assert torch.equal(o1, e.write(one.contiguous(), b, gate=g))
    both = torch.empty((T, 2 * n), dtype=torch.bfloat16, device="cuda")  # out and x side by side
    e.join(R, b, gate=g, out=both[:, :n], x=both[:, n:])
    assert torch.equal(both[:, :n], want) and torch.equal(both[:, n:], wx)


@pytest.mark.parametrize("n", [64, 2048, 777])
def test_rows_of_any_magnitude(n):
    """Rows whose squares leave f32, zeros, a row of infinities and NaN: each row's own."""
    say(f"case: ends magnitudes n={n}")
    R = normal(5, 8, n)
    R[1] *= 1e30
    R[2] *= 1e-30
    R[3] = 0.0
    R[4, 0] = float("inf")
    R[5, n // 2] = float("nan")
    R[6] *= 2e37
    for eps in (1e-6, 0.0):
        e = S.BlockEnds(n, eps=eps)
        x = e.read(R)
        keep = [0, 1, 2, 6, 7]
        _, _, wx, ex = D.ends(host(R[keep]), None, None, None, None, 1, 1, eps, False, "f32", "f32")
        close(x[keep], wx, ex)
        assert bool(torch.isnan(x[5]).all()) and bool(torch.isnan(x[4, 0]))
        assert bool((x[3] == 0).all()) if eps else bool(torch.isnan(x[3]).all())


def test_long_batch_offsets():
    """Rows past 2^31 values and 2^32 bytes."""
    T, n = 40000, 65536
    say("case: ends long offsets")
    big = torch.zeros((T, n), dtype=torch.bfloat16, device="cuda")
    R = big[:, :64]
    R.copy_(normal(1, T, 64))
    e = S.BlockEnds(64, eps=EPS)
    x = e.read(R, x=big[:, 128:192])
    assert torch.equal(x[-5:], e.read(R[-5:].contiguous())) and torch.equal(x[:5], e.read(R[:5].contiguous()))
    assert bool((big[-1, 192:] == 0).all())
