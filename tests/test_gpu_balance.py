"""GPU tests of the router's balance loss, counts and gradients against their plain form in 64 bits (dense_ref.py), and of
that form's gradient against differences of its loss."""
import numpy as np
import pytest
import torch

import dense_ref as D
import stratametal_amd as S
from test_gpu_ends import host, say


def make(seed, T, E, k, frac=None):
    rng = np.random.default_rng(seed)
    l = (rng.standard_normal((T, E)) + rng.standard_normal(E)).astype(np.float32)
    ids = np.argsort(-l, axis=1, kind="stable")[:, :k].astype(np.int32)
    return l, ids, None if frac is None else (rng.random(T) < frac)


def run(l, ids, mask, cb, cz, grad=True):
    m = None if mask is None else torch.from_numpy(mask).cuda()
    return S.router_balance(torch.from_numpy(l).cuda(), torch.from_numpy(ids).cuda(), mask=m, balance_coef=cb, z_coef=cz,
                            grad=grad)


def check(out, want, bound):
    for name, t in out.items():
        got = t.cpu().numpy().astype(np.float64)
        if name == "counts":
            assert np.array_equal(got, want[name])
        else:
            # (a result past f32's largest value by more than its bound rounds to infinity)
            past = np.abs(want[name]) - bound[name] > float(np.finfo(np.float32).max) * (1 + 2.0 ** -25)
            bad = np.where(past, got != np.copysign(np.inf, want[name]), ~(np.abs(got - want[name]) <= bound[name]))
            assert not bad.any(), (name, got[bad][:4], want[name][bad][:4], bound[name][bad][:4])


def test_plain_gradient_against_differences():
    l, ids, mask = make(1, 12, 9, 3, 0.7)
    cb, cz, h = 0.7, 0.3, 1e-5
    want, _ = D.balance(l, ids, mask, cb, cz)
    rng = np.random.default_rng(2)
    for _ in range(5):
        v = rng.standard_normal(l.shape)
        up, dn = (D.balance(l.astype(np.float64) + s * h * v, ids, mask, cb, cz)[0]["loss"][0] for s in (1, -1))
        assert abs((up - dn) / (2 * h) - (want["dlogits"] * v).sum()) <= 1e-8


SIZES = [(1, 1, 1), (1, 512, 10), (3, 5, 2), (4, 64, 6), (5, 65, 64), (17, 128, 8), (64, 512, 10), (63, 129, 1), (257, 300, 5),
         (500, 1024, 8), (2047, 16, 4), (2048, 60, 2), (3000, 257, 16), (5000, 512, 10)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k", SIZES)
@pytest.mark.parametrize("frac", [None, 0.6])
def test_balance(T, E, k, frac):
    say(f"case: balance T={T} E={E} k={k} frac={frac}")
    l, ids, mask = make(T + E, T, E, k, frac)
    want, bound = D.balance(l, ids, mask, 0.5, 0.1)
    out = run(l, ids, mask, 0.5, 0.1)
    check(out, want, bound)
    for name, t in run(l, ids, mask, 0.5, 0.1, grad=False).items():
        if name == "counts":
            assert torch.equal(t, out[name])
    check(run(l, ids, mask, 0.5, 0.1, grad=False), want, bound)


@pytest.mark.gpu
def test_empty_mask_and_masked_values():
    """No token counts: zeros.  What masked rows hold (NaN, infinities, ids of any value) reaches nothing."""
    say("case: balance masks")
    T, E, k = 40, 100, 4
    l, ids, _ = make(3, T, E, k)
    out = run(l, ids, np.zeros(T, bool), 1.0, 1.0)
    assert all(bool((t == 0).all()) for t in out.values())
    mask = np.arange(T) % 3 != 0
    want = run(l, ids, mask, 1.0, 0.2)
    l2, ids2 = l.copy(), ids.copy()
    l2[~mask] = np.nan
    l2[0] = np.inf
    l2[3] = -np.inf
    l2[6] = np.finfo(np.float32).min
    ids2[~mask] = -7
    ids2[9] = 1 << 30
    got = run(l2, ids2, mask, 1.0, 0.2)
    assert all(torch.equal(got[name], want[name]) for name in want)
    assert bool((got["dlogits"][torch.from_numpy(~mask).cuda()] == 0).all())


@pytest.mark.gpu
def test_excluded_experts_and_far_logits():
    """Experts at -inf or the type's lowest value, a counted row of -inf alone, logits of +-80, repeated and outside ids."""
    say("case: balance excluded experts")
    T, E, k = 50, 130, 3
    l, ids, _ = make(4, T, E, k)
    l[:, 5] = -np.inf
    l[:, 64:70] = np.finfo(np.float32).min
    l[7] = -np.inf
    l[8] = np.finfo(np.float32).min
    l[9] = 80.0 * np.sign(l[9])
    l[10] += 1000.0
    ids[11] = 3
    ids[12] = [-1, E, 2]
    want, bound = D.balance(l, ids, None, 1.0, 1e-4)
    check(run(l, ids, None, 1.0, 1e-4), want, bound)


@pytest.mark.gpu
def test_nan_spreads_only_where_the_formula_does():
    say("case: balance NaN")
    l, ids, _ = make(5, 30, 40, 2)
    l[4, 7] = np.nan
    out = run(l, ids, None, 1.0, 0.0)
    assert bool(torch.isnan(out["loss"][:3]).all()) and float(out["loss"][3]) == 30
    assert bool(torch.isnan(out["dlogits"][4]).all()) and not bool(torch.isnan(out["dlogits"][[3, 5]]).any())


@pytest.mark.gpu
def test_row_strides_and_gradient_in_place():
    say("case: balance strides")
    T, E, k = 70, 90, 4
    l, ids, _ = make(6, T, E, k)
    want = run(l, ids, None, 0.3, 0.2)
    wide = torch.full((T, E + 11), float("nan"), device="cuda")
    wide[:, 3:3 + E] = torch.from_numpy(l).cuda()
    ls, it = wide[:, 3:3 + E], torch.from_numpy(ids).cuda()
    got = S.router_balance(ls, it, balance_coef=0.3, z_coef=0.2, grad=True)
    assert all(torch.equal(got[name], want[name]) for name in want)
    import ctypes as C
    n = S.lib().smoe_router_balance_workspace_bytes(T, E)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    S._check(S.lib().smoe_router_balance(ls.data_ptr(), E + 11, it.data_ptr(), None, T, E, k, 0.3, 0.2,
                                         got["loss"].data_ptr(), got["counts"].data_ptr(), got["mean_p"].data_ptr(),
                                         ls.data_ptr(), E + 11, None, ws.data_ptr(), n, S._stream()))
    assert torch.equal(ls, want["dlogits"]) and bool(torch.isnan(wide[:, :3]).all()) and bool(torch.isnan(wide[:, 3 + E:]).all())


@pytest.mark.gpu
def test_results_share_no_memory():
    """Each result is a tensor of its own: one may be changed in place, by differentiable operands too."""
    say("case: balance results apart")
    l, ids, _ = make(4, 33, 40, 3)
    o = run(l, ids, None, 0.01, 0.001)
    assert len({t.untyped_storage().data_ptr() for t in o.values()}) == len(o)
    w = torch.ones(4, device="cuda", requires_grad=True)
    keep = {k: t.clone() for k, t in o.items()}
    o["loss"].mul_(w).sum().backward()
    assert torch.equal(w.grad, keep["loss"])
    for k in ("counts", "mean_p", "dlogits", "dbias"):
        assert torch.equal(o[k], keep[k])


@pytest.mark.gpu
@pytest.mark.parametrize("top", [1e6, 1e7, 2e9, 1e10, 1e12, 1e20, 9e29, 1e31])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("T,E", [(20, 130), (300, 512)])
def test_counted_rows_far_out(top, sign, T, E):
    """Counted rows whose largest logit is far from zero: all of them alike, as a fill leaves them, or some steps of f32 apart
    (p as of any row); by one work-group and by many, without gradients too."""
    say(f"case: balance far rows top={sign * top} T={T} E={E}")
    l, ids, _ = make(7, T, E, 4)
    far = np.float32(sign * top)
    l[1] = far
    l[2::5] = far + np.float32(np.spacing(np.abs(far))) * np.round(3 * l[2::5])
    l[3, ::2] = far if sign > 0 else -np.inf
    want, bound = D.balance(l, ids, None, 0.5, 1e-8)
    check(run(l, ids, None, 0.5, 1e-8), want, bound)
    check(run(l, ids, None, 0.5, 1e-8, grad=False), want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E", [(1, 12), (40, 129), (300, 512)])
def test_one_row_for_every_token(T, E):
    """Logits broadcast over the tokens (row stride 0) give what their copies give."""
    say(f"case: balance broadcast T={T} E={E}")
    l, ids, mask = make(9, T, E, 4, 0.8)
    one = torch.from_numpy(l[:1]).cuda().expand(T, E)
    it, m = torch.from_numpy(ids).cuda(), torch.from_numpy(mask).cuda()
    for grad in (False, True):
        got = S.router_balance(one, it, mask=m, balance_coef=0.3, z_coef=0.2, grad=grad)
        want = S.router_balance(one.contiguous(), it, mask=m, balance_coef=0.3, z_coef=0.2, grad=grad)
        assert all(torch.equal(got[name], want[name]) for name in want)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k", [(64, 512, 64), (64, 64, 64), (50, 1000, 63), (65, 512, 64)])
def test_few_tokens_of_many_experts(T, E, k):
    """The most pairs of one work-group, and the first batch of several."""
    say(f"case: balance few tokens T={T} E={E} k={k}")
    l, ids, mask = make(T + k, T, E, k, 0.8)
    want, bound = D.balance(l, ids, mask, 0.5, 0.1)
    check(run(l, ids, mask, 0.5, 0.1), want, bound)
