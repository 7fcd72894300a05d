"""CPU tests of what the dense operators refuse (smoe_block_ends, smoe_linear_run, smoe_router_balance and their binding):
every case returns during argument checking, so the pointers are never dereferenced."""
import ctypes as C

import pytest
import torch

import stratametal_amd as S

A = 0x10000000  # addresses of buffers far apart, 256-byte aligned
B, D, E, F, G = (A + (i << 34) for i in range(1, 6))
OK, EINVAL, ESIZE, ETYPE, EALIGN, ENULL = 0, -1, -2, -3, -5, -6
EDEVICE = -4
BIG = float("inf")


def ends(n=64, T=4, R=A, rt=S.F32, rld=None, y=B, yt=S.F32, yld=None, gate=None, gld=0, gstep=1, out=D, old=None, x=E, xt=S.BF16,
         xld=None, pre=F, post=G, eps=1e-6, rs=1.0, ys=1.0, act=0):
    e = S._Ends(pre, post, eps, rs, ys, act)
    ld = [n if v is None else v for v in (rld, yld, old, xld)]
    return S.lib().smoe_block_ends(C.byref(e), n, T, R, rt, ld[0], y, yt, ld[1], gate, gld, gstep, out, ld[2], x, xt, ld[3],
                                   None)


@pytest.mark.parametrize("want,kw", [
    (OK, dict(T=0)), (OK, dict(T=0, R=None, y=None, out=None, x=None)),
    (EINVAL, dict(T=-1)), (EINVAL, dict(n=0)), (EINVAL, dict(n=16385)),
    (EINVAL, dict(eps=-1e-6)), (EINVAL, dict(eps=BIG)), (EINVAL, dict(eps=float("nan"))), (EINVAL, dict(rs=BIG)),
    (EINVAL, dict(ys=float("nan"))), (EINVAL, dict(act=2)),
    (ETYPE, dict(rt=8)), (ETYPE, dict(yt=2)), (ETYPE, dict(xt=-1)),
    (ENULL, dict(R=None)), (ENULL, dict(y=None)), (ENULL, dict(out=None)), (ENULL, dict(y=None, out=None, x=None)),
    (EINVAL, dict(y=None, out=None, gate=B)),
    (EINVAL, dict(rld=-1)), (EINVAL, dict(old=63)), (EINVAL, dict(xld=0)), (EINVAL, dict(yld=1 << 41)),
    (EINVAL, dict(gate=B + (1 << 30), gstep=-1)), (EINVAL, dict(gate=B + (1 << 30), gld=-4)),
    (EALIGN, dict(R=A + 2)), (EALIGN, dict(x=E + 1)), (EALIGN, dict(gate=B + (1 << 30) + 2)), (EALIGN, dict(pre=F + 2)),
    (EINVAL, dict(out=A + 256)),            # R's rows, shifted
    (EINVAL, dict(out=A, old=65)),          # R's address, other rows
    (EINVAL, dict(x=A)),                    # f32 rows overwritten by bf16 ones
    (EINVAL, dict(x=D + 64)), (EINVAL, dict(x=D, xt=S.F32)),
    (EINVAL, dict(gate=D, gld=64)), (EINVAL, dict(post=D + 16)), (EINVAL, dict(out=F)),
    (EINVAL, dict(out=A + 4 * 32, old=64, rld=64)),
])
def test_ends(want, kw):
    assert ends(**kw) == want
    assert bool(S.lib().smoe_last_error()) == (want != OK)


def linear(n_in=64, n_out=32, wt=S.BF16, act=0, w=A, w2=None, b=None, b2=None, x=B, xld=None, T=4, r=None, rld=None, y=D, yt=S.F32,
           yld=None, ws=E, wsb=1 << 32):
    L = S._Linear(n_in, n_out, wt, act, w, w2, b, b2)
    return S.lib().smoe_linear_run(C.byref(L), x, n_in if xld is None else xld, T, r, n_out if rld is None else rld, y, yt,
                                   n_out if yld is None else yld, ws, wsb, None)


@pytest.mark.parametrize("want,kw", [
    (OK, dict(T=0)), (EINVAL, dict(T=-1)), (EINVAL, dict(n_in=0)), (EINVAL, dict(n_in=12)), (EINVAL, dict(n_in=65544)),
    (EINVAL, dict(n_out=0)), (EINVAL, dict(n_out=(1 << 24) + 1)), (ETYPE, dict(wt=S.F32)), (ETYPE, dict(wt=S.Q8_0)),
    (EINVAL, dict(act=6)), (EINVAL, dict(act=-1)), (ETYPE, dict(yt=8)),
    (ENULL, dict(x=None)), (ENULL, dict(y=None)), (ENULL, dict(w=None)), (ENULL, dict(b2=F)),
    (EINVAL, dict(xld=-8)), (EINVAL, dict(xld=68)), (EINVAL, dict(xld=(1 << 21) + 8)), (EINVAL, dict(yld=31)),
    (EINVAL, dict(r=F, rld=-1)), (EALIGN, dict(x=B + 8)), (EALIGN, dict(w=A + 8)), (EALIGN, dict(w2=A + 8)),
    (EALIGN, dict(y=D + 2)), (EALIGN, dict(r=F + 1, yt=S.F16)), (EALIGN, dict(b=F + 2)),
    (EINVAL, dict(y=B)), (EINVAL, dict(y=A)), (EINVAL, dict(b=D + 16)), (EINVAL, dict(r=D + 4)), (EINVAL, dict(r=D, rld=33)),
])
def test_linear(want, kw):
    assert linear(**kw) == want
    assert bool(S.lib().smoe_last_error()) == (want != OK)


def test_linear_workspace():
    L = S.lib()

    def size(T, n_in=8192, n_out=64):
        return L.smoe_linear_workspace_bytes(C.byref(S._Linear(n_in, n_out, S.BF16, 0, A, None, None, None)), T)

    assert size(0) > 0 and size(1) > 0 and size(-1) == 0 and size(4, n_in=9) == 0
    need = size(100)  # few tiles: K is sliced
    assert need > 256
    assert linear(n_in=8192, n_out=64, T=100, w=A, ws=None) == ENULL
    assert linear(n_in=8192, n_out=64, T=100, ws=E + 8) == EALIGN
    assert linear(n_in=8192, n_out=64, T=100, wsb=need - 257) == ESIZE


def balance(l=A, ld=None, ids=B, mask=None, T=8, n=16, k=4, cb=1.0, cz=0.0, loss=D, counts=D + 256, p=D + 8192, d=None, dld=None,
            db=None, ws=E, wsb=1 << 32):
    return S.lib().smoe_router_balance(l, n if ld is None else ld, ids, mask, T, n, k, cb, cz, loss, counts, p, d,
                                       n if dld is None else dld, db, ws, wsb, None)


@pytest.mark.parametrize("want,kw", [
    (OK, dict(T=0)), (EINVAL, dict(T=-1)), (EINVAL, dict(n=0)), (EINVAL, dict(n=1025)), (EINVAL, dict(k=0)),
    (EINVAL, dict(k=17)), (EINVAL, dict(n=512, k=65)), (EINVAL, dict(T=(1 << 22) + 1)), (EINVAL, dict(cb=BIG)),
    (EINVAL, dict(cz=float("nan"))), (ENULL, dict(l=None)), (ENULL, dict(ids=None)), (ENULL, dict(loss=None)),
    (ENULL, dict(counts=None)), (ENULL, dict(p=None)), (ENULL, dict(ws=None)), (ENULL, dict(db=F)),
    (EINVAL, dict(ld=15)), (EINVAL, dict(d=F, dld=8)), (EALIGN, dict(l=A + 2)), (EALIGN, dict(d=F + 1)),
    (EALIGN, dict(ws=E + 128)), (ESIZE, dict(wsb=100)), (EINVAL, dict(d=A + 64)), (EINVAL, dict(d=A, dld=20)),
])
def test_balance(want, kw):
    assert balance(**kw) == want
    assert bool(S.lib().smoe_last_error()) == (want != OK)


def test_binding_refuses_bad_tensors():
    x = torch.zeros((4, 64))
    g = torch.zeros((4, 2), dtype=torch.int32)
    e = object.__new__(S.BlockEnds)
    e.n_embd, e.pre, e.post, e._device = 64, None, None, -1
    for fn, why in [
        (lambda: S.BlockEnds(64, pre=x), "shape"), (lambda: S.BlockEnds(4, post=torch.zeros(4)), "not a GPU"),
        (lambda: e.read(x.double()), "float64"), (lambda: e.read(x[:, :32]), "shape"), (lambda: e.read(x[0]), "shape"),
        (lambda: e.read(torch.zeros((64, 4)).t()), "contiguous"), (lambda: e.read(x), "not a GPU"),
        (lambda: e.write(x, None), "None"), (lambda: e.join(x, None), "None"), (lambda: e.read(None), "not a tensor"),
        (lambda: S.Linear(64, 4, x), "not a GPU"), (lambda: S.Linear(64, 4, x.t()), "contiguous"),
        (lambda: S.router_balance(torch.zeros(4), g), "(tokens, experts)"),
        (lambda: S.router_balance(x.half(), g), "float16"), (lambda: S.router_balance(x, g), "not a GPU"),
    ]:
        with pytest.raises(S.SmoeError) as err:
            fn()
        assert why in str(err.value), (why, str(err.value))


def test_linear_refuses_weights_of_other_shapes():
    """A weight's shape is (n_out, n_in), or flat: the same number of values in other rows is not the layer's."""
    t = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16)  # noqa: E731
    for fn, why in [
        (lambda: S.Linear(64, 16, t(64, 16)), "w has shape (64, 16), needs (16, 64)"),
        (lambda: S.Linear(64, 16, t(8, 128)), "shape"), (lambda: S.Linear(64, 16, t(2, 8, 64)), "shape"),
        (lambda: S.Linear(64, 16, t(1023)), "shape"), (lambda: S.Linear(64, 16, t(17, 64)), "shape"),
        # (as far as the refusal of host memory: the shape is right)
        (lambda: S.Linear(64, 16, t(16, 64)), "not a GPU"), (lambda: S.Linear(64, 16, t(1024)), "not a GPU"),
    ]:
        with pytest.raises(S.SmoeError) as err:
            fn()
        assert why in str(err.value), (why, str(err.value))


@pytest.mark.parametrize("want,kw", [
    # an output over an input
    (EINVAL, dict(loss=B + 8)), (EINVAL, dict(counts=B + 64)), (EINVAL, dict(p=A + 448)), (EINVAL, dict(p=A - 60)),
    (EINVAL, dict(d=B)), (EINVAL, dict(d=B - 8 * 64 + 4)), (EINVAL, dict(d=F, db=B + 124)),
    (EINVAL, dict(mask=D + 12)), (EINVAL, dict(mask=D + 256 + 60)), (EINVAL, dict(mask=F, d=F)),
    # two outputs
    (EINVAL, dict(loss=D + 256)), (EINVAL, dict(counts=D + 12)), (EINVAL, dict(p=D + 256 + 60)), (EINVAL, dict(d=D)),
    (EINVAL, dict(d=F, db=F + 64)), (EINVAL, dict(d=F, db=D + 8192)), (EINVAL, dict(d=A, db=A + 4)),
    # columns of one matrix lie apart: the gradient beside the logits passes, its dbias over either does not
    (EINVAL, dict(ld=40, d=A + 64, dld=40, db=A + 32 * 4)), (EINVAL, dict(ld=40, d=F, dld=40, db=F + 160 + 60)),
    (EINVAL, dict(ld=40, d=F, dld=40, db=F + 160 - 60)), (EINVAL, dict(ld=40, p=A + 7 * 160 + 60)),
    # the workspace
    (EINVAL, dict(ws=A)), (EINVAL, dict(ws=B)), (EINVAL, dict(ws=D)), (EINVAL, dict(ws=D + 8192)), (EINVAL, dict(mask=E + 8)),
    (EINVAL, dict(d=E + 64)), (EINVAL, dict(d=F, db=E)),
])
def test_balance_overlaps(want, kw):
    """What one work-group writes while another reads it is refused; 8 tokens of 16 experts, 4 each."""
    assert balance(**kw) == want
    assert "overlap" in S.lib().smoe_last_error().decode()


def test_apart_is_not_overlapping():
    """What lies between a matrix's rows, or before and behind them, shares nothing with it: refused for another reason, that
    comes after the overlaps (no GPU here), or not at all."""
    if torch.cuda.is_available():
        pytest.skip("the calls would run, on addresses that are nobody's")
    for kw in (dict(ld=40, d=F, dld=40, db=F + 64), dict(ld=40, p=A + 3 * 160 + 96, loss=A + 5 * 160 + 64), dict(d=F, db=F + 512),
               dict(d=F, db=F - 64), dict(ld=40, d=A + 64, dld=40, db=G), dict(p=A + 512), dict(ids=D + 16, counts=D + 144),
               dict(ld=40, p=A + 7 * 160 + 64)):
        assert balance(**kw) == EDEVICE, kw


@pytest.mark.parametrize("kw", [dict(ws=A), dict(ws=B), dict(ws=D), dict(r=E + 4096), dict(b=E + 256), dict(w2=E + 16),
                                dict(w2=F, b2=E + 256), dict(y=E + 1024, yt=S.BF16), dict(x=E + 64, T=40)])
def test_linear_workspace_apart(kw):
    """Where K is sliced the workspace is written while x, the weights and the residual are read: it shares no byte with them."""
    kw = dict(dict(n_in=8192, n_out=64, T=100), **kw)
    assert linear(**kw) == EINVAL
    assert "workspace" in S.lib().smoe_last_error().decode()


def test_balance_row_strides():
    """Logits of one row for every token pass (to the launch, which finds no GPU here); rows that overlap, a gradient of one
    row and a gradient over the broadcast row do not."""
    for kw in (dict(ld=-16), dict(ld=1), dict(d=F, dld=0), dict(ld=0, d=A), dict(ld=0, d=A, dld=0), dict(ld=0, d=A - 448)):
        assert balance(**kw) == EINVAL, kw
    if not torch.cuda.is_available():
        assert balance(ld=0) == EDEVICE and balance(ld=0, d=A + 64) == EDEVICE
