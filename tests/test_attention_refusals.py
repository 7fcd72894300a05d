"""CPU tests of what the attention in front of the block and the product with 4-bit weights refuse (smoe_rope_table,
smoe_rope_run, smoe_kv_append, smoe_attend, smoe_linear4_run and their binding): every case returns during argument checking,
so the pointers are never dereferenced; and of the tables that smoe_rope_table makes on the host."""
import ctypes as C

import numpy as np
import pytest
import torch

import attention_ref as A
import stratametal_amd as S
from test_dense_refusals import BIG, EALIGN, EINVAL, ENULL, ESIZE, ETYPE, OK

P = [0x10000000 + (i << 36) for i in range(16)]  # addresses of buffers far apart, 256-byte aligned
NAN = float("nan")


def verdict(status, want):
    assert status == want, S.lib().smoe_last_error()
    assert bool(S.lib().smoe_last_error()) == (want != OK)


def rope(dim=64, rot=64, layout=0, scale=1.0, turns=P[0], pos=P[1], T=4, H=2, x=P[2], xt=S.F32, xld=None, y=P[3], yt=S.F32, yld=None):
    r = S._Rope(dim, rot, layout, scale, turns)
    ld = [H * dim if v is None else v for v in (xld, yld)]
    return S.lib().smoe_rope_run(C.byref(r), pos, T, H, x, xt, ld[0], y, yt, ld[1], None)


@pytest.mark.parametrize("want,kw", [
    (OK, dict(T=0)), (EINVAL, dict(T=-1)), (EINVAL, dict(dim=0, rot=2)), (EINVAL, dict(dim=65)), (EINVAL, dict(dim=1026)), (EINVAL, dict(rot=0)),
    (EINVAL, dict(rot=66)), (EINVAL, dict(rot=7)), (EINVAL, dict(layout=2)), (EINVAL, dict(scale=BIG)), (EINVAL, dict(scale=NAN)),
    (EINVAL, dict(H=0)), (EINVAL, dict(H=4097)), (ETYPE, dict(xt=8)), (ETYPE, dict(yt=2)), (ENULL, dict(turns=None)), (ENULL, dict(pos=None)),
    (ENULL, dict(x=None)), (ENULL, dict(y=None)), (EINVAL, dict(xld=-1)), (EINVAL, dict(yld=127)), (EINVAL, dict(xld=1 << 41)),
    (EALIGN, dict(x=P[2] + 2)), (EALIGN, dict(y=P[3] + 1, yt=S.F16)), (EALIGN, dict(turns=P[0] + 4)), (EALIGN, dict(pos=P[1] + 2)),
    (EINVAL, dict(y=P[2] + 4)), (EINVAL, dict(y=P[2], yld=129)), (EINVAL, dict(y=P[2], yt=S.F16)), (EINVAL, dict(y=P[0])), (EINVAL, dict(y=P[1])),
])
def test_rope(want, kw):
    verdict(rope(**kw), want)


@pytest.mark.parametrize("want,args", [
    (OK, (64, 1e4, 0, 0, 0, 0, 0)), (OK, (2, 1e4, 2, 8.0, 0, 0, 0)), (EINVAL, (0, 1e4, 0, 1, 0, 0, 0)), (EINVAL, (63, 1e4, 0, 1, 0, 0, 0)),
    (EINVAL, (1026, 1e4, 0, 1, 0, 0, 0)), (EINVAL, (64, 0.0, 0, 1, 0, 0, 0)), (EINVAL, (64, NAN, 0, 1, 0, 0, 0)), (EINVAL, (64, BIG, 0, 1, 0, 0, 0)),
    (EINVAL, (64, 1e4, 4, 1, 0, 0, 0)), (EINVAL, (64, 1e4, -1, 1, 0, 0, 0)), (EINVAL, (64, 1e4, 1, 0.0, 0, 0, 0)), (EINVAL, (64, 1e4, 2, NAN, 0, 0, 0)),
    (EINVAL, (64, 1e4, 3, 8.0, 0.0, 1, 32)), (EINVAL, (64, 1e4, 3, 8.0, 8192.0, 4, 4)), (EINVAL, (64, 1e4, 3, 8.0, 8192.0, 1, BIG)),
])
def test_rope_table(want, args):
    turns, scale = (C.c_double * 512)(), C.c_float()
    verdict(S.lib().smoe_rope_table(*args, turns, C.byref(scale)), want)
    verdict(S.lib().smoe_rope_table(*args, None, C.byref(scale)), ENULL)


@pytest.mark.parametrize("rot", [2, 4, 64, 128, 256])
@pytest.mark.parametrize("scaling", [None, ("linear", 4.0), ("ntk", 8.0), ("parts", 16.0, 8192, 1.0, 32.0), ("parts", 8.0, 8192, 1.0, 4.0)])
def test_rope_table_values(rot, scaling):
    turns, scale = S.rope_table(rot, 5e5, scaling)
    f, want = A.table(rot, 5e5, scaling)
    assert np.allclose(np.array(turns) * 2 * np.pi, f, rtol=1e-13, atol=0) and abs(scale - want) <= 2.0 ** -24 * 2


def kv(**kw):
    d = dict(k=P[4], v=P[5], type=S.BF16, n_pages=100, page_size=16, n_kv_heads=2, head_dim=64)
    d.update(kw)
    return S._Kv(*(d[n] for n, _ in S._Kv._fields_))


BAD_KV = [(ETYPE, dict(type=S.F32)), (EINVAL, dict(n_pages=0)), (EINVAL, dict(page_size=0)), (EINVAL, dict(page_size=65537)),
          (EINVAL, dict(n_kv_heads=0)), (EINVAL, dict(n_kv_heads=4097)), (EINVAL, dict(head_dim=4)), (EINVAL, dict(head_dim=60)),
          (EINVAL, dict(head_dim=264)), (EINVAL, dict(n_pages=1 << 26, page_size=32)), (EINVAL, dict(n_pages=2 ** 31 - 1, n_kv_heads=4096))]


def append(cache=None, r=(64, 64, 0, 1.0, P[0]), pos=P[1], slots=P[2], T=4, xt=S.BF16, q=P[6], qld=256, H=4, qo=P[7], qold=256, k=P[8], kld=128,
           v=P[9], vld=128):
    c = kv(**(cache or {}))
    rr = S._Rope(*r) if r else None
    return S.lib().smoe_kv_append(C.byref(c), C.byref(rr) if rr else None, pos, slots, T, xt, q, qld, H, qo, qold, k, kld, v, vld, None)


@pytest.mark.parametrize("want,kw", [
    (OK, dict(T=0)), (OK, dict(T=0, r=None, q=None, qo=None)), *[(w, dict(cache=c)) for w, c in BAD_KV],
    (EINVAL, dict(T=-1)), (EINVAL, dict(r=(128, 64, 0, 1.0, P[0]))), (EINVAL, dict(r=(64, 63, 0, 1.0, P[0]))), (ETYPE, dict(xt=8)),
    (ENULL, dict(q=None)), (ENULL, dict(qo=None)), (EINVAL, dict(r=None)), (EINVAL, dict(H=0)), (ENULL, dict(k=None)), (ENULL, dict(v=None)),
    (ENULL, dict(slots=None)), (ENULL, dict(pos=None)), (ENULL, dict(r=(64, 64, 0, 1.0, None))), (ENULL, dict(cache=dict(k=None))),
    (EINVAL, dict(kld=-1)), (EINVAL, dict(qold=255)), (EALIGN, dict(cache=dict(v=P[5] + 8))), (EALIGN, dict(k=P[8] + 1)), (EALIGN, dict(slots=P[2] + 4)),
    (EALIGN, dict(q=P[6] + 2, xt=S.F32)), (EINVAL, dict(qo=P[6] + 2)), (EINVAL, dict(qo=P[6], xt=S.F32)), (EINVAL, dict(qo=P[6], qold=264)),
    (EINVAL, dict(k=P[4])), (EINVAL, dict(v=P[4] + 512)), (EINVAL, dict(q=P[5])), (EINVAL, dict(qo=P[4])), (EINVAL, dict(cache=dict(v=P[4] + 1024))),
    (EINVAL, dict(qo=P[2])), (EINVAL, dict(qo=P[8])),
])
def test_append(want, kw):
    verdict(append(**kw), want)


def attend(cache=None, q=P[6], qld=256, T=4, H=4, qs=P[0], kl=P[1], B=2, pages=P[2], pld=8, mp=8, ml=128, scale=0.1, causal=1, window=0, out=P[7],
           old=256, lse=None, ws=P[10], wsb=1 << 34):
    c = kv(**(cache or {}))
    return S.lib().smoe_attend(C.byref(c), q, qld, T, H, qs, kl, B, pages, pld, mp, ml, scale, causal, window, out, old, lse, ws, wsb, None)


@pytest.mark.parametrize("want,kw", [
    (OK, dict(T=0)), (OK, dict(B=0)), *[(w, dict(cache=c)) for w, c in BAD_KV],
    (EINVAL, dict(T=-1)), (EINVAL, dict(B=-1)), (EINVAL, dict(H=3)), (EINVAL, dict(H=0)), (EINVAL, dict(H=8192)), (EINVAL, dict(T=1 << 21)),
    (EINVAL, dict(B=(1 << 20) + 1)), (EINVAL, dict(ml=-1)), (EINVAL, dict(ml=129)), (EINVAL, dict(mp=-1)), (EINVAL, dict(ml=(1 << 30) + 1, mp=1 << 30)),
    (EINVAL, dict(scale=NAN)), (EINVAL, dict(window=-1)), (EINVAL, dict(window=5, causal=0)), (ENULL, dict(q=None)), (ENULL, dict(qs=None)),
    (ENULL, dict(kl=None)), (ENULL, dict(pages=None)), (ENULL, dict(out=None)), (ENULL, dict(cache=dict(v=None))), (EINVAL, dict(qld=-8)),
    (EINVAL, dict(qld=257)), (EINVAL, dict(old=255)), (EINVAL, dict(pld=-1)), (EALIGN, dict(q=P[6] + 8)), (EALIGN, dict(out=P[7] + 1)),
    (EALIGN, dict(lse=P[8] + 2)), (EALIGN, dict(cache=dict(k=P[4] + 8))), (EALIGN, dict(qs=P[0] + 2)),
    (EINVAL, dict(out=P[6])), (EINVAL, dict(out=P[4])), (EINVAL, dict(lse=P[7])), (EINVAL, dict(lse=P[0])), (EINVAL, dict(out=P[2])),
])
def test_attend(want, kw):
    verdict(attend(**kw), want)


def test_attend_workspace():
    def size(H=4, T=4, B=2, ml=128, window=0, **c):
        return S.lib().smoe_attend_workspace_bytes(C.byref(kv(**c)), H, T, B, ml, window)

    assert size() > 0 and size(T=0) > 0 and size(T=-1) == 0 and size(H=3) == 0 and size(ml=-1) == 0 and size(head_dim=7) == 0 and size(window=-1) == 0
    need = size(T=1, B=1, ml=100000)
    if need > 256:
        kw = dict(T=1, B=1, mp=6250, ml=100000)
        verdict(attend(ws=None, **kw), ENULL)
        verdict(attend(ws=P[10] + 8, **kw), EALIGN)
        verdict(attend(wsb=need - 257, **kw), ESIZE)
        verdict(attend(ws=P[7], **kw), EINVAL)
        verdict(attend(ws=P[4], **kw), EINVAL)


def linear4(n_in=64, n_out=32, xt=S.BF16, act=0, group=64, st=S.F16, w=P[0], w2=None, s=P[1], s2=None, z=None, z2=None, b=None, b2=None, x=P[4],
            xld=None, T=4, r=None, rld=None, y=P[5], yt=S.F32, yld=None, ws=P[6], wsb=1 << 32):
    L = S._Linear4(n_in, n_out, xt, act, group, st, w, w2, s, s2, z, z2, b, b2)
    return S.lib().smoe_linear4_run(C.byref(L), x, n_in if xld is None else xld, T, r, n_out if rld is None else rld, y, yt,
                                    n_out if yld is None else yld, ws, wsb, None)


@pytest.mark.parametrize("want,kw", [
    (OK, dict(T=0)), (EINVAL, dict(T=-1)), (EINVAL, dict(n_in=0)), (EINVAL, dict(n_in=48)), (EINVAL, dict(n_in=65568)), (EINVAL, dict(n_out=0)),
    (EINVAL, dict(n_out=(1 << 24) + 1)), (ETYPE, dict(xt=S.F32)), (ETYPE, dict(st=2)), (EINVAL, dict(group=0)), (EINVAL, dict(group=48)),
    (EINVAL, dict(act=6)), (ETYPE, dict(yt=8)), (ENULL, dict(x=None)), (ENULL, dict(y=None)), (ENULL, dict(w=None)), (ENULL, dict(s=None)),
    (ENULL, dict(w2=P[2])), (ENULL, dict(b2=P[2])), (ENULL, dict(s2=P[2])), (ENULL, dict(z2=P[2])), (EINVAL, dict(xld=-8)), (EINVAL, dict(xld=68)),
    (EINVAL, dict(xld=(1 << 21) + 8)), (EINVAL, dict(yld=31)), (EINVAL, dict(r=P[7], rld=-1)), (EALIGN, dict(x=P[4] + 8)), (EALIGN, dict(w=P[0] + 8)),
    (EALIGN, dict(s=P[1] + 1)), (EALIGN, dict(y=P[5] + 2)), (EALIGN, dict(b=P[7] + 2)), (EINVAL, dict(y=P[4])), (EINVAL, dict(y=P[0])),
    (EINVAL, dict(y=P[1])), (EINVAL, dict(z=P[5] + 8)), (EINVAL, dict(b=P[5] + 16)), (EINVAL, dict(r=P[5] + 4)), (EINVAL, dict(r=P[5], rld=33)),
])
def test_linear4(want, kw):
    verdict(linear4(**kw), want)


def test_linear4_workspace():
    def size(T, n_in=8192, n_out=64, group=128):
        L = S._Linear4(n_in, n_out, S.BF16, 0, group, S.F16, P[0], None, P[1], None, None, None, None, None)
        return S.lib().smoe_linear4_workspace_bytes(C.byref(L), T)

    assert size(0) > 0 and size(1) > 0 and size(-1) == 0 and size(4, n_in=9) == 0 and size(4, group=1) == 0


def test_binding_refuses_bad_tensors():
    x, z = torch.zeros((4, 64)), torch.zeros((4, 2, 64))
    r = object.__new__(S.Rotary)
    r.head_dim, r._device = 64, -1
    c = object.__new__(S.PagedCache)
    c.head_dim, c.n_kv_heads, c._device, c._type, c.k = 64, 2, -1, S.BF16, z
    i32 = torch.zeros(4, dtype=torch.int32)
    for fn, why in [
        (lambda: S.rope_table(64, scaling=("other", 2.0)), "other"), (lambda: S.rope_table(7), "even"), (lambda: S.Rotary(64, device="cpu"), "not a GPU"),
        (lambda: S.Rotary(64, turns=torch.zeros(5), device="cpu"), "shape"), (lambda: r.run(x, i32), "shape"), (lambda: r.run(z.double(), i32), "float64"),
        (lambda: r.run(z.transpose(0, 1).contiguous().transpose(0, 1), i32), "contiguous"), (lambda: r.run(z, i32), "not a GPU"),
        (lambda: S.PagedCache(None, z), "None"), (lambda: S.PagedCache(z, z), "pages"), (lambda: S.PagedCache(z[None], z[None]), "not a GPU"),
        (lambda: S.PagedCache(z[None], z), "not a GPU"), (lambda: c.append(z[:, :1], z, i32), "shape"), (lambda: c.append(z, z, i32), "not a GPU"),
        (lambda: c.attend(x, i32, i32, i32), "shape"), (lambda: c.attend(z.bfloat16(), i32, i32, i32), "not a GPU"),
        (lambda: S.Linear4(64, 4, None, x), "None"), (lambda: S.Linear4(48, 4, x, x), "multiples of 32"), (lambda: S.Linear4(64, 4, x, x), "float32"),
        (lambda: S.Linear4(64, 4, torch.zeros((4, 32), dtype=torch.uint8), x[:1, :4]), "not a GPU"),
        (lambda: S.Linear4(64, 4, torch.zeros((4, 32), dtype=torch.uint8), x, w2=x), "together"),
    ]:
        with pytest.raises(S.SmoeError) as err:
            fn()
        assert why in str(err.value), (why, str(err.value))
