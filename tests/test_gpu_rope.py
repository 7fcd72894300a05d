"""GPU tests of rotary positions (Rotary) and the cache's writes (PagedCache.append) against their plain form in 64 bits
(attention_ref.py)."""
import numpy as np
import pytest
import torch

import attention_ref as A
import dense_ref as D
import stratametal_amd as S
from test_gpu_ends import TYPES, close, host, normal, say

pytestmark = pytest.mark.gpu


def positions_of(T, seed, top=100000):
    return np.random.default_rng(seed).integers(0, top, T).astype(np.int32)


def want_turned(x, pos, f, scale, pairs, t):
    y, err = A.turn(x, pos, f, scale, pairs)
    return y, 1.01 * err + D.rounding(y, t)


@pytest.mark.parametrize("dim,rot", [(2, 2), (6, 4), (64, 64), (80, 80), (80, 20), (96, 24), (128, 128), (256, 64), (128, 6), (512, 512),
                                     (1024, 1022)])
@pytest.mark.parametrize("layout", [S.ROPE_HALF, S.ROPE_PAIRS])
@pytest.mark.parametrize("x,y", [("f32", "f32"), ("bf16", "fp16"), ("fp16", "bf16"), ("f32", "bf16")])
def test_turned(dim, rot, layout, x, y):
    say(f"case: rope {dim} {rot} {layout} {x} {y}")
    T, H = 5, 3
    r = S.Rotary(dim, rot_dim=rot, base=5e5, layout=layout)
    f, scale = A.table(rot, 5e5)
    v, pos = normal(dim, T, H, dim).to(TYPES[x]), positions_of(T, rot)
    got = r.run(v, torch.from_numpy(pos).cuda(), y_dtype=TYPES[y])
    want, bound = want_turned(host(v), pos, f, scale, layout == S.ROPE_PAIRS, y)
    close(got, want, bound)
    if rot < dim and x == y:
        assert torch.equal(got[..., rot:], v[..., rot:])


@pytest.mark.parametrize("scaling", [None, ("linear", 4.0), ("ntk", 8.0), ("parts", 16.0, 8192, 1.0, 32.0), ("parts", 8.0, 8192, 1.0, 4.0)])
def test_scaled_for_long_contexts(scaling):
    say(f"case: rope scaling {scaling}")
    pos = np.array([0, 1, 8191, 131071, 1000003, 2 ** 31 - 1, -5, -2 ** 31], np.int32)
    r = S.Rotary(128, base=1e4, scaling=scaling)
    f, scale = A.table(128, 1e4, scaling)
    assert abs(r.scale - scale) <= 2.0 ** -24 * 2
    v = normal(1, len(pos), 2, 128)
    want, bound = want_turned(host(v), pos, f, r.scale, False, "f32")
    close(r.run(v, torch.from_numpy(pos).cuda()), want, bound)


def test_own_table_in_place_and_back():
    """A table of the caller's; x's own rows as output; the call at -p is the transpose: it undoes a turn of scale 1."""
    say("case: rope own table")
    f = np.linspace(0.001, 1.9, 32)
    r = S.Rotary(64, turns=torch.from_numpy(f / (2 * np.pi)), scale=0.5)
    pos = positions_of(9, 3, 3000)
    p = torch.from_numpy(pos).cuda()
    x = normal(4, 9, 4, 64)
    want, bound = want_turned(host(x), pos, f, 0.5, False, "f32")
    y = r.run(x, p)
    close(y, want, bound)
    z = x.clone()
    assert r.run(z, p, y=z) is z and torch.equal(z, y)
    back, e = want_turned(host(y), -pos, f, 0.5, False, "f32")
    close(r.run(y, -p), back, e)
    # <turn(x), g> = <x, turn back(g)>
    g = normal(5, 9, 4, 64)
    lhs, rhs = (y.double() * g.double()).sum(), (x.double() * r.run(g, -p).double()).sum()
    assert abs(float(lhs - rhs)) <= 1e-4


@pytest.mark.parametrize("T", [1, 2, 77, 2049, 3000])
@pytest.mark.parametrize("kv,dim,rot,page,x,t", [(2, 256, 64, 16, "bf16", "bf16"), (3, 80, 80, 24, "f32", "fp16"), (1, 8, 6, 1, "fp16", "bf16"),
                                                (8, 128, 128, 7, "f32", "bf16")])
@pytest.mark.parametrize("layout", [S.ROPE_HALF, S.ROPE_PAIRS])
def test_append(T, kv, dim, rot, page, x, t, layout):
    """Keys, values and queries as columns of one matrix; some tokens not stored, some slots outside; other slots keep theirs."""
    say(f"case: append T={T} kv={kv} dim={dim} page={page} {x} {t} {layout}")
    H = 2 * kv
    rows = normal(T, T, (H + 2 * kv) * dim + 8).to(TYPES[x])[:, 8:]
    q, k, v = (p.unflatten(1, (-1, dim)) for p in rows.split([H * dim, kv * dim, kv * dim], dim=1))
    rng = np.random.default_rng(T + kv)
    n_pages = -(-T // page) + 2
    slots = rng.permutation(n_pages * page)[:T]
    lost = rng.random(T) < 0.2
    slots = np.where(lost, rng.choice([-1, -2 ** 62, n_pages * page, 2 ** 62], T), slots).astype(np.int64)
    pos = positions_of(T, 9)
    cache = S.PagedCache(*(normal(20 + i, n_pages, kv, page, dim).to(TYPES[t]) for i in range(2)))
    before = [host(cache.k), host(cache.v)]
    r = S.Rotary(dim, rot_dim=rot, layout=layout)
    got = cache.append(k, v, torch.from_numpy(slots).cuda(), rotary=r, positions=torch.from_numpy(pos).cuda(), q=q)
    f, scale = A.table(rot, 1e4)
    want, bound = want_turned(host(q), pos, f, scale, layout == S.ROPE_PAIRS, t)
    assert got.dtype == TYPES[t] and got.shape == (T, H, dim)
    close(got, want, bound)
    wk, ek = want_turned(host(k), pos, f, scale, layout == S.ROPE_PAIRS, t)
    wv = host(v).astype(np.float64)
    for pages, old, value, err in ((cache.k, before[0], wk, ek), (cache.v, before[1], wv, D.rounding(wv, t))):
        w, e = old.astype(np.float64), np.zeros(old.shape)
        for i in np.flatnonzero(~lost):
            w[slots[i] // page, :, slots[i] % page], e[slots[i] // page, :, slots[i] % page] = value[i], err[i]
        close(pages, w, e)


def test_append_without_turning():
    say("case: append plain")
    cache = S.PagedCache.empty(3, 5, 2, 64, dtype=torch.float16)
    k, v = normal(1, 15, 2, 64), normal(2, 15, 2, 64)
    assert cache.append(k, v, torch.arange(15, device="cuda")) is None
    assert torch.equal(cache.k.transpose(1, 2).reshape(15, 2, 64), k.half()) and torch.equal(cache.v.transpose(1, 2).reshape(15, 2, 64), v.half())
    r = S.Rotary(64)
    p = torch.arange(15, dtype=torch.int32, device="cuda")
    assert cache.append(k, v, torch.arange(15, device="cuda"), rotary=r, positions=p) is None  # keys alone
    assert torch.equal(cache.k.transpose(1, 2).reshape(15, 2, 64), r.run(k, p, y_dtype=torch.float16))


def test_append_queries_in_place():
    say("case: append in place")
    cache = S.PagedCache.empty(4, 16, 2, 128)
    r = S.Rotary(128)
    qkv = normal(1, 40, 10 * 128).bfloat16()
    q, k, v = (t.unflatten(1, (-1, 128)) for t in qkv.split([6 * 128, 2 * 128, 2 * 128], dim=1))
    p = torch.arange(40, dtype=torch.int32, device="cuda")
    want = cache.append(k, v, torch.arange(40, device="cuda"), rotary=r, positions=p, q=q)
    assert cache.append(k, v, torch.arange(40, device="cuda"), rotary=r, positions=p, q=q, q_out=q) is q
    assert torch.equal(q, want)


def test_pages_past_32_bits():
    """A slot whose bytes lie past 4 GiB of the cache."""
    say("case: append long offsets")
    n_pages = (1 << 33) // (2 * 64 * 2 * 64) + 2
    cache = S.PagedCache.empty(n_pages, 64, 1, 128)
    k, v = normal(1, 3, 1, 128).bfloat16(), normal(2, 3, 1, 128).bfloat16()
    slots = torch.tensor([n_pages * 64 - 1, (1 << 25) + 5, 7], device="cuda")
    cache.append(k, v, slots)
    for i, s in enumerate(slots.tolist()):
        assert torch.equal(cache.k[s // 64, :, s % 64], k[i]) and torch.equal(cache.v[s // 64, :, s % 64], v[i])
