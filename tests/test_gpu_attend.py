"""GPU tests of attention over a paged cache (PagedCache.attend) against its plain form in 64 bits (attention_ref.py)."""
import numpy as np
import pytest
import torch

import attention_ref as A
import stratametal_amd as S
from test_gpu_ends import TYPES, close, host, normal, say

pytestmark = pytest.mark.gpu


class Batch:
    """Sequences of `new[b]` query rows and `lens[b]` keys on shuffled pages; spare pages and places past a sequence's end hold
    NaN."""

    def __init__(self, seed, new, lens, H, kv, D, page, t="bf16", before=0, behind=0, sigma=1.0):
        rng = np.random.default_rng(seed)
        self.new, self.lens, self.H, self.kv, self.D, self.page, self.t = new, lens, H, kv, D, page, t
        need = [-(-l // page) for l in lens]
        n_pages = sum(need) + 2
        order = rng.permutation(n_pages)
        self.table = np.full((len(lens), max(max(need), 1) + 1), -1, np.int32)
        k, v = (np.full((n_pages, kv, page, D), np.nan, np.float32) for _ in range(2))
        self.keys, self.values, at = [], [], 0
        for b, l in enumerate(lens):
            ids = order[at:at + need[b]]
            at += need[b]
            self.table[b, :need[b]] = ids
            kb, vb = (torch.from_numpy((rng.standard_normal((l, kv, D)) * s).astype(np.float32)).to(TYPES[t]).float().numpy()
                      for s in (sigma, 1.0))
            self.keys.append(kb), self.values.append(vb)
            for j in range(l):
                k[ids[j // page], :, j % page], v[ids[j // page], :, j % page] = kb[j], vb[j]
        self.cache = S.PagedCache(*(torch.from_numpy(p).cuda().to(TYPES[t]) for p in (k, v)))
        self.T = before + sum(new) + behind
        self.before, self.behind = before, behind
        self.start = np.cumsum([before] + list(new)).astype(np.int32)
        # the queries are columns of a wider matrix
        self.q = normal(seed + 1, self.T, (H + 2) * D).to(TYPES[t])[:, D:(H + 1) * D].unflatten(1, (H, D))

    def args(self):
        i32 = lambda v: torch.from_numpy(np.asarray(v, np.int32)).cuda()  # noqa: E731
        return self.q, i32(self.start), i32(self.lens), i32(self.table)

    def run(self, **kw):
        out = torch.full((self.T, self.H, self.D), 7.0, device="cuda").to(TYPES[self.t])
        o, lse = self.cache.attend(*self.args(), lse=True, out=out, **kw)
        torch.cuda.synchronize()
        return o, lse

    def check(self, o, lse, scale=None, causal=True, window=0, ends=False):
        """`ends`: the first and the last key head's queries alone."""
        scale = self.D ** -0.5 if scale is None else scale
        kv = [0, self.kv - 1] if ends else list(range(self.kv))
        g = self.H // self.kv
        heads = [i * g + j for i in kv for j in range(g)]
        for b in range(len(self.new)):
            if self.new[b] == 0:
                continue
            s = slice(self.start[b], self.start[b + 1])
            want, bound, wl, el = A.attend(host(self.q[s][:, heads]), self.keys[b][:, kv], self.values[b][:, kv], scale, causal, window, self.t)
            close(o[s][:, heads], want, bound)
            got = host(lse[s][:, heads]).astype(np.float64)
            assert np.array_equal(np.isneginf(got), np.isneginf(wl))
            live = np.isfinite(wl)
            assert (np.abs(got[live] - wl[live]) <= el[live]).all()
        rest = torch.cat([o[:self.before], o[self.T - self.behind:]] if self.behind else [o[:self.before]])
        assert bool((rest == 7).all())


HEADS = [(1, 1, 64), (8, 2, 128), (4, 4, 80), (16, 1, 256), (6, 2, 96), (14, 2, 8), (40, 2, 64), (3, 1, 200)]


@pytest.mark.parametrize("H,kv,D", HEADS)
@pytest.mark.parametrize("page", [1, 16, 24])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_single_tokens(H, kv, D, page, t):
    say(f"case: attend step H={H} kv={kv} D={D} page={page} {t}")
    lens = [1, 2, 31, 32, 33, 64, 65, 100, 257, 700]
    b = Batch(D + page, [1] * len(lens), lens, H, kv, D, page, t, behind=2)
    b.check(*b.run())


@pytest.mark.parametrize("H,kv,D", HEADS)
@pytest.mark.parametrize("page,window,causal", [(16, 0, True), (24, 0, True), (64, 37, True), (5, 1, True), (16, 0, False)])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_chunks(H, kv, D, page, window, causal, t):
    """Whole prompts, chunks over cached keys, single tokens between them, sequences without new tokens or without keys; rows
    before the first sequence and behind the last one are left."""
    say(f"case: attend chunks H={H} kv={kv} D={D} page={page} window={window} {causal} {t}")
    new, lens = [33, 1, 0, 70, 17, 130, 3, 2, 0], [33, 200, 50, 150, 17, 131, 3, 90, 0]
    b = Batch(H + D + page, new, lens, H, kv, D, page, t, before=1, behind=3)
    b.check(*b.run(window=window, causal=causal), window=window, causal=causal)


@pytest.mark.parametrize("n,L", [(1, 70), (1, 5000), (1, 20011), (4, 9000), (100, 6000), (600, 600), (129, 4099)])
@pytest.mark.parametrize("D,g", [(64, 4), (128, 8), (256, 5)])
def test_long(n, L, D, g):
    """Lengths whose keys are split over work-groups."""
    say(f"case: attend long n={n} L={L} D={D} g={g}")
    b = Batch(n + L, [n], [L], g if n < 100 else 2, 1, D, 32)
    b.check(*b.run())


@pytest.mark.parametrize("lens", [[700] * 9, [4000, 1, 130, 64, 2000, 65, 3], [1] * 70, [40, 9000], [2048] * 70])
@pytest.mark.parametrize("n,window", [(1, 0), (5, 0), (1, 300)])
@pytest.mark.parametrize("D", [64, 256])
def test_pieces_follow_the_lengths(lens, n, window, D):
    """Tables that hold far more keys than the sequences have, which settle the pieces of the split: the same answers as from
    tables of the longest's width."""
    say(f"case: attend pieces {len(lens)} sequences of up to {max(lens)} n={n} window={window} D={D}")
    b = Batch(len(lens) + n, [min(n, l) for l in lens], lens, 4, 2, D, 64)
    b.check(*b.run(window=window), window=window)
    b.table = np.concatenate([b.table, np.full((len(lens), 2048), -1, np.int32)], 1)
    b.check(*b.run(window=window), window=window)


# calls that tiles of 128 rows take (test_attention_rules.py): new tokens and lengths, heads, key heads, head size, window
MANY_NEW, MANY_LENS = [700, 1, 0, 300, 517, 2, 130], [700, 400, 50, 900, 517, 3, 1000]
MANY_HEADS = [(32, 4, 64), (32, 8, 128), (16, 2, 256), (40, 5, 80), (24, 4, 96), (64, 4, 8), (28, 4, 200)]
MANY_SPLIT = [([128], [4128], 32, 8, 128), ([32], [20032], 32, 8, 128), ([33, 30, 1, 32], [4000, 100, 2000, 3333], 32, 8, 128), ([256], [8200], 32, 4, 64),
              ([250], [4096], 16, 2, 256)]


@pytest.mark.parametrize("H,kv,D", MANY_HEADS)
@pytest.mark.parametrize("page,window,causal", [(24, 0, True), (64, 37, True), (16, 0, False)])
def test_many_rows(H, kv, D, page, window, causal):
    say(f"case: attend many rows H={H} kv={kv} D={D} page={page} window={window} {causal}")
    b = Batch(H + D + page, MANY_NEW, MANY_LENS, H, kv, D, page, "fp16" if (H + page) % 3 == 0 else "bf16", before=1, behind=3)
    b.check(*b.run(window=window, causal=causal), window=window, causal=causal, ends=True)


@pytest.mark.parametrize("new,lens,H,kv,D", MANY_SPLIT)
def test_many_rows_over_pieces_of_the_keys(new, lens, H, kv, D):
    say(f"case: attend many rows, splits {new} {lens} D={D}")
    b = Batch(D, new, lens, H, kv, D, 16)
    b.check(*b.run(), ends=True)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_rows_hidden_values_and_bad_pages(D):
    """As below for single tokens and short chunks: what a row does not see leaves it as it is, and a page outside the cache holds no
    keys."""
    say(f"case: attend many rows, hidden D={D}")
    H, kv = (16, 2) if D == 256 else (32, 8) if D == 128 else (32, 4)
    for value in (float("nan"), float("inf")):
        b = Batch(D, MANY_NEW, MANY_LENS, H, kv, D, 16)
        where = 650  # of the first sequence: its first 650 rows do not see it
        page, place = b.table[0][where // 16], where % 16
        b.cache.k[int(page), :, place] = value
        b.cache.v[int(page), :, place] = value
        o, lse = b.run()
        assert not bool(torch.isfinite(o[where:700]).all(dim=2).any())
        g, last = H // kv, kv - 1  # (the last key head's queries)
        want, bound, _, _ = A.attend(host(b.q[:where, -g:]), b.keys[0][:where, last:], b.values[0][:where, last:], D ** -0.5, True, 0, "bf16")
        close(o[:where, -g:], want, bound)
        for s in range(1, len(b.new)):
            rows = slice(b.start[s], b.start[s + 1])
            if b.new[s]:
                want, bound, _, _ = A.attend(host(b.q[rows, :g]), b.keys[s][:, :1], b.values[s][:, :1], D ** -0.5, True, 0, "bf16")
                close(o[rows, :g], want, bound)
    b = Batch(D + 1, MANY_NEW, MANY_LENS, H, kv, D, 16)
    b.table[6, 3] = b.cache.n_pages
    o, lse = b.run(causal=False)
    keep = np.ones(1000, bool)
    keep[48:64] = False
    rows = slice(b.start[6], b.start[7])
    want, bound, _, _ = A.attend(host(b.q[rows]), b.keys[6][keep], b.values[6][keep], D ** -0.5, False, 0, "bf16")
    close(o[rows], want, bound)


@pytest.mark.parametrize("n", [1, 40])
def test_window_far_from_the_start(n):
    say(f"case: attend window n={n}")
    b = Batch(3, [n, n], [9000, 300], 4, 2, 64, 16)
    b.check(*b.run(window=100), window=100)


def test_peaked_and_scaled():
    """Scores that grow all along, far apart, of either sign of the scale; a scale of 0 is a plain mean."""
    say("case: attend peaked")
    for scale in (4.0, -3.0, 0.0, 1e-3):
        b = Batch(5, [1, 30, 200], [900, 333, 700], 4, 2, 64, 16, sigma=2.0)
        for keys in b.keys:
            keys *= np.linspace(0.1, 1.0, len(keys), dtype=np.float32)[:, None, None]
        for i, ids in enumerate(b.table):
            kb = torch.from_numpy(b.keys[i]).bfloat16()
            b.keys[i] = kb.float().numpy()
            for j in range(b.lens[i]):
                b.cache.k[int(ids[j // 16]), :, j % 16] = kb[j].cuda()
        b.check(*b.run(scale=scale), scale=scale)


@pytest.mark.parametrize("n", [1, 3, 60, 200])
def test_more_queries_than_keys(n):
    """A sequence whose first queries lie before its first key (its keys were cut) sees nothing there: zeros and -inf."""
    say(f"case: attend empty rows n={n}")
    b = Batch(6, [n, n + 5], [n // 2, 0], 4, 2, 128, 16)
    o, lse = b.run()
    b.check(o, lse)
    assert bool((o[:n - n // 2] == 0).all()) and bool(torch.isneginf(lse[n:]).all())
    o, lse = b.run(causal=False)
    b.check(o, lse, causal=False)


@pytest.mark.parametrize("n", [1, 5, 90])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_hidden_values_reach_nothing(n, value):
    """NaN, infinities and the type's lowest value in keys and values that some queries do not see: theirs stay exact; those
    that see them get what the formula gives."""
    say(f"case: attend hidden n={n} {value}")
    L = 300
    bad = torch.finfo(torch.bfloat16).min if value == "lowest" else value
    for where in (L - 1, L - n, 40):
        b = Batch(7, [n], [L], 4, 2, 64, 16)
        clean, clean_lse = b.run(window=100)
        page, place = b.table[0][where // 16], where % 16
        b.cache.k[int(page), :, place] = bad
        b.cache.v[int(page), :, place] = bad
        o, lse = b.run(window=100)
        p = np.arange(L - n, L)
        sees = torch.from_numpy((p >= where) & (where > p - 100)).cuda()
        b.values[0][where], b.keys[0][where] = 0, 0
        # a tile without its usual sums may be added up in another order
        for i in np.flatnonzero(~sees.cpu().numpy()):
            want, bound, _, _ = A.attend(host(b.q[i:i + 1]), b.keys[0][:L - n + i + 1], b.values[0][:L - n + i + 1], 64 ** -0.5, True, 100, "bf16")
            close(o[i:i + 1], want, bound)
            assert bool(torch.isfinite(lse[i]).all())
        if value == "lowest" or not bool(sees.any()):
            continue
        assert not bool(torch.isfinite(o[sees]).all(dim=2).any())


def test_pages_outside_the_cache_hold_no_keys():
    say("case: attend bad pages")
    for n in (1, 2, 50):
        b = Batch(8, [n, n], [200, 64], 4, 2, 64, 16)
        for page in (-1, -2 ** 31, b.cache.n_pages, 2 ** 31 - 1):
            b2 = Batch(8, [n, n], [200, 64], 4, 2, 64, 16)
            b2.table[0, 5], b2.table[1, 0] = page, page
            o, lse = b2.run(causal=False)
            for s in range(2):
                gone = slice(80, 96) if s == 0 else slice(0, 16)
                keep = np.ones(b2.lens[s], bool)
                keep[gone] = False
                want, bound, wl, el = A.attend(host(b2.q[s * n:(s + 1) * n]), b2.keys[s][keep], b2.values[s][keep], 64 ** -0.5, False, 0, "bf16")
                close(o[s * n:(s + 1) * n], want, bound)
                assert (np.abs(host(lse[s * n:(s + 1) * n]) - wl) <= el).all()
        table = b.table.copy()
        b.table[:] = -1
        o, lse = b.run(causal=False)
        assert bool((o == 0).all()) and bool(torch.isneginf(lse).all())
        b.table = table


@pytest.mark.parametrize("n", [1, 30])
def test_keys_past_the_longest(n):
    """max_len and the table's width bound what a length on the device may ask for; a negative length is none."""
    say(f"case: attend bounds n={n}")
    b = Batch(9, [n, n, n], [100, 300, 20], 4, 2, 64, 16)
    full = b.lens
    keys = [k[:128] for k in b.keys]
    b.lens = [100, 2 ** 31 - 1, -5]
    o, lse = b.run(max_len=128, causal=False)
    for s, (k, v) in enumerate(zip(keys[:2], b.values)):
        want, bound, _, _ = A.attend(host(b.q[s * n:(s + 1) * n]), k, v[:128], 64 ** -0.5, False, 0, "bf16")
        close(o[s * n:(s + 1) * n], want, bound)
    assert bool((o[2 * n:] == 0).all()) and bool(torch.isneginf(lse[2 * n:]).all())
    b.lens = full
    o, lse = b.run(max_len=0)
    assert bool((o == 0).all()) and bool(torch.isneginf(lse).all())


def test_starts_out_of_order_stay_in_range():
    """q_start that is not ascending or not within the rows: rows of no sequence, nothing outside is read or written."""
    say("case: attend bad starts")
    b = Batch(10, [5, 6, 7], [50, 60, 70], 4, 2, 64, 16)
    for start in ([0, 5, 100, 18], [-7, 5, 11, 18], [0, 11, 5, 18], [18, 18, 18, 18], [2 ** 31 - 1, 0, 5, 9], [0, -1, -2, -3]):
        guard = torch.full((b.T + 64, b.H, b.D), 3.0, device="cuda").bfloat16()
        b.start = np.array(start, np.int64).astype(np.int32)
        b.cache.attend(*b.args(), out=guard[32:32 + b.T])
        torch.cuda.synchronize()
        assert bool((guard[:32] == 3).all()) and bool((guard[32 + b.T:] == 3).all())


def test_many_sequences():
    """More sequences than a wave looks through at once, empty ones among them."""
    say("case: attend many sequences")
    rng = np.random.default_rng(11)
    new = rng.integers(0, 3, 200)
    new[rng.random(200) < 0.3] = 0
    new[77] = 40
    lens = [int(n + rng.integers(0, 40)) for n in new]
    b = Batch(11, [int(n) for n in new], lens, 4, 2, 64, 8)
    b.check(*b.run())
    ones = Batch(12, [1] * 150, [int(v) for v in rng.integers(1, 60, 150)], 4, 2, 64, 8)
    ones.check(*ones.run())


@pytest.mark.parametrize("n", [1, 37])
def test_graphs_streams_and_runs(n):
    """The same bits in every run, in replays of a captured call whose lengths and pages change on the device, and in two
    graphs and an eager call at once."""
    say(f"case: attend graphs n={n}")
    b = Batch(13, [n, n], [5000, 900], 8, 2, 128, 16)
    args = b.args()
    call = lambda a: b.cache.attend(*a, lse=True, max_len=5000)  # noqa: E731
    want = [t.clone() for t in call(args)]
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(call(args), want))
    graphs, outs, ins = [], [], []
    for i in range(2):
        a = [t.clone() for t in args]
        a[0] = args[0]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(a))
        graphs.append(g), ins.append(a)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for lens in ([5000, 900], [n, 4000], [3333, n], [5000, 900]):
        for a in ins:
            a[2].copy_(torch.tensor(lens, dtype=torch.int32))
            a[3].copy_(torch.clamp(args[3], min=0))
        eager = [args[0], args[1], ins[0][2].clone(), ins[0][3].clone()]
        # (places past a sequence's end hold NaN in this batch: the changed lengths read only what the formula reads)
        ref = [t.clone() for t in call(eager)]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            again = call(eager)
        torch.cuda.synchronize()
        for got in (*outs, again):
            assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(got, ref))


def test_cache_past_32_bits():
    """Pages whose bytes lie past 4 GiB."""
    say("case: attend long offsets")
    n_pages, D, page = (1 << 33) // (2 * 64 * 2 * 64) + 4, 128, 64
    cache = S.PagedCache.empty(n_pages, page, 1, D)
    for n, L in ((1, 500), (70, 500)):
        ids = np.arange(n_pages - 8, n_pages)
        k, v = (normal(n + i, L, 1, D).bfloat16() for i in range(2))
        slots = torch.from_numpy(np.concatenate([i * page + np.arange(page) for i in ids])[:L].astype(np.int64)).cuda()
        cache.append(k, v, slots)
        q = normal(3, n, 4, D).bfloat16()
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        o = cache.attend(q, i32([0, n]), i32([L]), i32([ids.tolist()]))
        want, bound, _, _ = A.attend(host(q), host(k), host(v), D ** -0.5, True, 0, "bf16")
        close(o, want, bound)


def test_no_tokens_or_sequences():
    say("case: attend nothing")
    b = Batch(14, [1], [10], 4, 2, 64, 16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    assert b.cache.attend(b.q[:0], i32(2), i32(1), i32(1, 4)).shape == (0, 4, 64)
    assert b.cache.attend(b.q, i32(1), i32(0), i32(0, 4)).shape == (1, 4, 64)
    o = b.cache.attend(b.q, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), i32(1), i32(1, 0))
    assert bool((o == 0).all())
