"""GPU tests of attention over a paged cache at the edges of what the call allows (test_gpu_attend.py holds the ordinary ranges)."""
import numpy as np
import pytest
import torch

import attention_ref as A
from test_gpu_attend import Batch
from test_gpu_ends import close, host, say

pytestmark = pytest.mark.gpu


# new tokens and lengths of one sequence, heads, key heads, and whether its keys are split: tiles of 16 rows, then of 128
NAN_CASES = [(1, 90, 4, 1, False), (1, 5000, 4, 1, True), (3, 5000, 4, 2, True), (1024, 1024, 32, 8, False), (1024, 2100, 16, 2, True)]


@pytest.mark.parametrize("n,L,H,kv,split", NAN_CASES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_that_a_query_sees(n, L, H, kv, split, D):
    """A query row with a NaN, and keys that are all NaN over whole pieces of a split or everywhere, give NaN whatever the plan; the
    other rows and heads are as they were."""
    say(f"case: attend nan n={n} L={L} H={H} kv={kv} D={D}")
    b = Batch(D + n, [n], [L], H, kv, D, 16)
    size = b.cache.workspace_bytes(H, n, 1, 16 * b.table.shape[1])
    if D == 128 or n < 100:
        assert (size > 256) == split
    clean, clean_lse = b.run()
    q = b.q.clone()
    b.q = b.q.clone()
    row, head = n // 2, H - 1
    b.q[row, head, D // 2] = float("nan")
    o, lse = b.run()
    assert bool(o[row, head].isnan().all()) and bool(lse[row, head].isnan())
    g = H // kv
    assert torch.equal(o[:, :H - g], clean[:, :H - g]) and torch.equal(lse[:, :H - g], clean_lse[:, :H - g])
    for r in {0, row - 1, row, row + 1, n - 1} & set(range(n)):
        heads = [h for h in range(H - g, H) if (r, h) != (row, head)]
        p = L - n + r + 1
        for h in heads:
            want, bound, wl, el = A.attend(host(q[r:r + 1, h:h + 1]), b.keys[0][:p, -1:], b.values[0][:p, -1:], D ** -0.5, True, 0, "bf16")
            close(o[r:r + 1, h:h + 1], want, bound)
            assert abs(float(lse[r, h]) - wl[0, 0]) <= el[0, 0]
    b.q = q
    for first, last in ((0, L - n // 2), (0, L - 1), (0, L)):  # keys of the last head's that are NaN
        for i in range(-(-last // 16)):
            b.cache.k[int(b.table[0, i]), kv - 1, :min(16, last - 16 * i)] = float("nan")
        o, lse = b.run()
        assert bool(o[:, H - g:].isnan().all()) and bool(lse[:, H - g:].isnan().all())
        assert torch.equal(o[:, :H - g], clean[:, :H - g]) and torch.equal(lse[:, :H - g], clean_lse[:, :H - g])


@pytest.mark.parametrize("n,H,kv,D", [(1, 4, 2, 64), (4, 4, 2, 128), (60, 4, 2, 256), (200, 4, 2, 64), (700, 32, 8, 128), (1500, 16, 2, 256)])
def test_widest_window(n, H, kv, D):
    """A window as wide as its type holds hides nothing, in sequences with more queries than keys too."""
    say(f"case: attend widest window n={n} H={H} kv={kv} D={D}")
    b = Batch(n, [n, n + 5, 3], [n // 2, 3, 100], H, kv, D, 16)
    want, want_lse = b.run()
    for window in (2 ** 31 - 1, 2 ** 31 - 4, 2 ** 30):
        o, lse = b.run(window=window)
        assert torch.equal(o, want) and torch.equal(lse, want_lse), window
    b.check(o, lse)


@pytest.mark.parametrize("new,lens,H,kv,D,max_len", [
    ([10, 1, 7], [100, 2 ** 31 - 1, 93], 4, 2, 64, 90), ([1, 40, 3], [300, 130, 128], 6, 2, 128, 128), ([5, 30], [80, 70], 3, 1, 256, 64),
    ([600, 300], [900, 500], 32, 8, 128, 400), ([300, 400], [650, 2 ** 31 - 1], 16, 2, 256, 400)])
@pytest.mark.parametrize("window", [0, 20, 150])
def test_positions_of_sequences_past_the_longest(new, lens, H, kv, D, max_len, window):
    """Keys past max_len are not there; the queries' positions are those of the whole sequence."""
    say(f"case: attend past the longest {new} {lens} H={H} D={D} max_len={max_len} window={window}")
    there = [min(l, max_len) for l in lens]
    b = Batch(sum(new) + D, new, there, H, kv, D, 16)
    b.lens = lens
    o, lse = b.run(max_len=max_len, window=window)
    g, at = H // kv, [0, kv - 1]
    heads = [k * g + j for k in at for j in range(g)]
    for s in range(len(new)):
        for i in range(0, new[s], max(1, new[s] // 9)):
            p, t = lens[s] - new[s] + i, int(b.start[s]) + i
            lo, hi = max(0, p - window + 1) if window else 0, min(there[s], p + 1)
            if hi <= lo:
                assert bool((o[t] == 0).all()) and bool(torch.isneginf(lse[t]).all())
                continue
            want, bound, wl, el = A.attend(host(b.q[t:t + 1, heads]), b.keys[s][lo:hi][:, at], b.values[s][lo:hi][:, at], D ** -0.5, False, 0, "bf16")
            close(o[t:t + 1, heads], want, bound)
            assert (np.abs(host(lse[t:t + 1, heads]) - wl) <= el).all()


@pytest.mark.parametrize("n,L,H,kv", [(1, 1000, 4, 1), (3, 9000, 4, 2), (1024, 1024, 32, 8), (1024, 2100, 16, 2)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_small_weights_in_fp16(n, L, H, kv, D):
    """One key far above the rest, whose weights, 2^-25.2 of its own, are below half of fp16's smallest step: all that its value of
    0 leaves is theirs.  Weights are held 2^15 (tiles of 128 rows: 2^7) times up, so at most half a step of 2^-24 over that is lost of
    each: 2^-40 (2^-32), and half a step of those that are no subnormals, which averages over nothing here: the keys are equal."""
    say(f"case: attend tails n={n} L={L} H={H} kv={kv} D={D}")
    b = Batch(1, [n], [L], H, kv, D, 16, "fp16")
    far = 17.46875  # 25.2 ln 2, a whole number of fp16's steps
    b.q = torch.zeros_like(b.q)
    b.q[..., 0] = 1.0
    b.keys[0][:], b.values[0][:] = 0, 1024
    b.keys[0][0, :, 0], b.values[0][0] = far, 0
    for c in (b.cache.k, b.cache.v):
        c.zero_()
    b.cache.v.fill_(1024)
    b.cache.k[int(b.table[0, 0]), :, 0, 0], b.cache.v[int(b.table[0, 0]), :, 0] = far, 0
    o, lse = b.run(scale=1.0)
    seen = np.arange(L - n + 1, L + 1, dtype=np.float64)
    w = np.exp(-far)
    total = 1 + (seen - 1) * w
    want = (seen - 1) * w * 1024 / total
    bound = want * 2.0 ** -11 + 2.0 ** -25 + 1024 * (seen - 1) * 2.0 ** -32 + want * (2.0 ** -11 + (L / 16 + 200) * 2.0 ** -24)
    close(o, np.broadcast_to(want[:, None, None], o.shape), np.broadcast_to(bound[:, None, None], o.shape))


@pytest.mark.parametrize("new,lens", [([1] * 6, [1, 2, 33, 100, 700, 3000]), ([1], [9000]), ([5, 20, 1], [70, 300, 2000])])
@pytest.mark.parametrize("H,kv,D", [(8, 2, 64), (4, 1, 128), (5, 1, 256), (3, 1, 80)])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_weights_of_few_rows_keep_two_parts(new, lens, H, kv, D, t):
    """Tiles of 16 rows hold a weight as two numbers of the cache's type: it is off by half a step of half a step, 2^-16 in bf16
    and less in fp16, so an output differs from the formula's by f32 arithmetic, that, and its own rounding."""
    say(f"case: attend two parts {new} {lens} H={H} kv={kv} D={D} {t}")
    b = Batch(D + len(new), new, lens, H, kv, D, 16, t)
    o, lse = b.run()
    half, tiny = {"bf16": (2.0 ** -8, 2.0 ** -134), "fp16": (2.0 ** -11, 2.0 ** -25)}[t]
    for s in range(len(new)):
        rows = slice(b.start[s], b.start[s + 1])
        q = host(b.q[rows])
        want, e, _, _ = A.attend(q, b.keys[s], b.values[s], D ** -0.5, True, 0, "f32")
        size, *_ = A.attend(q, b.keys[s], np.abs(b.values[s]), D ** -0.5, True, 0, "f32")
        close(o[rows], want, e + 2.0 ** -16 * size + (np.abs(want) + e) * half + tiny)


def least(b, args):
    """The least of five times of a call among others, in us after one untimed, and its result."""
    b.cache.attend(*args)
    us = []
    for _ in range(5):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        for _ in range(4):
            out = b.cache.attend(*args)
        end.record()
        end.synchronize()
        us.append(start.elapsed_time(end) * 250)
    return min(us), out


@pytest.mark.parametrize("n,L,H,kv,D", [(2048, 2048, 32, 8, 128), (2048, 2048, 16, 2, 256), (40, 6000, 32, 8, 128), (1, 30000, 8, 1, 64)])
def test_a_nan_score_costs_no_second_pass(n, L, H, kv, D):
    """A key of NaN that all rows see makes them NaN where they are summed: they are not done anew one after the other, which took 10 to
    400 times the call (the bound is 3, of a least of five)."""
    say(f"case: attend nan's cost n={n} L={L} H={H} D={D}")
    b = Batch(n, [n], [L], H, kv, D, 16)
    args = b.args()

    clean, _ = least(b, args)
    b.cache.k[int(b.table[0, 0]), :, 0] = float("nan")
    b.cache.v[int(b.table[0, 0]), :, 0] = float("nan")
    broken, out = least(b, args)
    say(f"{clean:.0f} us, with NaN {broken:.0f}")
    assert bool(out.isnan().all()) and broken <= 3 * clean


@pytest.mark.parametrize("n,L,H,kv,D", [(2048, 2048, 32, 8, 128), (2048, 2048, 16, 2, 256), (40, 6000, 32, 8, 128), (1, 30000, 8, 1, 64)])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_a_broken_value_costs_no_second_pass(n, L, H, kv, D, t):
    """A value of inf that all rows see, in one place of the head, makes that place inf (or NaN, with a weight of 0) as it is summed: the
    rows are not done anew one after the other, and the head's other values are as they were."""
    say(f"case: attend broken value's cost n={n} L={L} H={H} D={D} {t}")
    b = Batch(n, [n], [L], H, kv, D, 16, t)
    args = b.args()
    clean, _ = least(b, args)
    want = b.cache.attend(*args)
    b.cache.v[int(b.table[0, 0]), :, 3, 5] = float("inf")
    broken, out = least(b, args)
    say(f"{clean:.0f} us, with inf {broken:.0f}")
    assert not bool(torch.isfinite(out[3:, :, 5]).any()) if n > 3 else not bool(torch.isfinite(out[:, :, 5]).any())
    keep = [d for d in range(D) if d != 5]
    assert bool(torch.isfinite(out[..., keep]).all()) and torch.equal(out[32:, :, keep], want[32:, :, keep])
    assert broken <= 5 * clean  # (the first rows of a prompt, which do not see the key, are done anew)


@pytest.mark.parametrize("n,L,H,kv,D", [(200, 200, 4, 2, 64), (700, 900, 32, 8, 128), (300, 400, 16, 2, 256), (20, 5000, 8, 2, 128), (3, 77, 4, 1, 256)])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_broken_values_reach_only_those_that_see_them(n, L, H, kv, D, window, t):
    """Infinities in single places of the values at several keys, the last among them: a row has them where it sees the key, and
    nothing else of them."""
    say(f"case: attend broken values n={n} L={L} H={H} D={D} window={window} {t}")
    b = Batch(n + D, [n], [L], H, kv, D, 16, t)
    clean = host(b.run(window=window)[0])
    places = {L - n: 1, L - n // 2 - 1: 2, L - n // 3 - 1: 3, L - 1: 4, max(L - n - 20, 0): 5, max(L - n - 60, 0): 6}
    for key, d in places.items():
        b.cache.v[int(b.table[0, key // 16]), kv - 1, key % 16, d] = float("inf")
    o = host(b.run(window=window)[0])
    g, p = H // kv, np.arange(L - n, L)
    for d in range(D):
        sees = np.zeros(n, bool)
        for key, at in places.items():
            if at == d:
                sees |= (p >= key) & ((p - key < window) if window else True)
        got, was = o[:, H - g:, d], clean[:, H - g:, d]
        assert not np.isfinite(got[sees]).any() and np.isfinite(got[~sees]).all(), d
        assert np.array_equal(o[:, :H - g, d], clean[:, :H - g, d])
    rows = sorted({0, n // 3, n // 2, n - 1})
    lo = [max(0, p[r] - window + 1) if window else 0 for r in rows]
    for r, first in zip(rows, lo):
        want, bound, _, _ = A.attend(host(b.q[r:r + 1, H - g:]), b.keys[0][first:p[r] + 1, -1:], b.values[0][first:p[r] + 1, -1:], D ** -0.5, False, 0, t)
        fine = np.isfinite(o[r, H - g:])
        assert (np.abs(o[r, H - g:] - want[0])[fine] <= bound[0][fine]).all()


@pytest.mark.parametrize("n,L,H,kv,D", [(700, 900, 32, 8, 128), (1500, 1500, 32, 8, 64), (300, 2000, 16, 2, 256), (5, 3000, 8, 2, 128), (1, 300, 4, 1, 256)])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_largest_values(n, L, H, kv, D, t):
    """The type's largest values, one key to a place of the head, and scores that rise along the keys, so that the running top lags:
    finite, as the formula's are."""
    say(f"case: attend largest values n={n} L={L} H={H} D={D} {t}")
    b = Batch(n + D, [n], [L], H, kv, D, 16, t)
    top = float(torch.finfo(b.cache.v.dtype).max)
    rng = np.random.default_rng(D)
    for d in range(0, D, 5):
        key = int(rng.integers(0, L))
        b.cache.v[int(b.table[0, key // 16]), kv - 1, key % 16, d] = top if d % 2 else -top
        b.values[0][key, kv - 1, d] = top if d % 2 else -top
    o, _ = b.run()
    g = H // kv
    for r in sorted({0, n // 3, n // 2, n - 1}):
        p = L - n + r + 1
        want, bound, _, _ = A.attend(host(b.q[r:r + 1, H - g:]), b.keys[0][:p, -1:], b.values[0][:p, -1:], D ** -0.5, True, 0, t)
        close(o[r:r + 1, H - g:], want, bound)


@pytest.mark.parametrize("n,L,H,kv", [(1, 90, 4, 2), (3, 5000, 4, 2), (40, 300, 4, 2), (700, 900, 32, 8), (1024, 2100, 16, 2)])
@pytest.mark.parametrize("D", [24, 64, 80, 96, 128, 200, 256])
def test_keys_of_minus_infinity(n, L, H, kv, D):
    """A key that is -inf in the head's last value: a weight of 0 for queries above 0 there, NaN for those below, whatever lies between
    the head's size and the tile's."""
    say(f"case: attend keys of -inf n={n} L={L} H={H} kv={kv} D={D}")
    b = Batch(n + D, [n], [L], H, kv, D, 16)
    b.q = b.q.clone()
    b.q[..., D - 1] = b.q[..., D - 1].abs() + 0.5
    below = n // 2
    if n > 1:
        b.q[below, :, D - 1] *= -1
    gone = [L - n, max(L - n - 40, 0)]
    for key in gone:
        b.cache.k[int(b.table[0, key // 16]), :, key % 16, D - 1] = -float("inf")
    o, lse = b.run()
    if n > 1:
        assert bool(o[below].isnan().all()) and bool(lse[below].isnan().all())
    g = H // kv
    for r in sorted({0, n // 3, n - 1} - ({below} if n > 1 else set())):
        p = L - n + r + 1
        keep = [j for j in range(p) if j not in gone]
        for h in ([0, kv - 1] if keep else []):
            want, bound, wl, el = A.attend(host(b.q[r:r + 1, h * g:(h + 1) * g]), b.keys[0][keep, h:h + 1], b.values[0][keep, h:h + 1], D ** -0.5, False, 0, "bf16")
            close(o[r:r + 1, h * g:(h + 1) * g], want, bound)
            assert (np.abs(host(lse[r:r + 1, h * g:(h + 1) * g]) - wl) <= el).all()


@pytest.mark.parametrize("n,L,H,kv", [(1, 300, 4, 1), (3, 9000, 4, 2), (700, 900, 32, 8), (1024, 2100, 16, 2)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("t,size", [("fp16", 2.0 ** 8), ("fp16", 2.0 ** 9), ("fp16", 2.0 ** 10), ("bf16", 2.0 ** 9), ("bf16", 2.0 ** 11)])
def test_far_scores(n, L, H, kv, D, t, size):
    """Scores of 2^22 to 2^28, where a step of f32 is up to 16: keys that rise along the sequence by more than such a step to each, so
    that a query's weight is its last key's and those equal to it, and the answer their values' mean: off by a weight's rounding and its
    own, half a step each, and f32's sum of some hundred."""
    say(f"case: attend far scores n={n} L={L} H={H} kv={kv} D={D} {t} {size}")
    b = Batch(n + D, [n], [L], H, kv, D, 16, t)
    q = torch.zeros_like(b.q)
    q[..., :64] = size
    b.q = q
    k = np.zeros((L, D), np.float32)
    steps = size * (np.linspace(0.5, 1.0, 64 * 100)[-1 - np.arange(L)[::-1] % 6400] if L > 6400 else np.linspace(0.5, 1.0, L))
    k[:, :64] = torch.from_numpy(steps.astype(np.float32)).to(b.cache.k.dtype).float().numpy()[:, None]
    rows = torch.from_numpy(k).to(b.cache.k.dtype).cuda()
    slots = torch.from_numpy(np.concatenate([p * 16 + np.arange(16) for p in b.table[0][:-(-L // 16)]])[:L].astype(np.int64)).cuda()
    v = torch.from_numpy(b.values[0]).to(b.cache.v.dtype).cuda()
    b.cache.append(rows[:, None].expand(L, kv, D).contiguous(), v, slots)
    o, lse = b.run(scale=1.0)
    s = k.astype(np.float64)[:, 0] * size * 64
    g = H // kv
    for r in sorted({0, n // 3, n - 1}):
        p = L - n + r + 1
        w = np.exp(s[:p] - s[:p].max())  # (keys as near as rounding left them are equal)
        assert np.all((w == 1) | (w < 1e-12))
        want = np.repeat((w @ b.values[0][:p].astype(np.float64).reshape(p, -1) / w.sum()).reshape(kv, D), g, axis=0)
        bound = np.abs(want) * 2.0 ** -7 + 2.0 ** -12
        close(o[r], want, bound)
