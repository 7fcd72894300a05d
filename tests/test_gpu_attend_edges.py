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
