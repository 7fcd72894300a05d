"""GPU tests of the product with 4-bit weights at the edges of what the call allows (test_gpu_linear4.py holds the ordinary
ranges)."""
import pytest
import torch

import stratametal_amd as S
from test_gpu_ends import say
from test_gpu_linear4 import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [2 ** 16 + 32, 2 ** 30, 2 ** 31 - 32])
@pytest.mark.parametrize("T,K,N", [(1, 256, 40), (3, 2080, 33), (16, 96, 70), (40, 2080, 200), (300, 32, 50)])
@pytest.mark.parametrize("pair", [False, True])
def test_groups_longer_than_any_row(T, K, N, group, pair):
    """One scale and zero to an output, as with a group of n_in."""
    say(f"case: linear4 long groups T={T} K={K} N={N} group={group} pair={pair}")
    x, _, L, layer = make(N, T, K, N, K, pair=pair)
    two = dict(w2=layer[1]["w"], scales2=layer[1]["scales"], zeros2=layer[1]["zeros"]) if pair else {}
    y = S.Linear4(K, N, layer[0]["w"], layer[0]["scales"], zeros=layer[0]["zeros"], group=group, **two).run(x, y_dtype=torch.float32)
    check(x, None, layer, K, "none", y, "f32")
