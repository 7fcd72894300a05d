"""GPU tests of the product with 4-bit weights at the edges of what the call allows (test_gpu_linear4.py holds the ordinary
ranges)."""
import numpy as np
import pytest
import torch

import stratametal_amd as S
from test_gpu_ends import TYPES, close, host, say
from test_gpu_linear4 import check, make

pytestmark = pytest.mark.gpu


def plain(x, layer, group):
    """x W' in 64 bits, products and sums of what is not finite as they come."""
    at = np.arange(x.shape[1]) // group
    w = layer["w"].cpu().numpy()
    codes = np.empty((w.shape[0], x.shape[1]))
    codes[:, 0::2], codes[:, 1::2] = w & 15, w >> 4
    z = 8.0 if layer["zeros"] is None else layer["zeros"].cpu().numpy().astype(np.float64).T[:, at]
    with np.errstate(invalid="ignore"):
        p = x[:, None, :] * (codes - z)[None] * host(layer["scales"]).astype(np.float64).T[:, at][None]
        return p.sum(axis=2)


@pytest.mark.parametrize("T", [1, 2, 4, 5, 16, 17, 40, 300])
@pytest.mark.parametrize("K,group", [(256, 32), (256, 64), (1184, 128), (1184, 96), (2048, 2048)])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("pair", [False, True])
def test_x_not_finite(T, K, group, t, pair):
    """An infinity or a NaN in a token's values gives what the formula gives, by the weight beside it, however many tokens the call
    has, and in that token alone; so does a value whose products with the codes as they are would pass f32's largest."""
    say(f"case: linear4 not finite T={T} K={K} group={group} {t} pair={pair}")
    N = 40
    x, _, L, layer = make(K + T, T, K, N, group, t, zeros=True, pair=pair)
    layer[0]["zeros"].random_(5, 11)
    if pair:
        layer[1]["zeros"].random_(5, 11)
    clean = x.clone()
    rows = sorted({0, T // 2})
    for value in (float("inf"), -float("inf"), float("nan")) + ((1.5 * 2.0 ** 124,) if t == "bf16" else ()):
        x[:] = clean
        for r in rows:
            x[r] = 0
            x[r, (37 * r + 70) % K] = value
        y = host(L.run(x, y_dtype=torch.float32)).astype(np.float64)
        want = [plain(host(x[rows]).astype(np.float64), p, group) for p in layer]
        if pair and np.isfinite(value):
            continue  # (the pair's product would pass f32's largest)
        with np.errstate(invalid="ignore"):
            want = want[0] * want[1] if pair else want[0]
        got = y[rows]
        assert np.array_equal(np.isnan(got), np.isnan(want)), value
        inf = np.isinf(want)
        assert np.array_equal(got[inf], want[inf]) and np.array_equal(np.isinf(got), inf), value
        live = np.isfinite(want)
        assert (np.abs(got[live] - want[live]) <= 2.0 ** -20 * np.abs(want[live])).all()
        rest = [r for r in range(T) if r not in rows]
        if rest:
            check(x[rest], None, layer, group, "none", torch.from_numpy(y[rest].astype(np.float32)), "f32")


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


@pytest.mark.parametrize("T", [1, 3, 16, 40, 300])
@pytest.mark.parametrize("first", [False, True])
def test_zeros_and_bias_of_one_matrix_alone(T, first):
    """A gated pair of which one matrix has zeros and a bias of its own, the other neither."""
    say(f"case: linear4 one of two T={T} first={first}")
    K, N, group = 416, 70, 96
    x, r, _, layer = make(T, T, K, N, group, pair=True, bias=True, residual="f32")
    bare = layer[1 if first else 0]
    bare["zeros"] = bare["bias"] = None
    a, b = layer
    L = S.Linear4(K, N, a["w"], a["scales"], zeros=a["zeros"], group=group, bias=a["bias"], w2=b["w"], scales2=b["scales"], zeros2=b["zeros"],
                  bias2=b["bias"], act=S.ACT_SILU)
    check(x, r, layer, group, "silu", L.run(x, residual=r), "f32")
