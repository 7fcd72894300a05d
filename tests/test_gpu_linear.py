"""GPU tests of the dense product (Linear) against its plain form in 64 bits (dense_ref.py)."""
import numpy as np
import pytest
import torch

import dense_ref as D
import stratametal_amd as S
from test_gpu_ends import TYPES, close, host, normal, say

pytestmark = pytest.mark.gpu
ACTS = dict(none=S.ACT_NONE, silu=S.ACT_SILU, gelu=S.ACT_GELU, relu=S.ACT_RELU, relu2=S.ACT_RELU2, sigmoid=S.ACT_SIGMOID)


def make(seed, T, K, N, w="bf16", pair=False, bias=True, act="none", residual=None):
    t = TYPES[w]
    x = normal(seed, T, K).to(t)
    ws = [normal(seed + 1 + i, N, K, sigma=K ** -0.5).to(t) if i == 0 or pair else None for i in range(2)]
    bs = [normal(seed + 3 + i, N, sigma=0.3) if bias and (i == 0 or pair) else None for i in range(2)]
    r = None if residual is None else normal(seed + 5, T, N).to(TYPES[residual])
    return x, r, S.Linear(K, N, ws[0], bias=bs[0], w2=ws[1], bias2=bs[1], act=ACTS[act])


def check(L, x, r, act, y, y_type):
    w, w2, b, b2 = (None if t is None else host(t) for t in L.tensors)
    want, bound = D.linear(host(x), w, b, w2, b2, act, None if r is None else host(r), y_type)
    close(y, want, bound)


SIZES = [(1, 8, 1), (1, 64, 5), (1, 2048, 640), (2, 72, 33), (3, 512, 4096), (4, 40, 16), (7, 136, 129), (8, 1000, 260), (16, 2048, 512),
         (17, 64, 64), (31, 520, 100), (33, 256, 1000), (64, 64, 64), (65, 72, 63), (100, 1032, 300), (128, 512, 256),
         (129, 136, 257), (200, 264, 511), (256, 2048, 512), (300, 648, 384), (513, 200, 130), (1000, 96, 72)]


@pytest.mark.parametrize("T,K,N", SIZES)
@pytest.mark.parametrize("w,y", [("bf16", "f32"), ("fp16", "fp16"), ("bf16", "bf16")])
def test_product(T, K, N, w, y):
    say(f"case: linear T={T} K={K} N={N} {w} {y}")
    x, r, L = make(K, T, K, N, w, residual=y)
    check(L, x, r, "none", L.run(x, residual=r), y)


@pytest.mark.parametrize("T,K,N", SIZES)
@pytest.mark.parametrize("w,y", [("bf16", "bf16"), ("fp16", "f32")])
def test_gated_pair(T, K, N, w, y):
    say(f"case: linear pair T={T} K={K} N={N} {w} {y}")
    x, _, L = make(N, T, K, N, w, pair=True, act="silu", bias=N % 2 == 1)
    check(L, x, None, "silu", L.run(x, y_dtype=TYPES[y]), y)


# sizes on every tile, whole and in slices of K, odd ones and with a short last step among them (test_dense_rules.py holds
# them to that): tokens, n_in, n_out, pair, residual and y's type
TILES = [(3000, 136, 2100, True, None, "bf16"), (2999, 200, 2099, True, "f32", "f32"), (1300, 1032, 4099, True, None, "fp16"),
         (4096, 520, 4096, False, "f32", "f32"), (640, 8192, 2048, False, "bf16", "bf16"), (640, 8192, 2048, True, None, "f32"),
         (900, 8192, 500, True, "fp16", "fp16"), (1300, 1032, 4099, False, "bf16", "bf16"), (520, 5000, 777, False, None, "f32"),
         (256, 2048, 512, False, "f32", "f32"), (600, 3000, 1000, True, "bf16", "bf16"), (700, 4104, 1500, False, None, "f32"),
         (1500, 72, 1203, True, "f32", "f32"), (300, 4096, 300, True, None, "bf16"), (500, 8192, 1000, False, "f32", "f32"),
         (257, 8200, 1003, False, "f32", "f32"), (9, 8200, 1003, False, "f32", "f32"), (33, 1032, 6000, True, None, "f32"),
         (257, 2056, 1501, True, "bf16", "bf16"), (700, 4104, 1500, True, "f32", "f32"), (600, 3000, 999, False, "fp16", "fp16"),
         (257, 2048, 5001, False, "bf16", "bf16"), (300, 1024, 2001, True, None, "f32"),
         # a last tile of one row and one token
         (2817, 200, 2433, True, "f32", "f32"), (513, 8192, 2305, False, None, "bf16"), (1281, 520, 4097, True, None, "fp16")]


@pytest.mark.parametrize("i", range(len(TILES)))
@pytest.mark.parametrize("w", ["bf16", "fp16"])
def test_tiles(i, w):
    T, K, N, pair, residual, y = TILES[i]
    say(f"case: linear tiles {TILES[i]} {w}")
    act = "silu" if pair else "gelu"
    x, r, L = make(40 + i, T, K, N, w, pair=pair, act=act, residual=residual)
    check(L, x, r, act, L.run(x, residual=r, y_dtype=TYPES[y]), y)


# rows in one and in two blocks of 128 at a time, whole and short last ones, few outputs and tokens past a multiple of 16
FEW = [(T, K, N) for K in (8, 72, 128, 1016, 1032, 2048, 2056, 2568, 4104) for T, N in ((1, 17), (3, 1), (16, 77))]


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("T,K,N", FEW)
def test_few_tokens(T, K, N, pair):
    say(f"case: linear few T={T} K={K} N={N} pair={pair}")
    x, r, L = make(60 + T, T, K, N, pair=pair, act="silu", residual="f32")
    check(L, x, r, "silu", L.run(x, residual=r), "f32")


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("T", [1, 5, 40, 300])
def test_activations(act, pair, T):
    say(f"case: linear act={act} pair={pair} T={T}")
    x, r, L = make(9, T, 104, 52, pair=pair, act=act, residual="f32")
    x = (x.float() * 3).bfloat16()
    check(L, x, r, act, L.run(x, residual=r), "f32")


@pytest.mark.parametrize("T", [1, 6, 70, 300])
def test_strides_in_place_and_rows_behind(T):
    say(f"case: linear strides T={T}")
    K, N = 136, 77
    x, r, L = make(2, T, K, N, residual="bf16")
    want = L.run(x, residual=r)
    xw = torch.full((T + 3, K + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    xw[:T, 8:8 + K] = x
    yw = torch.full((T + 3, N + 9), 3.0, dtype=torch.bfloat16, device="cuda")
    yw[:T, 5:5 + N] = r
    ys = yw[:T, 5:5 + N]
    y = L.run(xw[:T, 8:8 + K], residual=ys, y=ys)
    assert torch.equal(y, want)
    assert bool((yw[T:] == 3).all()) and bool((yw[:, :5] == 3).all()) and bool((yw[:, 5 + N:] == 3).all())
    one = x[:1].expand(T, K)
    assert torch.equal(L.run(one), L.run(one.contiguous()))


@pytest.mark.parametrize("T", [2, 20, 150])
def test_one_token_reaches_no_other(T):
    """Infinities and NaN in one token's row, or past a row's end, leave the others' bits."""
    say(f"case: linear others T={T}")
    K, N = 88, 100
    x, _, L = make(4, T, K, N, pair=True, act="silu")
    want = L.run(x)
    x2 = x.clone()
    x2[1] = float("nan")
    x2[1, ::3] = float("inf")
    got = L.run(x2)
    keep = [t for t in range(T) if t != 1]
    assert torch.equal(got[keep], want[keep]) and bool(torch.isnan(got[1]).all())


def test_nan_and_inf_activations():
    say("case: linear special values")
    w = torch.zeros((4, 8), dtype=torch.bfloat16, device="cuda")
    b = torch.tensor([float("nan"), float("inf"), -200.0, 200.0], device="cuda")
    x = torch.ones((1, 8), dtype=torch.bfloat16, device="cuda")
    for act, want in (("none", b.cpu()), ("relu", torch.tensor([float("nan"), float("inf"), 0, 200.0])),
                      ("relu2", torch.tensor([float("nan"), float("inf"), 0, 40000.0])),
                      ("sigmoid", torch.tensor([float("nan"), 1, 0, 1.0])),
                      ("silu", torch.tensor([float("nan"), float("inf"), 0, 200.0])),
                      ("gelu", torch.tensor([float("nan"), float("inf"), 0, 200.0]))):
        y = S.Linear(8, 4, w, bias=b, act=ACTS[act]).run(x, y_dtype=torch.float32).cpu()[0]
        assert torch.allclose(y, want, rtol=1e-6, atol=1e-30, equal_nan=True), (act, y)


def test_same_bits_each_run():
    say("case: linear repeats")
    for T in (1, 12, 200):
        x, _, L = make(8, T, 1032, 200)
        y = L.run(x, y_dtype=torch.float32)
        for _ in range(3):
            assert torch.equal(L.run(x, y_dtype=torch.float32), y)


def test_weight_shapes():
    """Flat weights are the (n_out, n_in) ones' rows; a second weight of another shape is refused as the first one is."""
    say("case: linear weight shapes")
    x, _, L = make(70, 5, 64, 16, pair=True, act="silu")
    w, w2, b, b2 = L.tensors
    flat = S.Linear(64, 16, w.reshape(-1), bias=b, w2=w2.reshape(-1), bias2=b2, act=S.ACT_SILU)
    assert torch.equal(flat.run(x), L.run(x))
    for bad in (w2.t().contiguous(), w2.reshape(8, 128), w2[:15]):
        with pytest.raises(S.SmoeError, match="w2 has shape"):
            S.Linear(64, 16, w, w2=bad)
