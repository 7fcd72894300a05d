"""GPU tests of the product with 4-bit weights (Linear4) against its plain form in 64 bits (attention_ref.py)."""
import numpy as np
import pytest
import torch

import attention_ref as A
import stratametal_amd as S
from test_gpu_ends import TYPES, close, host, normal, say
from test_gpu_linear import ACTS

pytestmark = pytest.mark.gpu


def make(seed, T, K, N, group, t="bf16", zeros=True, pair=False, bias=False, act="none", residual=None, s_type="fp16"):
    rng = np.random.default_rng(seed)
    n_groups = -(-K // group)
    layer = []
    for i in range(2 if pair else 1):
        layer.append(dict(
            w=torch.from_numpy(rng.integers(0, 256, (N, K // 2), dtype=np.uint8)).cuda(),
            scales=(torch.from_numpy(rng.uniform(-1, 1, (n_groups, N)).astype(np.float32)) * K ** -0.5 / 4).cuda().to(TYPES[s_type]),
            zeros=torch.from_numpy(rng.integers(0, 256 if i else 16, (n_groups, N), dtype=np.uint8)).cuda() if zeros else None,
            bias=normal(seed + 2 + i, N, sigma=0.3) if bias else None))
    x = normal(seed + 1, T, K).to(TYPES[t])
    r = None if residual is None else normal(seed + 5, T, N).to(TYPES[residual])
    two = dict(w2=layer[1]["w"], scales2=layer[1]["scales"], zeros2=layer[1]["zeros"], bias2=layer[1]["bias"]) if pair else {}
    L = S.Linear4(K, N, layer[0]["w"], layer[0]["scales"], zeros=layer[0]["zeros"], group=group, bias=layer[0]["bias"], act=ACTS[act], **two)
    return x, r, L, layer


def check(x, r, layer, group, act, y, y_type):
    plain = [{k: None if v is None else v.cpu().numpy() if v.dtype == torch.uint8 else host(v) for k, v in p.items()} for p in layer]
    want, bound = A.linear4(host(x), plain, group, act, None if r is None else host(r), y_type)
    close(y, want, bound)


SIZES = [(1, 32, 1, 32), (1, 64, 5, 64), (1, 2048, 640, 128), (2, 96, 33, 64), (3, 512, 4096, 32), (4, 160, 16, 160), (7, 416, 129, 128),
         (8, 992, 260, 256), (15, 1056, 47, 96), (16, 2048, 512, 128), (16, 8192, 70, 64), (17, 64, 64, 32), (31, 544, 100, 32),
         (33, 256, 1000, 256), (64, 64, 64, 64), (65, 96, 63, 32), (100, 1056, 300, 512), (128, 512, 256, 128), (129, 160, 257, 96),
         (200, 288, 511, 64), (256, 2048, 512, 128), (300, 640, 384, 32), (513, 224, 130, 1024), (1000, 96, 72, 32), (300, 4096, 200, 128),
         (1025, 512, 1029, 128), (2000, 2080, 515, 160)]


@pytest.mark.parametrize("T,K,N,group", SIZES)
@pytest.mark.parametrize("t,y", [("bf16", "f32"), ("fp16", "fp16"), ("bf16", "bf16")])
def test_product(T, K, N, group, t, y):
    say(f"case: linear4 T={T} K={K} N={N} group={group} {t} {y}")
    x, r, L, layer = make(K, T, K, N, group, t, zeros=y != "fp16", residual=y)
    check(x, r, layer, group, "none", L.run(x, residual=r), y)


@pytest.mark.parametrize("T,K,N,group", SIZES)
@pytest.mark.parametrize("t,y", [("bf16", "bf16"), ("fp16", "f32")])
def test_gated_pair(T, K, N, group, t, y):
    say(f"case: linear4 pair T={T} K={K} N={N} group={group} {t} {y}")
    x, _, L, layer = make(N, T, K, N, group, t, zeros=N % 2 == 0, pair=True, act="silu", bias=N % 2 == 1)
    check(x, None, layer, group, "silu", L.run(x, y_dtype=TYPES[y]), y)


# every tile, whole and in slices of K, groups that hold whole steps and others (test_attention_rules.py)
TILES = [(100, 1056, 300, 512, False), (100, 1056, 300, 512, True), (70, 2080, 1100, 32, False), (70, 2080, 1100, 32, True),
         (33, 2080, 2050, 64, False), (33, 2080, 1030, 128, True), (40, 2048, 2050, 32, False), (40, 2080, 1030, 96, True),
         (1025, 512, 1029, 128, False), (2000, 544, 515, 160, False), (300, 4096, 2049, 128, True), (300, 4128, 2049, 32, True),
         (4100, 512, 1030, 128, False), (4100, 544, 1030, 32, False), (1025, 512, 1029, 128, True), (2000, 544, 515, 160, True),
         (300, 4096, 2049, 128, False), (300, 4128, 2049, 32, False), (260, 8192, 2100, 64, True), (260, 4096, 4100, 32, True)]


@pytest.mark.parametrize("T,K,N,group,pair", TILES)
@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_tiles(T, K, N, group, pair, t):
    say(f"case: linear4 tile T={T} K={K} N={N} group={group} pair={pair} {t}")
    x, _, L, layer = make(T + N, T, K, N, group, t, zeros=t == "bf16", pair=pair, act="silu" if pair else "none", bias=True)
    check(x, None, layer, group, "silu" if pair else "none", L.run(x, y_dtype=torch.float32), "f32")


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("s_type", list(TYPES))
@pytest.mark.parametrize("T", [3, 90])
def test_epilogues(act, s_type, T):
    say(f"case: linear4 {act} {s_type} T={T}")
    x, r, L, layer = make(7, T, 320, 150, 64, "bf16", bias=True, act=act, residual="bf16", s_type=s_type)
    check(x, r, layer, 64, act, L.run(x, residual=r), "bf16")


@pytest.mark.parametrize("T", [1, 9, 40, 300])
def test_strided_rows(T):
    """x, y and residual as columns of wider matrices, y the residual's own rows; what lies beside them is kept."""
    say(f"case: linear4 strides T={T}")
    K, N = 256, 93
    x, r, L, layer = make(8, T, K, N, 64, "fp16", residual="f32")
    wx = torch.full((T, K + 24), float("nan"), device="cuda", dtype=torch.float16)
    wx[:, 8:8 + K] = x
    wr = torch.full((T, N + 6), 7.0, device="cuda")
    wr[:, 5:5 + N] = r
    got = L.run(wx[:, 8:8 + K], residual=wr[:, 5:5 + N], y=wr[:, 5:5 + N])
    assert torch.equal(got, L.run(x, residual=r))
    assert bool((wr[:, :5] == 7).all()) and bool((wr[:, 5 + N:] == 7).all())
    check(x, r, layer, 64, "none", got, "f32")


@pytest.mark.parametrize("T", [1, 16, 200])
def test_codes_exact(T):
    """Whole numbers all through: every code against every zero, bit for bit."""
    say(f"case: linear4 exact T={T}")
    K, N = 256, 256
    w = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(128, 1).t().contiguous()  # row o: the byte o
    zeros = (torch.arange(8 * 256, device="cuda") % 256).to(torch.uint8).view(8, 256)
    for t in (torch.bfloat16, torch.float16):
        L = S.Linear4(K, N, w, torch.ones((8, N), device="cuda"), zeros=zeros, group=32)
        x = ((torch.arange(T * K, device="cuda") * 7919 % 17) - 8).view(T, K).to(t)
        codes = torch.empty((N, K), dtype=torch.float64, device="cuda")
        codes[:, 0::2], codes[:, 1::2] = (w & 15).double(), (w >> 4).double()
        codes -= zeros.double().t().repeat_interleave(32, dim=1)
        assert torch.equal(L.run(x, y_dtype=torch.float32).double(), x.double() @ codes.t().contiguous())


@pytest.mark.parametrize("T", [1, 16, 60])
def test_weights_past_32_bits(T):
    say(f"case: linear4 long offsets T={T}")
    K, N = 8192, 1100000
    w = torch.full((N, K // 2), 0x88, dtype=torch.uint8, device="cuda")
    w[-100:] = torch.from_numpy(np.random.default_rng(1).integers(0, 256, (100, K // 2), dtype=np.uint8)).cuda()
    scales = torch.full((K // 2048, N), 0.01, device="cuda", dtype=torch.bfloat16)
    x = normal(2, T, K).bfloat16()
    y = S.Linear4(K, N, w, scales, group=2048).run(x)
    assert bool((y[:, :-100] == 0).all())
    small = S.Linear4(K, 100, w[-100:].clone(), scales[:, :100].contiguous(), group=2048)
    check(x, None, [dict(w=w[-100:], scales=scales[:, :100], zeros=None, bias=None)], 2048, "none", y[:, -100:], "bf16")
    check(x, None, [dict(w=w[-100:], scales=scales[:, :100], zeros=None, bias=None)], 2048, "none", small.run(x), "bf16")


def test_bits_empty_and_given_stream():
    say("case: linear4 forms")
    x, _, L, _ = make(9, 21, 128, 50, 64)
    want = L.run(x)
    assert torch.equal(L.run(x.view(torch.int16)), want.view(torch.int16))
    assert L.run(x[:0]).shape == (0, 50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = x * 1
    got = L.run(late, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
