"""GPU tests of the dense operators as a program uses them: a dense layer in front of the mixture-of-experts block and the load
of its router, stage by stage against the plain forms (dense_ref.py) and as one captured graph; streams, graphs side by
side, empty batches, bf16 bits, and offsets past 32 bits."""
import numpy as np
import pytest
import torch

import dense_ref as D
import stratametal_amd as S
from test_gpu_balance import check as check_balance
from test_gpu_ends import EPS, close, host, normal, say

pytestmark = pytest.mark.gpu


class Layer:
    """A dense layer (norm, SwiGLU products, norm back onto the stream) and a mixture-of-experts layer after it."""

    def __init__(self, n=256, ff=640, T=64):
        g = S.Geom(n_embd=n, n_ff=128, n_ff_shared=128, n_expert=16, top_k=4)
        v = lambda s, *shape, sigma=1.0: normal(s, *shape, sigma=sigma)  # noqa: E731
        self.pre, self.post, self.pre2 = (1 + v(i, n, sigma=0.2) for i in range(3))
        self.gate = v(3, n)
        self.ends = S.BlockEnds(n, pre=self.pre, eps=EPS)
        self.mid = S.BlockEnds(n, pre=self.pre2, post=self.post, eps=EPS, gate_act=S.GATE_SIGMOID, y_scale=2.0)
        self.last = S.BlockEnds(n, eps=EPS, res_scale=0.5)
        self.up = S.Linear(n, ff, v(4, ff, n, sigma=n ** -0.5).bfloat16(), w2=v(5, ff, n, sigma=n ** -0.5).bfloat16(), act=S.ACT_SILU)
        self.down = S.Linear(ff, n, v(6, n, ff, sigma=ff ** -0.5).bfloat16(), bias=v(7, n, sigma=0.1))
        self.router = S.Linear(n, 16, v(8, 16, n, sigma=0.1).bfloat16(), bias=v(9, 16))
        self.moe = S.MoELayer(g, S.synth_layer(g, 77), max_tokens=T)

    def __call__(self, R, mask=None):
        x = self.ends.read(R, x_dtype=torch.bfloat16)
        h = self.up.run(x)
        y = self.down.run(h, y_dtype=torch.float32)
        R1, x1 = self.mid.join(R, y, gate=self.gate)
        y1 = self.moe.forward(x1)
        R2 = self.last.write(R1, y1)
        logits = self.router.run(x1.bfloat16(), y_dtype=torch.float32)
        ids, weights = S.router_topk(logits, 4)
        load = S.router_balance(logits, ids, mask=mask, balance_coef=0.5, z_coef=0.1, grad=True)
        return dict(x=x, h=h, y=y, R1=R1, x1=x1, y1=y1, R2=R2, logits=logits, ids=ids, **load)


@pytest.mark.parametrize("T", [1, 5, 40])
def test_layer_stage_by_stage(T):
    say(f"case: dense layer T={T}")
    L = Layer()
    R = normal(20, T, 256)
    mask = torch.from_numpy(np.arange(T) % 5 != 3).cuda()
    o = L(R, mask)
    h = {k: host(t) for k, t in o.items()}
    _, _, x, ex = D.ends(host(R), None, None, host(L.pre), None, 1, 1, EPS, False, "f32", "bf16")
    close(o["x"], x, ex)
    w = lambda lin: [None if t is None else host(t) for t in lin.tensors]  # noqa: E731
    wu, wu2, _, _ = w(L.up)
    v, e = D.linear(h["x"], wu, None, wu2, None, "silu", None, "bf16")
    close(o["h"], v, e)
    wd, _, bd, _ = w(L.down)
    v, e = D.linear(h["h"], wd, bd, None, None, "none", None, "f32")
    close(o["y"], v, e)
    out, eo, x1, ex1 = D.ends(host(R), h["y"], np.broadcast_to(host(L.gate), R.shape), host(L.pre2), host(L.post), 1.0, 2.0, EPS, True,
                              "f32", "f32")
    close(o["R1"], out, eo)
    close(o["x1"], x1, ex1)
    assert torch.equal(o["y1"], L.moe.forward(o["x1"]))
    out, eo, _, _ = D.ends(h["R1"], h["y1"], None, None, None, 0.5, 1.0, EPS, False, "f32", "f32")
    close(o["R2"], out, eo)
    wr, _, br, _ = w(L.router)
    v, e = D.linear(host(o["x1"].bfloat16()), wr, br, None, None, "none", None, "f32")
    close(o["logits"], v, e)
    want, bound = D.balance(h["logits"], o["ids"].cpu().numpy(), mask.cpu().numpy(), 0.5, 0.1)
    check_balance({k: o[k] for k in ("loss", "counts", "mean_p", "dlogits", "dbias")}, want, bound)


@pytest.mark.parametrize("T", [1, 33])
def test_layer_in_a_graph(T):
    """One captured graph, replayed with other inputs and eager work between: every replay's bits are the eager call's."""
    say(f"case: dense layer graph T={T}")
    L = Layer()
    R = normal(30, T, 256)
    L(R)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = L(R)
    for i in range(4):
        R.copy_(normal(31 + i, T, 256))
        g.replay()
        torch.cuda.synchronize()
        got = {k: t.clone() for k, t in o.items()}
        want = L(R)
        for k in want:
            assert torch.equal(got[k], want[k]), (i, k)


def test_two_graphs_and_streams_share_nothing():
    """Two graphs of one sliced product and of one batch's balance replayed on two streams at once, with eager calls on a third."""
    say("case: dense graphs side by side")
    K, N, T = 8192, 128, 48
    L = S.Linear(K, N, normal(1, N, K, sigma=K ** -0.5).bfloat16())
    assert L.workspace_bytes(T) > 256  # K is sliced
    l = normal(2, 3000, 64)
    ids = torch.topk(l, 4, dim=1).indices.int()
    xs = [normal(3 + i, T, K).bfloat16() for i in range(3)]
    call = lambda x: (L.run(x, y_dtype=torch.float32), S.router_balance(l, ids, grad=True)["dbias"])  # noqa: E731
    want = [[t.clone() for t in call(x)] for x in xs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(x))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = call(xs[2])
        torch.cuda.synchronize()
        for got, w in zip([*outs, eager], want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_given_stream():
    """A call on a given stream runs behind that stream's work, its outputs and workspace that stream's."""
    say("case: dense given stream")
    L = Layer()
    R = normal(50, 40, 256)
    want, wj = L.ends.read(R), L.mid.join(R, R, gate=L.gate)
    lin, bal = L.router.run(R.bfloat16()), S.router_balance(normal(51, 40, 16), torch.zeros((40, 1), dtype=torch.int32, device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    late = torch.empty_like(R)
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(10):
            big = big @ big * 1e-3
        late.copy_(R)
    x = L.ends.read(late, stream=side)
    out, x2 = L.mid.join(late, late, gate=L.gate, stream=side)
    with torch.cuda.stream(side):
        lb = late.bfloat16()
    y = L.router.run(lb, stream=side)
    b = S.router_balance(normal(51, 40, 16), torch.zeros((40, 1), dtype=torch.int32, device="cuda"), stream=side)
    torch.cuda.synchronize()
    assert torch.equal(x, want) and torch.equal(out, wj[0]) and torch.equal(x2, wj[1]) and torch.equal(y, lin)
    assert torch.equal(b["loss"], bal["loss"])


def test_empty_batches():
    say("case: dense empty batches")
    L = Layer()
    z = torch.empty((0, 256), device="cuda")
    assert L.ends.read(z).shape == (0, 256) and L.mid.join(z, z, gate=L.gate)[1].shape == (0, 256)
    assert L.up.run(z.bfloat16()).shape == (0, 640)
    o = S.router_balance(torch.empty((0, 16), device="cuda"), torch.empty((0, 4), dtype=torch.int32, device="cuda"), grad=True)
    assert all(bool((t == 0).all()) for t in o.values()) and o["counts"].shape == (16,)


def test_bf16_bits():
    """int16 tensors are bf16 bits, as in the package's other calls."""
    say("case: dense bf16 bits")
    L = Layer()
    R = normal(60, 7, 256)
    a, b = L.ends.read(R, x_dtype=torch.int16), L.ends.read(R, x_dtype=torch.bfloat16)
    assert a.dtype == torch.int16 and torch.equal(a, b.view(torch.int16))
    w = L.down.tensors[0]
    bits = S.Linear(640, 256, w.view(torch.int16), bias=L.down.tensors[2])
    h = normal(61, 7, 640).bfloat16()
    assert torch.equal(bits.run(h.view(torch.int16)), L.down.run(h).view(torch.int16))


@pytest.mark.parametrize("T", [2, 20, 200])
def test_weights_and_rows_past_32_bits(T):
    """Weights of more than 2^32 bytes; x and y rows far apart in memory."""
    say(f"case: linear long offsets T={T}")
    K, N = 2048, 1100000
    w = torch.zeros((N, K), dtype=torch.bfloat16, device="cuda")
    w[-100:] = normal(1, 100, K, sigma=K ** -0.5).bfloat16()
    x = normal(2, T, K).bfloat16()
    y = S.Linear(K, N, w).run(x)
    assert bool((y[:, :-100] == 0).all())
    want, bound = D.linear(host(x), host(w[-100:]), None, None, None, "none", None, "bf16")
    close(y[:, -100:], want, bound)
    del w, y
    ld = 1 << 21
    xs = torch.empty((2200, ld), dtype=torch.bfloat16, device="cuda")[2200 - T:, :K]
    xs.copy_(x)
    ys = torch.empty((2200, ld), dtype=torch.bfloat16, device="cuda")[2200 - T:, 7:7 + 70]
    small = S.Linear(K, 70, normal(3, 70, K, sigma=K ** -0.5).bfloat16())
    assert torch.equal(small.run(xs, y=ys), small.run(x))


def test_balance_rows_past_32_bits():
    say("case: balance long offsets")
    T, E = 40000, 48
    wide = torch.empty((T, 1 << 15), device="cuda")
    l = normal(1, T, E)
    wide[:, 16:16 + E] = l
    ids = torch.topk(l, 2, dim=1).indices.int()
    a = S.router_balance(wide[:, 16:16 + E], ids, grad=True, z_coef=0.1)
    b = S.router_balance(l, ids, grad=True, z_coef=0.1)
    assert all(torch.equal(a[k], b[k]) for k in a)
