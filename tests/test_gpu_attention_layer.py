"""GPU tests of a whole layer as a program runs it: norm, 4-bit products, rotary positions into the cache, attention, back onto the
stream, then the mixture-of-experts block; a prompt in chunks, then generated tokens, against the prompt at once; stage by stage
against the plain forms (attention_ref.py, dense_ref.py), and a step as one captured graph."""
import numpy as np
import pytest
import torch

import attention_ref as A
import dense_ref as D
import stratametal_amd as S
from test_gpu_ends import EPS, close, host, normal, say
from test_gpu_linear4 import make as make4

pytestmark = pytest.mark.gpu
N, H, KV, DIM, ROT, PAGE = 256, 4, 2, 64, 32, 16


class Layer:
    def __init__(self, n_pages=40, T=128):
        g = S.Geom(n_embd=N, n_ff=128, n_ff_shared=128, n_expert=16, top_k=4)
        self.pre, self.post, self.pre2 = (1 + normal(i, N, sigma=0.2) for i in range(3))
        self.ends = S.BlockEnds(N, pre=self.pre, eps=EPS)
        self.mid = S.BlockEnds(N, pre=self.pre2, post=self.post, eps=EPS)
        self.last = S.BlockEnds(N, eps=EPS)
        _, _, self.qkv, self.qkv_w = make4(1, 1, N, (H + 2 * KV) * DIM, 64)
        _, _, self.o, self.o_w = make4(2, 1, H * DIM, N, 128, zeros=False)
        self.rotary = S.Rotary(DIM, rot_dim=ROT, base=1e4, scaling=("parts", 4.0, 64, 1.0, 8.0))
        self.cache = S.PagedCache.empty(n_pages, PAGE, KV, DIM)
        self.moe = S.MoELayer(g, S.synth_layer(g, 77), max_tokens=T)

    def __call__(self, R, positions, slots, q_start, kv_len, pages, max_len=None):
        x = self.ends.read(R, x_dtype=torch.bfloat16)
        rows = self.qkv.run(x)
        q, k, v = (p.unflatten(1, (-1, DIM)) for p in rows.split([H * DIM, KV * DIM, KV * DIM], dim=1))
        qr = self.cache.append(k, v, slots, rotary=self.rotary, positions=positions, q=q)
        a = self.cache.attend(qr, q_start, kv_len, pages, max_len=max_len)
        y = self.o.run(a.flatten(1), y_dtype=torch.float32)
        R1, x1 = self.mid.join(R, y)
        R2 = self.last.write(R1, self.moe.forward(x1))
        return dict(x=x, rows=rows, q=qr, a=a, y=y, R1=R1, x1=x1, R2=R2)


def plan(new, lens, table):
    """positions, slots, q_start, kv_len and pages of a step that adds new[b] tokens to sequences, lens[b] with them."""
    pos = np.concatenate([np.arange(l - n, l) for n, l in zip(new, lens)])
    slots = np.concatenate([table[b][np.arange(l - n, l) // PAGE] * PAGE + np.arange(l - n, l) % PAGE
                            for b, (n, l) in enumerate(zip(new, lens))])
    i32 = lambda v: torch.from_numpy(np.asarray(v, np.int32)).cuda()  # noqa: E731
    return i32(pos), torch.from_numpy(slots.astype(np.int64)).cuda(), i32(np.cumsum([0] + list(new))), i32(lens), i32(table)


TABLE = np.random.default_rng(5).permutation(40)[:36].reshape(3, 12)


def test_stage_by_stage():
    say("case: attention layer stages")
    L = Layer()
    new = [21, 1, 40]
    before = [30, 100, 0]
    cached = [normal(10 + i, 130, KV, DIM).bfloat16() for i in range(2)]
    start = np.cumsum([0] + before)
    slots = np.concatenate([TABLE[b][np.arange(n) // PAGE] * PAGE + np.arange(n) % PAGE for b, n in enumerate(before)])
    L.cache.append(*cached, torch.from_numpy(slots.astype(np.int64)).cuda())
    lens = [a + b for a, b in zip(new, before)]
    args = plan(new, lens, TABLE)
    R = normal(20, sum(new), N)
    o = L(R, *args)
    _, _, x, e = D.ends(host(R), None, None, host(L.pre), None, 1, 1, EPS, False, "f32", "bf16")
    close(o["x"], x, e)
    plain = lambda w: [{k: None if v is None else v.cpu().numpy() if v.dtype == torch.uint8 else host(v) for k, v in p.items()} for p in w]  # noqa: E731
    v, e = A.linear4(host(o["x"]), plain(L.qkv_w), 64, "none", None, "bf16")
    close(o["rows"], v, e)
    rows = host(o["rows"]).reshape(sum(new), H + 2 * KV, DIM)
    f, scale = A.table(ROT, 1e4, ("parts", 4.0, 64, 1.0, 8.0))
    pos = args[0].cpu().numpy()
    q, e = A.turn(rows[:, :H], pos, f, scale, False)
    close(o["q"], q, 1.01 * e + D.rounding(q, "bf16"))
    k, e = A.turn(rows[:, H:H + KV], pos, f, scale, False)
    t0 = 0
    for b in range(3):
        n, l = new[b], lens[b]
        ids = torch.from_numpy(TABLE[b][:-(-l // PAGE)]).cuda()
        keys, values = (host(p[ids].transpose(1, 2).reshape(-1, KV, DIM)[:l]) for p in (L.cache.k, L.cache.v))
        close(torch.from_numpy(keys[l - n:]), k[t0:t0 + n], 1.01 * e[t0:t0 + n] + D.rounding(k[t0:t0 + n], "bf16"))
        assert np.array_equal(values[l - n:], rows[t0:t0 + n, H + KV:])
        assert np.array_equal(keys[:l - n], host(cached[0][start[b]:start[b + 1]]))
        want, bound, _, _ = A.attend(host(o["q"][t0:t0 + n]), keys, values, DIM ** -0.5, True, 0, "bf16")
        close(o["a"][t0:t0 + n], want, bound)
        t0 += n
    v, e = A.linear4(host(o["a"].flatten(1)), plain(L.o_w), 128, "none", None, "f32")
    close(o["y"], v, e)
    out, eo, x1, ex = D.ends(host(R), host(o["y"]), None, host(L.pre2), host(L.post), 1, 1, EPS, False, "f32", "f32")
    close(o["R1"], out, eo)
    close(o["x1"], x1, ex)
    out, eo, _, _ = D.ends(host(o["R1"]), host(L.moe.forward(o["x1"])), None, None, None, 1, 1, EPS, False, "f32", "f32")
    close(o["R2"], out, eo)


def test_step_in_a_graph():
    """One token of each of three sequences as a captured graph; positions, slots and lengths move on between its replays, with
    eager work between: every replay's bits are the eager call's, and its cache's."""
    say("case: attention layer graph")
    L, E = Layer(), Layer()
    for c in (L.cache, E.cache):
        c.k.zero_(), c.v.zero_()
    lens = np.array([3, 40, 100])
    args = [t.clone() for t in plan([1, 1, 1], lens, TABLE)]
    R = normal(30, 3, N)
    L(R, *args, max_len=12 * PAGE)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = L(R, *args, max_len=12 * PAGE)
    for i in range(5):
        R.copy_(normal(31 + i, 3, N))
        for a, b in zip(args, plan([1, 1, 1], lens + i, TABLE)):
            a.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        got = {k: t.clone() for k, t in o.items()}
        want = E(R, *args, max_len=12 * PAGE)
        for k in want:
            assert torch.equal(got[k], want[k]), (i, k)
        assert torch.equal(L.cache.k, E.cache.k) and torch.equal(L.cache.v, E.cache.v)


def test_chunks_and_steps_answer_as_the_prompt_at_once():
    """The last token's attention, the cache filled by one prompt, by chunks and by single tokens: the same keys and values bit for
    bit, attention within its bound."""
    say("case: attention layer chunks")
    T = 90
    x = normal(40, T, (H + 2 * KV) * DIM).bfloat16()
    q, k, v = (p.unflatten(1, (-1, DIM)) for p in x.split([H * DIM, KV * DIM, KV * DIM], dim=1))
    rotary = S.Rotary(DIM)
    caches, outs = [], []
    for pieces in ([T], [37, 50, 3], [1] * T):
        c = S.PagedCache.empty(40, PAGE, KV, DIM)
        at = 0
        for n in pieces:
            a = plan([n], [at + n], TABLE[:1])
            qr = c.append(k[at:at + n], v[at:at + n], a[1], rotary=rotary, positions=a[0], q=q[at:at + n])
            o = c.attend(qr, *a[2:])
            at += n
        caches.append(c), outs.append(o[-1])
    ids = torch.from_numpy(TABLE[0][:-(-T // PAGE)]).cuda()
    keys = [p[ids].transpose(1, 2).reshape(-1, KV, DIM)[:T] for p in (caches[0].k, caches[0].v)]
    for c in caches[1:]:
        assert torch.equal(c.k[ids].transpose(1, 2).reshape(-1, KV, DIM)[:T], keys[0]) and torch.equal(c.v[ids].transpose(1, 2).reshape(-1, KV, DIM)[:T], keys[1])
    want, bound, _, _ = A.attend(host(qr), host(keys[0]), host(keys[1]), DIM ** -0.5, True, 0, "bf16")
    for o in outs:
        close(o[None], want, bound)
