"""GPU tests of the block ends' row loop: batches of more rows than the work-groups hold, so that each takes several in turn
(test_dense_rules.py holds the sizes to that), every row against the plain form in 64 bits (dense_ref.py)."""
import numpy as np
import pytest
import torch

import dense_ref as D
import stratametal_amd as S
from test_gpu_ends import TYPES, check, make, say

pytestmark = pytest.mark.gpu

# tokens, values: every shape of the kernel, with vectors and without, work-groups with a second and with a third set of rows
ROWS = [(33000, 64), (33001, 37), (16500, 128), (16501, 99), (8300, 256), (8301, 205), (8302, 512), (8303, 301), (2100, 1024),
        (2101, 1001), (2102, 2048), (2103, 1537), (1060, 4096), (1061, 2571), (530, 8192), (531, 5001), (532, 16384), (533, 8200),
        (534, 8201)]
GATES = [("none", False), ("channel", True), ("token", True), ("token", False), ("both", True), ("both", False)]


@pytest.mark.parametrize("gate,sigmoid", GATES)
@pytest.mark.parametrize("T,n", ROWS)
def test_rows_in_turn(T, n, gate, sigmoid):
    """join, its parts, and join in place (out over R, x over y), every row."""
    types = [("f32", "bf16", "f32"), ("bf16", "f32", "bf16"), ("fp16", "fp16", "fp16")][(n + len(gate)) % 3]
    r, y, xt = types
    say(f"case: ends rows T={T} n={n} gate={gate} sigmoid={sigmoid} {types}")
    R, b, g, e = make(n, T, n, r, y, gate, res_scale=0.5, y_scale=1.5, gate_act=S.GATE_SIGMOID if sigmoid else S.GATE_NONE)
    out, x = e.join(R, b, gate=g, x_dtype=TYPES[xt])
    check(e, R, b, g, r, xt, out, x)
    assert torch.equal(e.write(R, b, gate=g), out)
    if r == y == xt:
        o2, x2 = e.join(R, b, gate=g, out=R, x=b)
        assert o2 is R and x2 is b and torch.equal(x2, x)
    else:
        o2 = e.write(R, b, gate=g, out=R)
    assert torch.equal(o2, out)


@pytest.mark.parametrize("T,n", ROWS)
def test_read_and_no_post(T, n):
    """The norm before a block alone, and a write without the norm after one (no sum meets between its rows)."""
    say(f"case: ends rows read T={T} n={n}")
    R, b, g, e = make(n + 1, T, n, "f32", "f32", "both", post=False)
    check(e, R, None, None, "f32", "bf16", None, e.read(R, x_dtype=torch.bfloat16))
    check(e, R, b, g, "f32", "f32", e.write(R, b, gate=g), None)


@pytest.mark.parametrize("T,n", [(8300, 256), (2101, 1001), (1060, 4096), (532, 16384)])
def test_rows_of_any_magnitude_in_turn(T, n):
    """Rows summed a second time, scaled, among ordinary ones of the same work-group."""
    say(f"case: ends rows magnitudes T={T} n={n}")
    R, b, g, _ = make(n + 2, T, n, "f32", "f32", "channel")
    scale = torch.ones((T, 1), device="cuda")
    scale[::3], scale[1::7], scale[5::11] = 1e30, 1e-30, 2e37
    R, b = R * scale, b * scale.flip(0)
    e = S.BlockEnds(n, post=torch.ones(n, device="cuda"), eps=0.0)
    x = e.read(R)
    check(e, R, None, None, "f32", "f32", None, x)
    # the norm after the block alone: its bound times the gate, and the few roundings beside the norm's
    zero = torch.zeros_like(R)
    _, _, wz, ez = D.ends(b.cpu().numpy(), None, None, None, None, 1, 1, 0.0, False, "f32", "f32")
    got = e.write(zero, b, gate=g).cpu().numpy().astype(np.float64)  # g y rs(y)
    wg = wz * g.cpu().numpy().astype(np.float64)
    assert (np.abs(got - wg) <= ez * np.abs(g.cpu().numpy()) + 8 * D.U * np.abs(wg) + D.TINY["f32"]).all()
