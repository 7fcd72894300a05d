"""CPU tests of the bounds that attention over a paged cache and the product with 4-bit weights keep at the edges of what their
calls allow (test_gpu_attend_edges.py and test_gpu_linear4_edges.py run them)."""
import ctypes as C

import pytest
import torch

import stratametal_amd as S
from test_attention_refusals import append, attend, rope, verdict
from test_dense_refusals import EINVAL
from test_dispatch_rules import ask  # noqa: F401

INT_MAX = 2 ** 31 - 1


def test_linear4_group_sums_stay_in_32_bits(ask):  # noqa: F811
    """A group of any length has ceil(n_in / group) scales to an output, formed in 32 bits, and never none."""
    for group in (32, 96, 128, 65504, 65536, 65568, 2 ** 30, 2 ** 31 - 64, 2 ** 31 - 32):
        got, = ask([f"linear4_group({group})"])
        for n_in in (32, 64, 2080, 65536):
            assert 0 < n_in + got - 1 <= INT_MAX and (n_in + got - 1) // got == -(-n_in // group), (group, n_in)
            if group <= n_in:
                assert got == group
        assert got % 32 == 0 and (group < 65536 or got % 128 == 0)


def test_binding_refuses_numbers_past_32_bits():
    """The binding passes 32-bit numbers by their low bits: a group of 2^32 + 128 would pass the shape check and run as 128."""
    z = torch.zeros((1, 2, 64))
    w, s = torch.zeros((4, 128), dtype=torch.uint8), torch.zeros((1, 4))
    r, c = object.__new__(S.Rotary), object.__new__(S.PagedCache)
    r.head_dim, r._device = 64, -1
    c.head_dim, c.n_kv_heads, c._device, c._type, c.k, c._ref = 64, 2, -1, S.F32, z, None
    tokens = torch.zeros(1, dtype=torch.int32).expand(2 ** 31)
    many, pages = z.expand(2 ** 31, 2, 64), torch.empty((2 ** 32 + 1, 1, 1, 8), device="meta")
    for fn in (lambda: S.Linear4(256, 4, w, s, group=2 ** 32 + 128), lambda: S.Linear4(2 ** 32 + 256, 4, w, s), lambda: S.Linear4(256, 2 ** 32 + 4, w, s),
               lambda: S.Linear4(256, 4, w, s, act=2 ** 32), lambda: S.Rotary(2 ** 32 + 64, rot_dim=64, device="cpu"),
               lambda: S.Rotary(64, rot_dim=2 ** 32 + 64, turns=[0.0], device="cpu"), lambda: S.Rotary(64, layout=2 ** 32, device="cpu"),
               lambda: r.run(many, tokens), lambda: c.append(many, many, tokens), lambda: c.attend(many, tokens, tokens, tokens),
               lambda: S.PagedCache(pages, pages), lambda: c.workspace_bytes(4, 1, 1, 100, window=2 ** 32 + 5),
               lambda: c.workspace_bytes(4, 2 ** 32 + 1, 1, 100), lambda: c.workspace_bytes(2 ** 32 + 4, 1, 1, 100),
               lambda: c.workspace_bytes(4, 1, -2 ** 31 - 1, 100), lambda: c.workspace_bytes(4, 1, 1, 2 ** 40)):
        with pytest.raises(S.SmoeError) as err:
            fn()
        assert "32 bits" in str(err.value), str(err.value)


def test_attend_join_reads_its_arrays(ask):  # noqa: F811
    """The threads that join a row's groups find every one of them within the work-group's 256 places, for every head size and
    number of groups to a row; and each row has all of its groups."""
    for dim in (8, 24, 40, 64, 80, 96, 120, 128, 168, 200, 240, 256):
        per, per_row = dim // 4, 1
        while per_row <= 256 // per:
            got = ask([f"attend_join_place({i}, {per}, {per_row}).row * 1000 + attend_join_place({i}, {per}, {per_row}).group" for i in range(256)])
            rows, seen = 256 // per // per_row, set()
            for i, both in enumerate(got):
                row, group = both // 1000, both % 1000
                assert -1 <= row < rows and 0 <= group < per_row
                if row >= 0:
                    seen.add((row, group, i % per))
                    assert i - group * per + (per_row - 1) * per < 256, (dim, per_row, i)
            assert len(seen) == rows * per_row * per
            per_row *= 2


@pytest.mark.parametrize("scale", [3e38, -3e38, 2.4e38, float("inf")])
def test_attend_scale_that_leaves_f32(scale):
    """Scores travel in units of ln 2: scale times log2 e has to be a number, too."""
    verdict(attend(scale=scale), EINVAL)


def test_rope_launch_holds_its_tokens(ask):  # noqa: F811
    """A launch has at most 2^32 - 1 threads, 256 to a work-group: more tokens are refused before one starts."""
    sizes = [1, 2047, 2048, 2 ** 26 - 8, 2 ** 26 - 7, 2 ** 26, INT_MAX]
    got = ask([e for T in sizes for e in (f"rope_groups({T}) * rope_tokens({T})", f"rope_groups({T})", f"rope_fits({T})")])
    for T, held, groups, fits in zip(sizes, got[::3], got[1::3], got[2::3]):
        assert T <= held < T + 4 and bool(fits) == (256 * groups < 2 ** 32 - 256)
    for T in (2 ** 26, INT_MAX):
        verdict(rope(T=T, x=1 << 40, y=1 << 50), EINVAL)
        verdict(append(T=T, q=1 << 40, qo=1 << 42, k=1 << 44, v=1 << 46, slots=1 << 48, pos=1 << 50), EINVAL)


@pytest.mark.parametrize("args", [(64, 1e4, 1, 1e-320, 0, 0, 0), (64, 1e4, 2, 1e-320, 0, 0, 0), (64, 1e4, 3, 1e-320, 8192.0, 1, 32)])
def test_rope_table_that_leaves_64_bits(args):
    """Frequencies that are no numbers would turn every head to NaN."""
    turns, scale = (C.c_double * 32)(), C.c_float()
    verdict(S.lib().smoe_rope_table(*args, turns, C.byref(scale)), EINVAL)
