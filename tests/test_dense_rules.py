"""The dense operators' rules of stratametal_amd/csrc/smoe_rules.hpp at sizes whose sides were measured (the figures stand
beside the rules), and their bounds; and what k_linear_big's hand-written matrix instructions need of the code round them."""
import os
import re
import shutil
import subprocess

import pytest

from test_dispatch_rules import ROOT, ask  # noqa: F401

HIPCC = "/opt/rocm/bin/hipcc"
FEW, T6432, T64, T12864, T128, T256 = range(6)


def test_linear_plan(ask):  # noqa: F811
    """tokens, n_in, n_out, pair -> a kernel and slices within a tenth of the fastest measured."""
    cases = [(1, 2048, 2048, 0, {(FEW, 1)}), (1, 4096, 4096, 0, {(FEW, 1)}), (1, 2048, 8192, 1, {(FEW, 1), (T6432, 1), (T64, 1)}),
             (12, 2048, 8192, 0, {(FEW, 1)}), (16, 8192, 2048, 0, {(FEW, 1)}), (16, 8192, 2048, 1, {(T6432, 4)}), (128, 2048, 8192, 0, {(T64, 1)}),
             (12, 4096, 4096, 1, {(FEW, 1), (T6432, 1), (T6432, 4), (T64, 1), (T12864, 4), (T128, 4)}),
             (512, 4096, 4096, 0, {(T12864, 1), (T128, 2)}), (4096, 4096, 4096, 0, {(T256, 1)}),
             (4096, 2048, 8192, 1, {(T256, 1)}), (4096, 8192, 8192, 0, {(T256, 1)})]
    got = ask([e for T, K, N, p, _ in cases for e in (f"linear_plan({T}, {K}, {N}, {p}).kind", f"linear_plan({T}, {K}, {N}, {p}).slices")])
    for i, c in enumerate(cases):
        assert (got[2 * i], got[2 * i + 1]) in c[-1], (c, got[2 * i:2 * i + 2])


def test_linear_plan_bounds(ask):  # noqa: F811
    """Any size has a kernel that takes it: the rows' kernel at most 16 tokens, no slice without steps, grids that fit."""
    sizes = [(T, K, N, p) for T in (1, 2, 16, 17, 500, 70000, 2 ** 31 - 1) for K in (8, 64, 72, 200, 8192, 65536)
             for N in (1, 63, 5003, 2 ** 24) for p in (0, 1)]
    got = ask([e for T, K, N, p in sizes for e in
               (f"linear_plan({T}, {K}, {N}, {p}).kind", f"linear_plan({T}, {K}, {N}, {p}).slices",
                f"linear_groups(linear_plan({T}, {K}, {N}, {p}), {T}, {N}, {p})")])
    for i, (T, K, N, p) in enumerate(sizes):
        kind, slices, groups = got[3 * i:3 * i + 3]
        assert kind > FEW or (T <= 16 and slices == 1)
        assert slices in (1, 2, 4, 8) and (slices == 1 or (K // 64 >= 2 * slices and groups * slices <= 1100))
        assert groups >= 1


def test_tile_cases_reach_every_kernel(ask):  # noqa: F811
    from test_gpu_linear import FEW as ROWS, SIZES, TILES
    sizes = [(T, K, N, p) for T, K, N in SIZES for p in (0, 1)] + [(T, K, N, int(p)) for T, K, N, p, _, _ in TILES]
    got = ask([e for T, K, N, p in sizes for e in (f"linear_plan({T}, {K}, {N}, {p}).kind", f"linear_plan({T}, {K}, {N}, {p}).slices > 1")])
    seen = {(k, s, bool(c[3])) for k, s, c in zip(got[::2], got[1::2], sizes)}
    assert {(FEW, 0, p) for p in (False, True)} <= seen
    kinds = ask([f"linear_plan({T}, {K}, {N}, {p}).kind" for T, K, N in ROWS for p in (0, 1)])
    blocks = ask([f"linear_few_blocks({K})" for _, K, _ in ROWS for p in (0, 1)])
    assert {(b, p) for k, b, p in zip(kinds, blocks, (0, 1) * len(ROWS)) if k == FEW} == {(1, 0), (1, 1), (2, 0), (2, 1)}
    assert {(k, 0, p) for k in (T6432, T64, T12864, T128, T256) for p in (False, True)} <= seen
    assert {k for k, s, _ in seen if s} >= {T6432, T64, T12864, T128, T256}
    # last tiles of 256 rows with one row, whole and in slices: the loads past the end of K stay out of range of its buffer
    ones = {(k, s, bool(c[3])) for k, s, c in zip(got[::2], got[1::2], sizes)
            if k == T256 and c[0] % 256 == 1 and c[2] % (128 if c[3] else 256) == 1}
    assert ones == {(T256, 0, True), (T256, 1, False)}


def test_balance_rules(ask):  # noqa: F811
    tokens = list(range(1, 700)) + [1024, 2048, 4096, 32768, 2 ** 24]
    got = ask([e for T in tokens for e in (f"balance_groups({T})", f"balance_count_groups({T})", f"balance_one({T}, 10)")])
    groups, counts, one = got[::3], got[1::3], got[2::3]
    assert groups == sorted(groups) and groups[0] == 1 and max(groups) <= 1024 and max(g * 4 - T for g, T in zip(groups, tokens)) < 4
    assert counts == sorted(counts) and counts[0] == 1 and max(counts) <= 64
    assert all(o == (T <= 64) for o, T in zip(one, tokens))


def test_balance_counts_only_where_read(ask):  # noqa: F811
    """One work-group for a few tokens counts for itself: no launch of counts beside it."""
    calls = [(T, k, g) for T in (1, 40, 47, 63, 64, 65, 300, 301, 4096) for k in (1, 8, 10, 46, 47, 63, 64) for g in ("true", "false")]
    got = ask([e for T, k, g in calls for e in (f"balance_one({T}, {k})", f"balance_counts_apart({T}, {k}, {g})")])
    for c, one, apart in zip(calls, got[::2], got[1::2]):
        assert not (one and apart), c
        assert one or bool(apart) == (c[0] * c[1] > (3000 if c[2] == "true" else 12000)), c


def test_ends_shapes(ask):  # noqa: F811
    """A row's slots hold it, and few lanes more."""
    widths = [1, 8, 64, 65, 128, 129, 256, 257, 512, 513, 1024, 1025, 2048, 2049, 4096, 4097, 8192, 8193, 16384]
    got = ask([e for n in widths for e in (f"ends_shape({n}).lanes", f"ends_shape({n}).slots", f"ends_groups(100000, {n})",
                                           f"ends_groups(5, {n})")])
    for i, n in enumerate(widths):
        lanes, slots, groups, few = got[4 * i:4 * i + 4]
        assert n <= 4 * lanes * slots and (n > 2 * lanes * slots or n <= 64), n
        assert groups * max(lanes, 256) == 256 * 1024
        assert few == (5 if lanes >= 256 else (5 * lanes + 255) // 256)


def test_row_loop_cases_reach_every_shape(ask):  # noqa: F811
    """The sizes of test_gpu_ends_rows.py make every shape of the kernel take rows in turn, with vectors and without."""
    from test_gpu_ends_rows import ROWS
    got = ask([e for T, n in ROWS for e in (f"ends_shape({n}).lanes", f"ends_shape({n}).slots", f"ends_groups({T}, {n})")])
    seen = set()
    for i, (T, n) in enumerate(ROWS):
        lanes, slots, groups = got[3 * i:3 * i + 3]
        at_once = max(256 // lanes, 1)
        sets = (T + at_once - 1) // at_once
        assert 2 * groups < sets < 3 * groups, (T, n)  # some work-groups a third set, some two
        seen.add((lanes, slots, n % 4 == 0))
    shapes = ((16, 1), (32, 1), (64, 1), (64, 2), (256, 1), (256, 2), (512, 2), (1024, 2), (1024, 4))
    assert seen == {(*s, v) for s in shapes for v in (True, False)}


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason="no hipcc")
def test_big_tile_code(tmp_path):
    """k_linear_big writes its matrix instructions itself, and the hardware waits for neither a VALU write of their operands
    nor a read of their results: in the code between the first and the last of them no sum is moved, no VALU instruction
    writes an operand's register less than 16 instructions before it is read as one, and two long waits precede the reads."""
    from stratametal_amd import build as B
    out = str(tmp_path / "linear.s")
    subprocess.run([HIPCC, *B.COMMON, "-S", "--cuda-device-only", os.path.join(B.CSRC, "smoe_linear.hip"), "-o", out], check=True,
                   capture_output=True)
    text = open(out).read()

    def regs(operand):
        r = set()
        for a, b in re.findall(r"\bv\[(\d+):(\d+)\]", operand):
            r |= set(range(int(a), int(b) + 1))
        return r | {int(a) for a in re.findall(r"\bv(\d+)\b", operand)}

    seen = 0
    for m in re.finditer(r"^(_ZN4smoe12k_linear_bigI\S+?):(.*?)\.Lfunc_end", text, re.S | re.M):
        lines = [x.strip().split(";")[0].strip() for x in m.group(2).split("\n")]
        lines = [x for x in lines if x and not x.startswith((";", "."))]
        mfma = [i for i, x in enumerate(lines) if x.startswith("v_mfma")]
        assert len(mfma) == 128 and not any("accvgpr" in x for x in lines[mfma[0]:mfma[-1]])
        loop = lines[mfma[0]:mfma[-1] + 1] * 2
        written = {}
        for i, x in enumerate(loop):
            op, _, rest = x.partition(" ")
            ops = rest.split(",")
            if op.startswith("v_mfma"):
                for r in regs(ops[1]) | regs(ops[2]):
                    assert i - written.get(r, -99) >= 16, (x, r)
            elif op.startswith("v_") and not op.startswith("v_cmp"):
                written.update({r: i for r in regs(ops[0])})
        after = lines[mfma[-1] + 1:]
        first_read = next(i for i, x in enumerate(after) if re.search(r"\ba(\[|\d)", x))
        assert sum(x.startswith("s_nop 15") for x in after[:first_read]) == 2
        seen += 1
    assert seen == 4
