"""The rules of stratametal_amd/csrc/smoe_rules.hpp for attention over a paged cache and the product with 4-bit weights, at
sizes whose sides were measured (the figures stand beside the rules), and their bounds; and what the attention's hand-written
matrix instructions need of the code round them."""
import os
import random
import re
import shutil
import subprocess

import pytest

from test_dispatch_rules import ROOT, ask  # noqa: F401

HIPCC = "/opt/rocm/bin/hipcc"


def test_attend_plan(ask):  # noqa: F811
    """tokens, sequences, heads, key heads, head size, longest, window -> tiles of few rows or not, and splits, within a tenth of the
    fastest measured."""
    cases = [(1, 1, 32, 4, 128, 131072, 0, 1, range(32, 257)), (64, 64, 32, 8, 128, 8193, 0, 1, range(4, 17)), (1, 1, 16, 2, 256, 1001, 0, 1, range(6, 33)),
             (796, 6, 14, 2, 64, 2333, 500, 1, (1,)), (1024, 1, 32, 8, 128, 33792, 0, 0, range(2, 5)), (8192, 1, 32, 8, 128, 8192, 0, 0, (1,)),
             (1, 1, 32, 8, 128, 64, 0, 1, (1,)), (1, 1, 32, 8, 128, 0, 0, 1, (1,)), (8, 8, 32, 8, 128, 4001, 0, 1, range(4, 17)),
             (32, 4, 32, 8, 128, 4008, 0, 1, range(4, 17)), (32, 1, 32, 8, 128, 20032, 0, 0, range(20, 100)), (512, 1, 16, 2, 256, 512, 0, 1, (1,))]
    got = ask([e for T, B, H, kv, D, L, w, *_ in cases for e in (f"attend_plan({T}, {B}, {H}, {kv}, {D}, {L}, {w}).few",
                                                                 f"attend_plan({T}, {B}, {H}, {kv}, {D}, {L}, {w}).splits")])
    for few, splits, c in zip(got[::2], got[1::2], cases):
        assert few == c[-2] and splits in c[-1], (few, splits, c)


def test_attend_cases_reach_both_tiles(ask):  # noqa: F811
    from test_gpu_attend import HEADS, MANY_HEADS, MANY_LENS, MANY_NEW, MANY_SPLIT
    plans = lambda T, B, H, kv, D, L, w: (f"attend_plan({T}, {B}, {H}, {kv}, {D}, {L}, {w}).few", f"attend_plan({T}, {B}, {H}, {kv}, {D}, {L}, {w}).splits")  # noqa: E731
    many = [(sum(MANY_NEW) + 4, len(MANY_NEW), H, kv, D, -(-max(MANY_LENS) // page + 1) * page, w) for H, kv, D in MANY_HEADS
            for page, w in ((24, 0), (64, 37), (16, 0))]
    got = ask([e for c in many for e in plans(*c)])
    assert not any(got[::2]) and {c[4] for c in many} >= {64, 128, 256}
    split = [(sum(new), len(new), H, kv, D, -(-max(lens) // 16 + 1) * 16, 0) for new, lens, H, kv, D in MANY_SPLIT]
    got = ask([e for c in split for e in plans(*c)])
    assert not any(got[::2]) and all(s > 1 for s in got[1::2]) and {c[4] for c in split} == {64, 128, 256}
    ones = [(12, 10, H, kv, D, 720, 0) for H, kv, D in HEADS] + [(260, 9, H, kv, D, 224, 0) for H, kv, D in HEADS]
    ones += [(1, 1, 4, 1, 64, 96, 0), (1, 1, 4, 1, 128, 96, 0), (1, 1, 5, 1, 256, 96, 0)]
    got = ask([e for c in ones for e in plans(*c)])
    assert all(got[::2]) and {(c[4], s > 1) for c, s in zip(ones, got[1::2])} >= {(D, s) for D in (64, 128, 256) for s in (False, True)}


def test_attend_plan_bounds(ask):  # noqa: F811
    """The splits hold the longest sequence, a launch its work-groups, and the partial sums their place."""
    sizes = [(T, B, H, kv, D, L, w) for T, B in ((1, 1), (5, 3), (64, 64), (3, 1000), (4000, 1), (60000, 7)) for H, kv, D in ((1, 1, 8), (32, 8, 128), (128, 2, 256))
             for L in (0, 1, 63, 64, 65, 5000, 131072, 2 ** 30) for w in (0, 1, 500, 2 ** 31 - 1)]
    got = ask([e for s in sizes for e in (f"attend_plan{s}.tiles", f"attend_plan{s}.splits", f"attend_plan{s}.part_floats")])
    for i, (T, B, H, kv, D, L, w) in enumerate(sizes):
        tiles, splits, floats = got[3 * i:3 * i + 3]
        assert tiles >= 1 and splits >= 1
        assert splits == 1 or tiles * kv * splits <= 4096
        assert tiles * kv * splits < 2 ** 24
        assert splits == 1 or floats >= 2 * T * H * splits and floats % 64 == 0
        keys = min(L, w + 129) if w else L
        assert splits == 1 or (splits - 1) * 64 < keys


def test_attend_tiles_hold_any_batch(ask):  # noqa: F811
    rng = random.Random(1)
    batches = []
    for _ in range(300):
        group, B = rng.choice([1, 2, 3, 4, 5, 7, 8, 16, 40, 128, 129, 200, 300]), rng.randint(1, 12)
        batches.append(([rng.choice([0, 1, 1, 2, 5, 30, 128, 129, 700]) for _ in range(B)], group))
    got = ask([f"attend_tiles({max(sum(n), 1)}, {len(n)}, {g}, {rows})" for n, g in batches for rows in (16, 128)])
    for i, (n, g) in enumerate(batches):
        for rows, tiles in zip((16, 128), got[2 * i:2 * i + 2]):
            assert sum((x * g + rows - 1) // rows for x in n) <= tiles, (n, g)


def test_divisor(ask):  # noqa: F811
    """A quotient by a page size: exact for every number below 2^31."""
    sizes = [1, 2, 3, 5, 7, 16, 24, 31, 32, 33, 100, 255, 256, 257, 641, 4096, 4097, 65535, 2 ** 20, 2 ** 20 + 1, 2 ** 30, 2 ** 31 - 1]
    got = ask([e for d in sizes for e in (f"divisor({d}).mul", f"divisor({d}).shift")])
    rng = random.Random(2)
    for d, mul, shift in zip(sizes, got[::2], got[1::2]):
        assert mul < 2 ** 32
        for n in [0, 1, d - 1, d, d + 1, 2 ** 31 - 1, (2 ** 31 - 1) // d * d - 1, (2 ** 31 - 1) // d * d] + [rng.randrange(2 ** 31) for _ in range(2000)]:
            if 0 <= n < 2 ** 31:
                total = (n * mul >> 32) + n
                assert total < 2 ** 32 and total >> shift == n // d, (n, d)


def test_linear4_plan(ask):  # noqa: F811
    """tokens, n_in, n_out, pair -> a tile and slices within a tenth of the fastest measured."""
    cases = [(1, 2048, 8192, 1, {(1, 1)}), (4, 2048, 8192, 0, {(4, 1)}), (16, 8192, 2048, 0, {(16, 1)}), (17, 4096, 4096, 0, {(32, 4), (32, 8), (64, 8)}),
             (33, 4096, 4096, 0, {(32, 4), (64, 4), (64, 8)}), (48, 2048, 8192, 1, {(32, 1), (64, 1), (64, 2)}), (90, 4096, 4096, 0, {(64, 4), (128, 8)}),
             (128, 2048, 16384, 0, {(64, 1)}), (160, 4096, 4096, 0, {(64, 2), (128, 4), (128, 8)}), (256, 4096, 4096, 0, {(64, 2), (128, 4)}),
             (301, 2560, 5003, 0, {(64, 1), (128, 4)}), (512, 4096, 4096, 0, {(64, 1), (128, 4)}), (2048, 4096, 4096, 0, {(128, 1)})]
    got = ask([e for T, K, N, p, _ in cases for e in (f"linear4_plan({T}, {K}, {N}, {p}).tokens", f"linear4_plan({T}, {K}, {N}, {p}).slices")])
    for i, c in enumerate(cases):
        assert (got[2 * i], got[2 * i + 1]) in c[-1], (c, got[2 * i:2 * i + 2])


def test_linear4_plan_bounds(ask):  # noqa: F811
    """Any size has a kernel that takes it, no slice is without steps, and a launch that fits is the one that runs."""
    sizes = [(T, K, N, p) for T in (1, 4, 5, 16, 17, 500, 70000, 2 ** 31 - 1) for K in (32, 64, 96, 2048, 65536) for N in (1, 63, 5003, 2 ** 24)
             for p in (0, 1)]
    got = ask([e for T, K, N, p in sizes for e in
               (f"linear4_plan({T}, {K}, {N}, {p}).tokens", f"linear4_plan({T}, {K}, {N}, {p}).slices",
                f"linear4_groups(linear4_plan({T}, {K}, {N}, {p}), {T}, {N}, {p})", f"linear4_fits({T}, {K}, {N}, {p}, 64)")])
    for i, (T, K, N, p) in enumerate(sizes):
        tokens, slices, groups, fits = got[4 * i:4 * i + 4]
        assert tokens in (1, 4, 16, 32, 64, 128) and (tokens >= T or tokens >= 32)
        assert slices in (1, 2, 4, 8) and (slices == 1 or K // 64 >= 4 * slices)
        assert bool(fits) == (512 * groups < 2 ** 32 - 512), (T, K, N, p)


def test_linear4_rings_fit(ask):  # noqa: F811
    """k_linear4_few's stages in the 160 KB of LDS, and the waves' sums in them."""
    got = ask([e for pair in ("true", "false") for t in (1, 4, 16) for e in (f"8 * kLinear4Ring<{pair}, {t}> * kLinear4Stage<{pair}, {t}>",
                                                                             f"kLinear4Ring<{pair}, {t}>")])
    assert all(b <= 160 * 1024 for b in got[::2]) and all(r >= 2 for r in got[1::2])


def test_linear4_cases_reach_every_tile(ask):  # noqa: F811
    from test_gpu_linear4 import SIZES, TILES
    got = ask([e for T, K, N, _, p in TILES for e in (f"linear4_plan({T}, {K}, {N}, {int(p)}).tokens", f"linear4_plan({T}, {K}, {N}, {int(p)}).slices > 1")])
    seen = {(t, bool(s), g % 64 != 0, p) for t, s, (_, _, _, g, p) in zip(got[::2], got[1::2], TILES)}
    want = {(t, s, small, p) for t in (32, 64, 128) for s in (False, True) for small in (False, True) for p in (False, True)}
    assert want - {(32, False, small, p) for small in (False, True) for p in (False, True)} <= seen
    got = ask([e for T, K, N, _ in SIZES for p in (0, 1) for e in (f"linear4_plan({T}, {K}, {N}, {p}).tokens", f"linear4_plan({T}, {K}, {N}, {p}).slices")])
    seen = {(t, s, g % 64 != 0) for t, s, g in zip(got[::2], got[1::2], [c[3] for c in SIZES for _ in (0, 1)])}
    assert {(t, 1, small) for t in (1, 16, 32) for small in (False, True)} <= seen and any(t == 4 for t, _, _ in seen)


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason="no hipcc")
def test_wide_heads_code(tmp_path):
    """Heads of up to 256 have their sums in accumulation registers, by matrix instructions written by hand, and the hardware
    waits for neither a VALU write of their operands nor a move of their sums: eight instructions or waits lie behind each
    write, and 20 before a sum is read (an instruction of 16 passes has written it after 19)."""
    from stratametal_amd import build as B
    out = str(tmp_path / "attend.s")
    subprocess.run([HIPCC, *B.COMMON, "-S", "--cuda-device-only", os.path.join(B.CSRC, "smoe_attend.hip"), "-o", out], check=True, capture_output=True)

    def regs(operand, kind):
        r = set()
        for a, b in re.findall(rf"\b{kind}\[(\d+):(\d+)\]", operand):
            r |= set(range(int(a), int(b) + 1))
        return r | {int(a) for a in re.findall(rf"\b{kind}(\d+)\b", operand)}

    seen = 0
    for m in re.finditer(r"^(_ZN4smoe13k_attend_tileILi256\S+?):(.*?)\.Lfunc_end", open(out).read(), re.S | re.M):
        lines = [x.strip().split(";")[0].strip() for x in m.group(2).split("\n")]
        lines = [x for x in lines if x and not x.startswith((";", "."))]
        byhand = [i for i, x in enumerate(lines) if x.startswith("v_mfma_f32_32x32x16") and re.match(r"a\[", x.split(None, 1)[1])]
        assert byhand
        for i in byhand:
            ops = lines[i].split(None, 1)[1].split(",")
            operands, sums = regs(ops[1], "v") | regs(ops[2], "v"), regs(ops[0], "a")
            waits, j = 0, i - 1
            while waits < 8 and j >= 0:
                op, _, rest = lines[j].partition(" ")
                if op.startswith("v_") and not op.startswith(("v_mfma", "v_cmp")):
                    first = rest.split(",")[0]
                    assert not regs(first, "v") & operands and not regs(first, "a") & sums, (lines[j], lines[i])
                if op in ("s_branch", "s_endpgm"):
                    break
                waits += int(rest) + 1 if op == "s_nop" else 1
                j -= 1
            waits, j = 0, i + 1
            while waits < 20 and j < len(lines):
                op, _, rest = lines[j].partition(" ")
                if not op.startswith("v_mfma"):
                    assert not regs(rest, "a") & sums, (lines[i], lines[j])
                if op in ("s_branch", "s_endpgm"):
                    break
                waits += int(rest) + 1 if op == "s_nop" else 1
                j += 1
        seen += 1
    assert seen == 2
