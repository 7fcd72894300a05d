"""CPU tests of the bounds that attention over a paged cache and the product with 4-bit weights keep at the edges of what their
calls allow (test_gpu_attend_edges.py and test_gpu_linear4_edges.py run them)."""
import pytest

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
