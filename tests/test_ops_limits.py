"""Sizes at which a kernel's 32-bit counts would pass their end: the C entry points refuse them, before anything reaches a GPU."""
import pytest

from test_ops_refusals import P, refused

LAST = (1 << 31) - 1


@pytest.mark.parametrize("n", [(1 << 30) + 1, LAST - 8, LAST])
def test_widths(n):
    refused("sizes", "svae_lookup_fwd", P, 0, n, P, 0, P, 0, n, 2, 10, n, 1.0, None)
    refused("sizes", "svae_dropout", P, n, P, n, 0, 2, n, 0.5, 1, 0, None, None, None)


@pytest.mark.parametrize("n", [(1 << 25) + 1, 1 << 26, LAST])
def test_width_of_the_lookup_gradient(n):
    for accumulate in (0, 1):
        refused("wide", "svae_lookup_bwd", P, 0, n, P, P, 5, 10, n, 1.0, P, 0, n, accumulate, P, 1 << 62, None)


@pytest.mark.parametrize("n", [(1 << 24) + 1, LAST - 1000, LAST])
def test_rows_of_the_reduced_loss(n):
    refused("bad arguments", "svae_xent_reduce", P, P, 0, n, 10, 1, P, None)
