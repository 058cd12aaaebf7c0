"""What svae_xent_bytes asks for, term by term, without a GPU."""
import ctypes

import pytest

from svae_cf_amd import _lib

MIB = 1 << 20
SIZE = {0: 4, 1: 2, 2: 2}


def asked(kind, R, V, D, grad):
    n = ctypes.c_longlong()
    _lib.call("svae_xent_bytes", 0, D, kind, R, V, D, int(grad), ctypes.byref(n))
    return n.value


def up(n, to):
    return -(-n // to) * to


def copies(kind, R, V, D, grad):
    """Weight and hidden rows in 16-bit blocks (fp32: three parts), rows of hidden twice for gradients."""
    parts = 3 if kind == 0 else 1
    return 2 * parts * up(D, 32) * (up(V, 256) + up(R, 128) * (2 if grad else 1))


def rows_and_columns(R, V):
    """Five numbers for a row, one for a column; what every array is rounded up to."""
    return 4 * (4 * up(R, 128) + up(V, 256)) + 64 * 1024


def pieces(kind, R):
    """G of two pieces, each of 512 MiB or 256 columns."""
    return 2 * max(512 * MIB, 2 * (3 if kind == 0 else 1) * up(R, 128) * 256)


SIZES = [(65, 1000, 64), (257, 131072, 1024), (2049, 17770, 150), (8192, 131072, 1024), (21800, 20000, 200), (32768, 32768, 1024), (131072, 1000000, 128),
         (131072, 1000000, 256), (1048576, 131072, 256), (1048576, 131072, 1024), (1 << 24, 4000, 64), (100, 1 << 28, 8), (3000, 500, 65536)]


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("R,V,D", SIZES)
def test_gradient_workspace(R, V, D, kind):
    """fp32 sums: one of all of dH, or 128 MiB of parts of it; 128 MiB of parts of dW's piece, twice.  The loss's statistics (eight
    bytes for a row and 256 columns) lie where G comes to."""
    statistics = 8 * up(R, 128) * (up(V, 256) // 256)
    sums = max(4 * up(R, 128) * up(D, 32), 128 * MIB) + 2 * 129 * MIB
    most = copies(kind, R, V, D, True) + rows_and_columns(R, V) + max(statistics, pieces(kind, R)) + sums
    assert asked(kind, R, V, D, True) <= most


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("R,V,D", SIZES)
def test_statistics_of_large_losses(R, V, D, kind):
    """No more than 512 MiB of the tiles' statistics at a time, and eight bytes for a row where they are taken in several goes."""
    statistics = min(8 * up(R, 128) * (up(V, 256) // 256), 512 * MIB) + 8 * up(R, 128)
    assert asked(kind, R, V, D, False) <= copies(kind, R, V, D, False) + rows_and_columns(R, V) + statistics
    sums = max(4 * up(R, 128) * up(D, 32), 128 * MIB) + 2 * 129 * MIB
    assert asked(kind, R, V, D, True) <= copies(kind, R, V, D, True) + rows_and_columns(R, V) + 8 * up(R, 128) + pieces(kind, R) + sums


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("R", [1, 16, 17, 32, 33, 64])
def test_few_rows(R, kind):
    """Statistics, a copy of hidden, the logits, 33 MiB of parts of dH; no copy of the weight."""
    for V in (1, 1000, 70000, 1 << 24):
        for D in (1, 64, 65, 260, 5000, 65536):
            if kind == 0 or R <= 32 or V * D >= 1 << 23:
                loss = 8 * up(R, 64) * -(-V // 256) + up(R, 64) * up(D, 64) * SIZE[kind] + 8 * 1024
                assert asked(kind, R, V, D, False) <= loss and asked(kind, R, V, D, True) <= loss + 4 * V * up(R, 4) + 33 * MIB
