"""What the operators of svae_cf_amd.ops and their C entry points refuse, before anything reaches a GPU."""
import ctypes

import pytest
import torch

from svae_cf_amd import _lib, ops


def test_no_cpu_fallback():
    t = torch.zeros(4, 4)
    tok = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: ops.embedding(t, tok), lambda: ops.embedding_grad(t[:3], tok, 4), lambda: ops.dropout(t, 0.1, 1)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_types():
    with pytest.raises(TypeError, match="float64"):
        ops.embedding(torch.zeros(4, 4, dtype=torch.float64), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(TypeError, match="tensor"):
        ops.dropout([1.0], 0.1, 1)


P = ctypes.c_void_p(256)          # a pointer that is never followed: every call here is refused before a launch


def refused(match, name, *args):
    with pytest.raises(_lib.SvaeHipError, match=match):
        _lib.call(name, *args)


def test_lookup_entry_points_refuse():
    refused("sizes", "svae_lookup_fwd", P, 0, 4, P, 0, P, 0, 4, -1, 10, 4, 1.0, None)
    refused("sizes", "svae_lookup_fwd", P, 0, 3, P, 0, P, 0, 4, 2, 10, 4, 1.0, None)
    refused("types", "svae_lookup_fwd", P, 3, 4, P, 0, P, 0, 4, 2, 10, 4, 1.0, None)
    refused("null", "svae_lookup_fwd", None, 0, 4, P, 0, P, 0, 4, 2, 10, 4, 1.0, None)
    refused("sizes", "svae_token_sort", P, 0, 5, 0, -1, P, P, P, 1 << 20, None)
    refused("workspace", "svae_token_sort", P, 0, 5000, 10, -1, P, P, P, 8, None)
    refused("null", "svae_token_sort", P, 0, 5000, 10, -1, P, P, None, 1 << 20, None)
    refused("null", "svae_token_sort", P, 0, 5, 10, -1, P, None, P, 1 << 20, None)
    refused("workspace", "svae_lookup_bwd", P, 0, 4, P, P, 5, 10, 4, 1.0, P, 0, 4, 0, P, 8, None)
    refused("sizes", "svae_lookup_bwd", P, 0, 4, P, P, 5, 10, 0, 1.0, P, 0, 4, 0, P, 1 << 20, None)
    refused("null", "svae_lookup_bwd", P, 0, 4, P, P, 5, 10, 4, 1.0, None, 0, 4, 0, P, 1 << 20, None)


def test_workspace_sizes():
    n = ctypes.c_longlong()
    _lib.call("svae_token_sort_bytes", 0, 1, ctypes.byref(n))
    assert n.value == 0
    _lib.call("svae_token_sort_bytes", 4096, 3000000, ctypes.byref(n))          # in one workgroup's LDS
    assert n.value == 0
    _lib.call("svae_token_sort_bytes", 5000, 3000000, ctypes.byref(n))          # five workgroups, two digits of 11 bits
    assert n.value == 5 * 2048 * 4 + 2 * 20224
    _lib.call("svae_lookup_bwd_bytes", 65, 10, ctypes.byref(n))
    assert n.value == 256                                                       # two chunks, two slots, 10 floats


def test_dropout_entry_point_refuses():
    refused("probability", "svae_dropout", P, 8, P, 8, 0, 2, 8, 1.5, 1, 0, None, None, None)
    refused("probability", "svae_dropout", P, 8, P, 8, 0, 2, 8, float("nan"), 1, 0, None, None, None)
    refused("2\\^-17", "svae_dropout", P, 8, P, 8, 0, 2, 8, 1e-9, 1, 0, None, None, None)
    refused("2\\^-17", "svae_dropout", P, 8, P, 8, 0, 2, 8, 1 - 1e-9, 1, 0, None, None, None)
    refused("sizes", "svae_dropout", P, 7, P, 8, 0, 2, 8, 0.5, 1, 0, None, None, None)
    refused("type", "svae_dropout", P, 8, P, 8, 5, 2, 8, 0.5, 1, 0, None, None, None)
    refused("null", "svae_dropout", P, 8, None, 8, 0, 2, 8, 0.5, 1, 0, None, None, None)


def test_xent_entry_points_refuse():
    n = ctypes.c_longlong()
    for bad in ((0, 8, 7, 4, 10, 8, 0), (0, 7, 1, 4, 10, 8, 0), (0, 8, 1, 0, 10, 8, 0), (0, 8, 1, 4, 0, 8, 1), (0, 8, 1, 4, 10, 0, 1),
                (0, 1 << 21, 1, 4, 10, 8, 0), (0, 1 << 17, 1, 4, 10, (1 << 16) + 1, 0)):
        refused("svae_xent: (type|sizes)", "svae_xent_bytes", *bad, ctypes.byref(n))
    refused("null", "svae_xent_bytes", 0, 8, 1, 4, 10, 8, 0, None)
    refused("null", "svae_xent_fwd", None, 8, P, 8, None, P, 0, 1, 4, 10, 8, P, P, P, 1 << 30, None)
    refused("ld", "svae_xent_fwd", P, 7, P, 8, None, P, 0, 1, 4, 10, 8, P, P, P, 1 << 30, None)
    refused("workspace", "svae_xent_fwd", P, 8, P, 8, None, P, 0, 1, 4, 10, 8, P, P, P, 100, None)
    refused("aligned", "svae_xent_fwd", P, 8, P, 8, None, P, 0, 1, 4, 10, 8, P, P, ctypes.c_void_p(264), 1 << 30, None)
    refused("null", "svae_xent_fwd", P, 8, P, 8, None, P, 0, 1, 4, 10, 8, None, P, P, 1 << 30, None)
    refused("null", "svae_xent_bwd", P, 8, P, 8, None, P, 0, 1, 4, 10, 8, None, P, P, 8, P, 8, None, P, 1 << 30, None)
    refused("ld", "svae_xent_bwd", P, 8, P, 8, None, P, 0, 1, 4, 10, 8, P, P, P, 7, P, 8, None, P, 1 << 30, None)
    refused("bias gradient", "svae_xent_bwd", P, 8, P, 8, P, P, 0, 1, 4, 10, 8, P, P, P, 8, None, 8, P, P, 1 << 30, None)
    refused("null", "svae_xent_fwd_bwd", P, 8, P, 8, None, P, 0, 1, 4, 10, 8, None, P, P, P, 8, P, 8, None, P, 1 << 30, None)
    refused("workspace", "svae_xent_fwd_bwd", P, 8, P, 8, None, P, 0, 1, 4, 10, 8, P, P, P, P, 8, P, 8, None, P, 1 << 10, None)
    refused("bad arguments", "svae_xent_reduce", P, P, 0, 0, 10, 1, P, None)


def test_xent_refuses_what_does_not_fit():
    t = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.linear_nll(t, t, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="reduction"):
        ops.linear_cross_entropy(t, t, torch.zeros(4, dtype=torch.int64), reduction="max")
