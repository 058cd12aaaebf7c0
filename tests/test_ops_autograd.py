"""How the operators of svae_cf_amd.ops stand to autograd's forward mode, before anything reaches a GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from svae_cf_amd import ops

TOKENS = torch.zeros(3, dtype=torch.int64)
CALLS = [lambda x, y: ops.embedding(x, TOKENS), lambda x, y: ops.embedding_grad(x, TOKENS, 3, out=y, accumulate=True), lambda x, y: ops.dropout(x, 0.5, 1),
         lambda x, y: ops.linear_nll(x, y, TOKENS), lambda x, y: ops.linear_nll_grad(x, y, TOKENS, torch.ones(3)), lambda x, y: ops.linear_cross_entropy(x, y, TOKENS),
         lambda x, y: ops.linear_cross_entropy(y, x, TOKENS), lambda x, y: ops.linear_cross_entropy(y, y, TOKENS, x[:, 0])]


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("call", CALLS)
def test_tangents_are_refused(call, grad):
    """(before these tensors are refused for being on the CPU)"""
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        x = forward_ad.make_dual(torch.ones(3, 8), torch.ones(3, 8))
        with pytest.raises(NotImplementedError, match="tangent"):
            call(x, torch.ones(3, 8))


def test_plain_tensors_in_a_dual_level():
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.embedding(torch.ones(3, 8), TOKENS)
