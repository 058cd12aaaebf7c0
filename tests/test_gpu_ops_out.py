"""``out`` of svae_cf_amd.ops: what autograd knows of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["dropout in place", "dropout", "embedding_grad", "embedding_grad accumulate"])
def test_out_that_a_graph_keeps(how):
    """A tensor that an eager graph has kept for its backward pass and that a call writes: the backward pass refuses, as after any
    in-place operation of torch, instead of using the new values."""
    from svae_cf_amd import ops
    w = torch.ones(30, 8, device="cuda", requires_grad=True)
    kept, other, tok = torch.randn(30, 8, device="cuda"), torch.randn(30, 8, device="cuda"), torch.arange(30, device="cuda")
    loss = (w * kept).sum()
    at = kept._version
    with torch.no_grad():
        if how == "dropout in place":
            ops.dropout(kept, 0.5, 1, out=kept)
        elif how == "dropout":
            ops.dropout(other, 0.5, 1, out=kept)
        else:
            ops.embedding_grad(other, tok, 30, out=kept, accumulate="accumulate" in how)
    assert kept._version > at
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_out_in_inference_mode():
    from svae_cf_amd import ops
    with torch.inference_mode():
        x, tok = torch.randn(30, 8, device="cuda"), torch.arange(30, device="cuda")
        want = ops.dropout(x, 0.5, 1)
        assert torch.equal(ops.dropout(x, 0.5, 1, out=x), want)
        assert torch.equal(ops.embedding_grad(want, tok, 30, out=torch.empty_like(x)), want)
