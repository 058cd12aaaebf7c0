"""embedding_grad(..., accumulate=True) of svae_cf_amd.ops at widths that no vector divides: small whole numbers, so every sum is exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,V,D", [(3, 2, 65535 * 64 + 1), (3, 3, 65535 * 64 + 7), (900, 7, 515), (900, 7, 1031), (500, 40, 65), (500, 40, 9), (70, 5, 3), (70, 5, 1)])
def test_each_column_is_added_once(R, V, D, dtype):
    from svae_cf_amd import ops
    g = torch.Generator(device="cuda").manual_seed(D)
    tok = torch.randint(-1, V, (R,), generator=g, device="cuda")
    if R > 500:
        tok[:400] = 2                                      # a segment of many chunks: at most 900 ones and a 5, exact in every sum
    dy = torch.randint(-1, 2, (R, D), generator=g, device="cuda").to(dtype)
    old = torch.randint(-5, 6, (V, D + 3), generator=g, device="cuda").to(dtype)
    out = old.clone()
    ops.embedding_grad(dy, tok, V, out=out[:, 2:2 + D], accumulate=True)
    want = old.double()
    here = tok >= 0
    want[:, 2:2 + D].index_add_(0, tok[here], dy[here].double())
    assert torch.equal(out, want.to(dtype))                # (rounded once)


def test_captured_with_more_tokens_than_one_workgroup_sorts():
    """A graph over 21 800 tokens, replayed on new ones between eager calls: the bits of the eager call, added to what is there."""
    from svae_cf_amd import ops
    R, V, D = 21800, 5000, 72
    g = torch.Generator(device="cuda").manual_seed(3)
    tok, dy = torch.randint(-1, V, (R,), generator=g, device="cuda"), torch.randn(R, D, generator=g, device="cuda")
    out = torch.zeros(V, D, device="cuda")
    ops.embedding_grad(dy, tok, V, out=out.clone(), accumulate=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.embedding_grad(dy, tok, V, out=out, accumulate=True)
    for _ in range(4):
        tok.copy_(torch.randint(-1, V, (R,), generator=g, device="cuda"))
        want = ops.embedding_grad(dy, tok, V, out=out.clone(), accumulate=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
