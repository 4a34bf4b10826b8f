"""Gradients of the routing operators where autograd does not keep the saved tensors itself: offloaded to the host, handed
through hooks, computed again under checkpointing. The kernels and their order are those of the plain run, so the gradients
are too, bit for bit."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def g():
    import gpu_kernels_b200
    return gpu_kernels_b200


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


# The first two: positions as large as a gradient, in the allocator's pool of small blocks.
SHAPES = ((256, 4, 8, 8, BF16), (512, 2, 16, 4, BF16), (64, 6, 16, 1000, F32), (3000, 3, 33, 257, BF16), (1, 1, 1, 1, F32))


def make(tokens, topk, experts, hidden, dtype):
    ids = torch.randint(-1, experts, (tokens, topk), generator=torch.Generator(device="cuda").manual_seed(tokens), device="cuda")
    x, w = normal((tokens, hidden), dtype, 1).requires_grad_(), normal((tokens, topk), F32, 2).requires_grad_()
    return ids, x, w, normal((tokens, hidden), dtype, 3)


def layer(g, ids, experts, x, w):
    """An expert layer whose experts multiply by 1.5, weighted and unweighted."""
    routes = g.sort_routes(ids, experts)
    rows = g.gather_tokens(x, routes) * 1.5
    return g.combine_tokens(rows, routes, w) + g.combine_tokens(rows, routes)


@pytest.mark.parametrize("how", ("save_on_cpu", "hooks", "checkpoint"))
@pytest.mark.parametrize("tokens,topk,experts,hidden,dtype", SHAPES)
def test_gradients_are_those_of_the_plain_run(g, tokens, topk, experts, hidden, dtype, how):
    ids, x, w, d_y = make(tokens, topk, experts, hidden, dtype)
    want = torch.autograd.grad(layer(g, ids, experts, x, w), (x, w), d_y)
    for _ in range(10):
        if how == "checkpoint":
            y = checkpoint(lambda a, b: layer(g, ids, experts, a, b), x, w, use_reentrant=False)
        elif how == "save_on_cpu":
            with torch.autograd.graph.save_on_cpu():
                y = layer(g, ids, experts, x, w)
        else:
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
                y = layer(g, ids, experts, x, w)
        got = torch.autograd.grad(y, (x, w), d_y)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
