"""A captured backward pass of chunk_delta or token_logprobs beside an eager graph of the same leaves, where the autograd rules of Python run: logits whose rows or
features lie apart, and recorded calls."""
import pytest
import torch

from gla_jax_amd import chunk_delta, token_logprobs
from tests.delta_reference import inputs

pytestmark = pytest.mark.gpu
F32 = torch.float32


def shifted():
    """The next token of each position: rows of two sequences that are not one distance apart."""
    g = torch.Generator().manual_seed(1)
    x, t = torch.randn(2, 7, 300, generator=g).cuda(), torch.randint(300, (2, 7), generator=g).cuda()
    return x, lambda x: token_logprobs(x[:, :-1], t[:, 1:])[0]


def turned():
    """Features apart."""
    g = torch.Generator().manual_seed(2)
    x, t = torch.randn(300, 5, generator=g).cuda(), torch.randint(300, (5,), generator=g).cuda()
    return x, lambda x: token_logprobs(x.t(), t, 3)[0]


def traced_logprobs():
    x, _ = turned()
    t = torch.arange(5, device="cuda")
    return x, torch.jit.trace(lambda x: token_logprobs(x.t(), t)[0], (x,), check_trace=False)


def traced_delta():
    arrays = inputs(3, 40, 4, 2, 32, 32, F32, seed=3)[:6]
    return arrays[4], torch.jit.trace(lambda k: chunk_delta(*arrays[:4], k, arrays[5])[1], (arrays[4],), check_trace=False)


@pytest.mark.parametrize("projected", [False, True])
@pytest.mark.parametrize("make", [shifted, turned, traced_logprobs, traced_delta])
def test_refused_while_the_eager_graph_lives(make, projected):
    x, call = make()
    leaf = x.detach().clone().requires_grad_()

    def gradient():
        out = call(2 * leaf if projected else leaf)
        return torch.autograd.grad(out, [leaf], torch.ones_like(out))[0]
    for _ in range(3):                       # (a recorded call is compiled on its way)
        want = gradient()
    alive = call(leaf)
    with pytest.raises(RuntimeError, match="graph of the same leaves"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            gradient()
    torch.cuda.synchronize()
    assert torch.equal(gradient(), want)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gradient()
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
