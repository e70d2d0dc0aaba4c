"""chunk_delta where few sequences are long: their walks go in segments, joined by what each makes of a basis of its start."""
import pytest
import torch

from gla_jax_amd import chunk_delta
from tests.delta_reference import check_step, inputs, step

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("case", [
    # B, T, H, HK, DK, DV, dtype, hidden: 64 chunks and more (128 for float32) of few pairs
    (1, 4096, 1, 1, 32, 32, BF16, F32), (1, 4100, 2, 1, 128, 64, BF16, BF16), (2, 5000, 2, 2, 48, 48, BF16, F32), (1, 4097, 3, 3, 64, 128, BF16, F32),
    (1, 2081, 2, 1, 64, 64, F32, F32), (1, 2048, 1, 1, 128, 32, F32, F32), (1, 4500, 4, 2, 16, 256, BF16, F32)],
    ids=lambda c: "x".join(str(x).replace("torch.", "") for x in c))
def test_sizes(case):
    x = inputs(*case, seed=1)
    check_step(step(chunk_delta, *x), *x)


@pytest.mark.parametrize("lengths", [[0, 4200], [4200, 1], [1100, 3000], [1024, 64]])
def test_lengths(lengths):
    x = inputs(2, 4200, 2, 1, 64, 32, seed=2)
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    past = torch.arange(4200, device="cuda")[None, :] >= n[:, None]
    for t in (x[1], x[2], x[3], x[4], x[5], x[7]):
        t[past] = float("nan")                       # not read
    got = step(chunk_delta, *x, n)
    clean = [t.clone() for t in x]
    for t in (clean[1], clean[2], clean[3], clean[4], clean[5], clean[7]):
        t[past] = 0
    check_step(got, *clean, n)
    for t in (got[1], *got[3:]):
        assert not t[past].any()


@pytest.mark.parametrize("decay", ["mild", "resets", "hard"])
def test_gates(decay):
    x = inputs(1, 4096, 2, 1, 32, 32, decay=decay, beta="ends", seed=3)
    check_step(step(chunk_delta, *x), *x)


def test_runs_are_the_same_bits_and_a_graph_replays():
    x = inputs(1, 4096, 2, 1, 64, 64, seed=4)
    first = step(chunk_delta, *x)
    assert all(torch.equal(s, t) for s, t in zip(first, step(chunk_delta, *x)))
    arrays = [t.detach().clone().requires_grad_() for t in x[:6]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(chunk_delta(*arrays), arrays, x[6:])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hT, out = chunk_delta(*arrays)
        grads = torch.autograd.grad((hT, out), arrays, x[6:])
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for s, t in zip((hT, out) + grads, first))
