"""chunk_delta, delta_step and token_logprobs where places pass 32 bits, and two calls at once: the same bits as compact arrays give, and one call
after the other."""
import math

import pytest
import torch

from gla_jax_amd import chunk_delta, delta_step, token_logprobs
from tests.delta_reference import inputs, step
from tests.test_gpu_logprobs import close, exact, off

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def far(x, apart):
    """A copy of x [2,...] whose two rows begin `apart` elements from each other."""
    buffer = torch.empty(apart + x[0].numel(), dtype=x.dtype, device=x.device)
    return buffer.as_strided(x.shape, (apart,) + x[0].contiguous().stride()).copy_(x)


def test_sequences_that_lie_far_apart():
    h0, a, b, v, k, q, dh, do = inputs(2, 200, 4, 2, 64, 32, seed=1)
    want = step(chunk_delta, h0, a, b, v, k, q, dh, do)
    apart = 2 ** 31 + 64
    got = step(chunk_delta, h0, a, b, far(v, apart), far(k, apart), far(q, apart), dh, do)
    assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_rows_of_tokens_that_lie_far_apart():
    """2^23 - 64 elements from one token to the next: a chunk spans 2^29, a sequence more than 2^31."""
    h0, a, b, v, k, q, _, _ = inputs(1, 300, 2, 2, 32, 32, seed=2)
    st = 2 ** 23 - 64
    buffer = torch.zeros(300 * st, dtype=BF16, device="cuda")
    cut = [buffer[at:].as_strided((1, 300, 2, 32), (0, st, 32, 1)).copy_(x) for at, x in ((0, q), (64, k), (128, v))]
    with torch.no_grad():
        want, got = chunk_delta(h0, a, b, v, k, q), chunk_delta(h0, a, b, cut[2], cut[1], cut[0])
    assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_a_pool_of_more_states_than_32_bits_count():
    h0, a, b, v, k, q, _, _ = inputs(3, 1, 32, 4, 128, 128, seed=3)
    a, b, v, k, q = (x[:, 0] for x in (a, b, v, k, q))
    N = 2 ** 31 // (32 * 128 * 128) + 5
    pool = torch.empty(N, 32, 128, 128, device="cuda")
    slots = torch.tensor([N - 1, 0, N - 3], device="cuda")
    pool[slots] = h0
    want_states = h0.clone()
    want = delta_step(want_states, a, b, v, k, q)
    got = delta_step(pool, a, b, v, k, q, slots=slots)
    assert torch.equal(want, got) and torch.equal(pool[slots], want_states)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_of_logits_that_lie_far_apart(dtype):
    x = torch.randn(2, 5001, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).to(dtype)
    t = torch.tensor([5000, 17], device="cuda")
    g = torch.ones(2, device="cuda")

    apart = 2 ** 31 + (8 if dtype == BF16 else 4)
    leaf = far(x, apart).detach().requires_grad_()
    found = token_logprobs(leaf, t, 7)
    d, = torch.autograd.grad(found[:2], [leaf], (g, g))
    # (rows that begin elsewhere within 16 bytes are summed in another order: against 64 bits, by the tolerances of test_gpu_logprobs.py)
    want = exact(x, t, g, g)
    close(found[0], want[0], off(want[0], 5001))
    close(found[1], want[1], 2 * off(want[1], 5001))
    assert torch.equal(found[3], x.float().sort(dim=-1, descending=True, stable=True)[1][:, :7])
    close(found[2], want[3].gather(-1, found[3]), off(want[3].gather(-1, found[3]), 5001))
    factor = 2 + want[3].abs().amax() + math.log(5001)
    close(d, want[2], 2 * off(want[3], 5001) * factor * want[3].exp() + (2.0 ** -8 if dtype == BF16 else 2.0 ** -22) * want[2].abs())


@pytest.mark.parametrize("T", [200, 4160])             # in one piece, and in segments
def test_calls_on_two_streams_at_once(T):
    sets = [inputs(1, T, 2, 1, 64, 32, seed=5 + i) for i in range(2)]
    logits = [torch.randn(300, 7001, device="cuda") for _ in range(2)]
    tokens = torch.randint(7001, (300,), device="cuda")
    want = [step(chunk_delta, *x) + token_logprobs(y, tokens, 5) for x, y in zip(sets, logits)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step(chunk_delta, *sets[i]) + token_logprobs(logits[i], tokens, 5))
    torch.cuda.synchronize()
    for i in range(2):
        for found in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(want[i], found))


def test_two_graphs_replayed_in_turns():
    """Each has its own workspace."""
    sets = [inputs(1, 4160, 2, 1, 32, 32, seed=8 + i) for i in range(2)]
    graphs, outs = [], []
    for x in sets:
        with torch.no_grad():
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                chunk_delta(*x[:6])
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(chunk_delta(*x[:6]))
            graphs.append(graph)
    with torch.no_grad():
        want = [chunk_delta(*x[:6]) for x in sets]
    for _ in range(3):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(want, outs) for a, b in zip(x, y))
