"""chunk_delta, delta_step and token_logprobs recorded by a tracer, given arrays with tangents,
after their saved arrays were changed, and captured beside eager graphs."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from gla_jax_amd import chunk_delta, delta_step, token_logprobs
from tests.delta_reference import inputs

pytestmark = pytest.mark.gpu
F32 = torch.float32


def rows(T, seed):
    return inputs(3, T, 4, 2, 32, 32, F32, seed=seed)[:6]


def token(seed):
    h0, *more = rows(1, seed)
    return [h0] + [x[:, 0].contiguous() for x in more]


def logits(seed, n=5, v=300):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, v, generator=g).cuda(), torch.randint(v, (n,), generator=g).cuda()


@pytest.mark.parametrize("ragged", [False, True])
def test_traced_sequences(ragged):
    fn = lambda *x: chunk_delta(*x)  # noqa: E731
    n = (torch.tensor([3, 0, 20], device="cuda", dtype=torch.int32),) if ragged else ()
    traced = torch.jit.trace(fn, (*rows(20, 1), *n), check_trace=False)
    new = rows(70, 2)
    for x, y in zip(traced(*new, *n), fn(*new, *n)):
        assert torch.equal(x, y)
    h0, a, b, v, k, q = new
    for other in ((h0[:2], a, b, v, k, q), (h0[..., :16].contiguous(), a, b, v, k, q), (h0, a, b[:, :30], v, k, q), (h0, a[:, :30], b, v, k, q),
                  (h0, a, b, v, k[:, :30], q), (h0, a, b, v, k, q[:, :30]), (h0, a, b, v, k.bfloat16(), q)):
        with pytest.raises(Exception, match="chunk_delta|size|shape"):
            traced(*other, *n)


def test_traced_steps_update_their_states():
    slots = torch.tensor([2, -1, 0], device="cuda")
    fn = lambda s, *x: delta_step(s, *x, slots=slots)  # noqa: E731
    traced = torch.jit.trace(fn, tuple(token(1)), check_trace=False)
    mine, want = token(2)[0], token(2)[0]
    for seed in (3, 4, 5):
        _, a, b, v, k, q = token(seed)
        assert torch.equal(traced(mine, a, b, torch.stack((v, v), -1)[..., 0], k, q), fn(want, a, b, v, k, q)) and torch.equal(mine, want)
    for other in (mine[:, :, :16].contiguous(), mine.transpose(2, 3), mine.double()):      # (a pool of another size is a pool)
        before = other.clone()
        with pytest.raises(Exception, match="states"):
            traced(other, a, b, v, k, q)
        assert torch.equal(other, before)


def test_traced_logprobs():
    traced = torch.jit.trace(lambda x, t: token_logprobs(x, t, 3), logits(1), check_trace=False)
    for new in (logits(2), logits(3, 9, 77)):
        for x, y in zip(traced(*new), token_logprobs(*new, 3)):
            assert torch.equal(x, y)
    x, t = logits(4)
    for other in ((x, t[:3]), (x.half(), t), (x[:, :2], t), (x, t.float())):
        with pytest.raises(Exception, match="tokens|float32|alternatives"):
            traced(*other)


def test_tangents_are_refused():
    calls = [(delta_step, token(1)), (chunk_delta, rows(20, 1)), (lambda x: token_logprobs(x, logits(1)[1], 2), [logits(1)[0]])]
    with fwAD.dual_level():
        for fn, plain in calls:
            for i, x in enumerate(plain):
                dual = list(plain)
                dual[i] = fwAD.make_dual(x.clone(), torch.ones_like(x))
                before = [t.clone() for t in dual]
                for mode in (torch.enable_grad, torch.no_grad):
                    with mode(), pytest.raises(RuntimeError):
                        fn(*dual)
                for t, y in zip(dual, before):
                    assert torch.equal(t, y)


def test_saved_arrays_that_were_changed_are_not_used():
    h0, a, b, v, k, q = (x.requires_grad_() for x in rows(20, 1))
    hT, out = chunk_delta(h0, a, b, v, k, q)
    with torch.no_grad():
        k.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        (hT.sum() + out.sum()).backward()
    x, t = logits(1)
    leaf = x.requires_grad_()
    given, _ = token_logprobs(leaf, t)
    t.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        given.sum().backward()


def test_calls_under_inference_mode():
    x = rows(20, 1)
    want = chunk_delta(*x)
    with torch.inference_mode():
        assert all(torch.equal(s, t) for s, t in zip(want, chunk_delta(*x)))
        made = torch.zeros(3, 4, 32, 32, device="cuda")
        _, a, b, v, k, q = token(1)
        delta_step(made, a, b, v, k, q)
        y, t = logits(1)
        assert all(torch.equal(s, u) for s, u in zip(token_logprobs(y, t, 4), token_logprobs(y.clone(), t, 4)))
    plain = torch.zeros(3, 4, 32, 32, device="cuda")
    delta_step(plain, a, b, v, k, q)
    assert torch.equal(plain, made)


@pytest.mark.parametrize("projected", [False, True])
@pytest.mark.parametrize("op", ["chunk_delta", "token_logprobs"])
def test_a_captured_backward_is_refused_while_an_eager_graph_of_its_leaves_lives(op, projected):
    """(The default stream accumulates their gradients then, and cannot wait for a capture.)  Without that graph it is captured."""
    if op == "chunk_delta":
        arrays = rows(40, 31)
        leaf = arrays[4].detach().clone().requires_grad_()
        call = lambda k: chunk_delta(*arrays[:4], k, arrays[5])[1]  # noqa: E731
    else:
        x, tokens = logits(32)
        leaf = x.detach().clone().requires_grad_()
        call = lambda x: token_logprobs(x, tokens)[0]  # noqa: E731

    def gradient():
        out = call(2 * leaf if projected else leaf)
        return torch.autograd.grad(out, [leaf], torch.ones_like(out))[0]
    want = gradient()
    alive = call(leaf)
    with pytest.raises(RuntimeError, match="graph of the same leaves"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            gradient()
    torch.cuda.synchronize()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gradient()
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
