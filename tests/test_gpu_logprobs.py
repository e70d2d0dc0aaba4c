"""token_logprobs on the GPU against log_softmax in 64 bits.

Tolerances.  log p = (x - m) - log s.  Each exponential is off by two units in its last place and by the rounding of its exponent, 2^-24 of a distance d
that weighs e^-d: 2^-22 each of s, and with the order of summation 2^-21 of log s.  The logarithm is off by a unit, 2^-23 of log s <= log V, and
the two differences by half of one: together 2^-21 + 2^-23 (log V + |log p|) (`off`).  (At 700 equal logits among others, log s = 6.6, a flat 2^-20 was
missed by 9e-8: a unit of the logarithm alone is 4.8e-7 there.)  The entropy takes two such sums.  A gradient is a probability, off by as much
relative to itself as its log is absolutely, times a sum off by as much of its own terms: twice `off` of each; 16-bit ones are
rounded once, 2^-8 of themselves.
"""
import math

import pytest
import torch

from gla_jax_amd import token_logprobs

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def logits_of(N, V, dtype, seed=0, apart=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 3.0 * torch.randn(N, V + apart, device="cuda", generator=g) + 5.0 * torch.randn(N, 1, device="cuda", generator=g)
    x = x.to(dtype)[:, :V]
    t = torch.randint(V, (N,), device="cuda", generator=g)
    return x, t


def exact(x, t, g, h):
    V = x.shape[-1]
    p = torch.log_softmax(x.double(), -1)
    counts = (t >= 0) & (t < V)
    at = t.clamp(0, V - 1).long()[..., None]
    w = p.exp()
    H = torch.special.entr(w).sum(-1)
    given = torch.where(counts, p.gather(-1, at)[..., 0], 0.0)
    g, h = torch.where(counts, g.double(), 0.0)[..., None], torch.where(counts, h.double(), 0.0)[..., None]
    d = -g * w - h * torch.where(w > 0, w * (p + H[..., None]), 0.0)
    return given, torch.where(counts, H, 0.0), d.scatter_add(-1, at, g), p


def off(p, V):
    return 2.0 ** -21 + 2.0 ** -23 * (math.log(V) + p.double().abs())


def close(x, y, bound):
    assert bool(((x.double() - y).abs() <= bound).all()), float(((x.double() - y).abs() - bound).max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N, V, apart, top", [
    (1, 1, 0, 1), (1, 2, 0, 2), (3, 7, 0, 3), (2, 8, 8, 8), (5, 63, 1, 5), (4, 64, 0, 64), (3, 1000, 24, 20), (7, 1001, 0, 1), (9, 4099, 5, 8), (2, 32000, 0, 5),
    (1100, 515, 0, 4), (1030, 9000, 8, 20), (3, 70001, 0, 64), (2, 131072, 0, 20), (1025, 33, 0, 0), (2, 300007, 1, 33)])
def test_sizes(N, V, apart, top, dtype):
    x, t = logits_of(N, V, dtype, apart=apart)
    if N > 2:
        t[1], t[2] = -100, V                       # do not count
    r = torch.Generator(device="cuda").manual_seed(1)
    g, h = torch.randn(N, device="cuda", generator=r), torch.randn(N, device="cuda", generator=r)
    want = exact(x, t, g, h)
    leaf = x.detach().requires_grad_()
    found = token_logprobs(leaf, t, top)
    d, = torch.autograd.grad(found[:2], [leaf], (g, h))
    assert found[0].dtype == found[1].dtype == F32 and d.dtype == dtype and d.shape == x.shape
    span = want[3].abs().amax(-1).clamp(max=1e4)
    close(found[0], want[0], off(want[0], V))
    close(found[1], want[1], 2 * off(want[1], V))
    factor = (g.abs() + h.abs() * (span + math.log(V) + 1)).double()[:, None]
    close(d, want[2], 2 * off(want[3].clamp(min=-1e4), V) * factor * want[3].exp().clamp(min=2.0 ** -100) + (2.0 ** -8 if dtype == BF16 else 2.0 ** -22) * want[2].abs() + 1e-30)
    with torch.no_grad():
        plain = token_logprobs(x, t, top)
    assert all(torch.equal(a, b) for a, b in zip(found, plain))
    if top:
        counts = (t >= 0) & (t < V)
        order = x.float().sort(dim=-1, descending=True, stable=True)[1][:, :top]
        assert torch.equal(found[3], order.masked_fill(~counts[:, None], -1))
        close(found[2][counts], want[3].gather(-1, order)[counts], off(want[3].gather(-1, order)[counts], V))
        assert bool((found[2][~counts] == -math.inf).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V, rows", [(3000, 3), (130000, 2), (700, 1050)])
def test_equal_values_come_in_the_order_of_their_tokens(V, rows, dtype):
    x = torch.randint(0, 3, (rows, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dtype)
    x[0] = 1.0
    x[1] = -math.inf
    x[1, [5, V - 1, V // 2]] = torch.tensor([1.0, 1.0, -0.0], device="cuda", dtype=dtype)
    t = torch.zeros(rows, device="cuda", dtype=torch.int32)
    t[1] = V - 1
    given, entropy, near, index = token_logprobs(x, t, 9)
    order = x.float().sort(dim=-1, descending=True, stable=True)[1][:, :9]
    assert torch.equal(index, order)
    p = torch.log_softmax(x.double(), -1)
    want = p.gather(-1, order)
    assert torch.equal(near == -math.inf, want == -math.inf)
    want = want.masked_fill(want == -math.inf, 0)
    close(near.masked_fill(near == -math.inf, 0), want, off(want, V))
    want = p.gather(-1, t.long()[:, None])[:, 0]
    close(given, want, off(want, V))
    want = torch.special.entr(p.exp()).sum(-1)
    close(entropy, want, 2 * off(want, V))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_infinities_and_nan(dtype):
    x, t = logits_of(8, 1000, dtype, seed=3)
    t[:] = 4
    x[0, ::2] = -math.inf
    x[0, 4] = -math.inf                           # the given token may not come
    x[1] = -math.inf
    x[2, 7] = math.nan
    x[3, 9] = math.inf
    x[4] = -3e38
    x[5, 0], x[5, 1:] = 3e38, -3e38
    x[6] = 1e4 * x[6]
    r = torch.ones(8, device="cuda")
    leaf = x.detach().requires_grad_()
    given, entropy, near, index = token_logprobs(leaf, t, 3)
    d, = torch.autograd.grad((given, entropy), [leaf], (r, r))
    p = torch.log_softmax(x.double(), -1)
    assert float(given[0]) == -math.inf and torch.isfinite(entropy[0])
    for i in (1, 2, 3):
        assert torch.isnan(given[i]) and torch.isnan(entropy[i]) and torch.isnan(d[i]).any()
    for i in (4, 5, 6, 7):
        if i == 5:                                # -6e38 is no 32-bit number
            assert float(given[i]) == -math.inf == float(p[i, 4].float())
        else:
            close(given[i], p[i, 4], off(p[i, 4], 1000))
        want = torch.special.entr(p[i].exp()).sum()
        close(entropy[i], want, 2 * off(want, 1000))
        assert torch.isfinite(d[i]).all()
    number = torch.where(torch.isnan(x), -math.inf, x.float())
    assert torch.equal(index, number.sort(dim=-1, descending=True, stable=True)[1][:, :3])
    assert torch.equal(d[0].float()[x[0] == -math.inf], torch.where(torch.arange(1000, device="cuda") == 4, 1.0, 0.0)[x[0] == -math.inf])


def test_layouts_types_and_axes():
    x, t = logits_of(24, 1000, F32, seed=4)
    want = token_logprobs(x, t, 4)
    shaped = token_logprobs(x.view(2, 3, 4, 1000), t.view(2, 3, 4), 4)
    assert all(torch.equal(a, b.flatten(0, 2)) for a, b in zip(want, shaped))
    one = token_logprobs(x[3], t[3], 4)
    assert all(torch.equal(a[3], b) for a, b in zip(want, one)) and one[0].ndim == 0
    odd = torch.empty(24 * 1000 + 3, device="cuda")[3:].view(24, 1000).copy_(x)
    far = torch.empty(24, 2000, device="cuda")[:, ::2].copy_(x)
    turned = x.view(4, 6, 1000).transpose(0, 1)
    for y, s, back in ((odd, t.int(), lambda a: a), (far, t, lambda a: a), (turned, t.view(4, 6).t(), lambda a: a.transpose(0, 1).flatten(0, 1))):
        leaf = y.detach().requires_grad_()
        got = token_logprobs(leaf, s, 4)
        for a, b in zip(want, got):
            c = back(b)
            assert torch.equal(a, c) if a.dtype == torch.int64 else bool(((a - c).abs() <= 2.0 ** -19 * (1 + a.abs())).all())
        g = torch.autograd.grad(got[0].sum(), [leaf])[0]
        whole = x.detach().requires_grad_()
        w = torch.autograd.grad(token_logprobs(whole, t)[0].sum(), [whole])[0]
        assert g.shape == y.shape and float((back(g) - w).abs().max()) <= 2.0 ** -19
    none = token_logprobs(x[:0], t[:0], 4)
    assert none[0].shape == (0,) and none[3].shape == (0, 4)


def test_gradient_against_differences_and_cross_entropy():
    x, t = logits_of(6, 50, F32, seed=5)
    t[2] = -100
    leaf = x.detach().requires_grad_()
    loss = -token_logprobs(leaf, t)[0].sum()
    ours, = torch.autograd.grad(loss, [leaf])
    leaf2 = x.detach().requires_grad_()
    theirs, = torch.autograd.grad(torch.nn.functional.cross_entropy(leaf2, t, reduction="sum", ignore_index=-100), [leaf2])
    assert float((ours - theirs).abs().max()) <= 2.0 ** -20
    g = torch.Generator(device="cuda").manual_seed(6)
    v = torch.randn(x.shape, device="cuda", generator=g)
    r = torch.randn(2, 6, device="cuda", generator=g)

    def f(s):
        a, b = token_logprobs(x + s * v, t)
        return float((a.double() * r[0]).sum() + (b.double() * r[1]).sum())
    e = 2.0 ** -5
    got = (f(-2 * e) - 8 * f(-e) + 8 * f(e) - f(2 * e)) / (12 * e)
    leaf = x.detach().requires_grad_()
    want = float((torch.autograd.grad(token_logprobs(leaf, t), [leaf], (r[0], r[1]))[0].double() * v).sum())
    assert abs(got - want) <= 1e-3 * max(1.0, abs(want))          # the fourth power of the step, and 2^-20 over it


def test_graph_stream_maps_and_second_gradients():
    x, t = logits_of(40, 3001, BF16, seed=7, apart=7)
    leaf = x.detach().clone().requires_grad_()
    r = torch.ones(40, device="cuda")

    def run():
        found = token_logprobs(leaf, t, 3)
        return found + torch.autograd.grad(found[:2], [leaf], (r, r))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for seed in range(3):
        y, s = logits_of(40, 3001, BF16, seed=8 + seed)
        with torch.no_grad():
            leaf.copy_(y)
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, run()))
    mapped = torch.func.vmap(lambda a, b: token_logprobs(a, b, 3))(x.view(4, 10, 3001), t.view(4, 10))
    assert all(torch.equal(a, b.flatten(0, 1)) for a, b in zip(token_logprobs(x, t, 3), mapped))
    got = torch.func.grad(lambda a: token_logprobs(a, t)[0].sum())(x)
    leaf2 = x.detach().requires_grad_()
    assert torch.equal(got, torch.autograd.grad(token_logprobs(leaf2, t)[0].sum(), [leaf2])[0])
    first, = torch.autograd.grad(token_logprobs(leaf2, t)[0].sum(), [leaf2], create_graph=True)
    with pytest.raises(NotImplementedError):
        first.float().sum().backward()


def test_rows_that_do_not_count_are_not_read():
    x, t = logits_of(6, 500, F32, seed=9)
    t[::2] = torch.tensor([-1, 500, 2 ** 40], device="cuda")
    x[::2] = math.nan
    leaf = x.detach().requires_grad_()
    given, entropy, near, index = token_logprobs(leaf, t, 2)
    d, = torch.autograd.grad((given, entropy), [leaf], (torch.ones(6, device="cuda"),) * 2)
    assert not given[::2].any() and not entropy[::2].any() and not d[::2].any()
    assert bool((near[::2] == -math.inf).all()) and bool((index[::2] == -1).all())
    assert torch.isfinite(given[1::2]).all() and torch.isfinite(d[1::2]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [70, 1000, 40001])
def test_rows_that_allow_few_tokens(V, dtype):
    """Fewer above -inf than alternatives are asked for, none to 63 of them: the rest are the first tokens of -inf."""
    rows, top = 66, 64
    g = torch.Generator(device="cuda").manual_seed(10)
    x = torch.full((rows, V), -math.inf, device="cuda", dtype=dtype)
    for i in range(rows - 1):
        at = torch.randperm(V, device="cuda", generator=g)[:i]
        x[i, at] = torch.randn(i, device="cuda", generator=g).to(dtype)
    x[rows - 1] = -3e38                            # the type's lowest (nearly) is above -inf
    t = torch.randint(V, (rows,), device="cuda", generator=g)
    given, entropy, near, index = token_logprobs(x, t, top)
    assert torch.equal(index, x.float().sort(dim=-1, descending=True, stable=True)[1][:, :top])
    p = torch.log_softmax(x.double(), -1)
    assert torch.isnan(given[0]) and torch.isnan(entropy[0]) and torch.isnan(near[0]).all()
    want = p.gather(-1, index)[1:]
    assert torch.equal(near[1:] == -math.inf, want == -math.inf)
    want = want.masked_fill(want == -math.inf, 0)
    close(near[1:].masked_fill(near[1:] == -math.inf, 0), want, off(want, V))
    want = torch.special.entr(p[1:].exp()).sum(-1)
    close(entropy[1:], want, 2 * off(want, V))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_more_rows_than_a_launch_holds(dtype):
    N = (1 << 22) + 3
    x = torch.randint(-3, 4, (N, 3), device="cuda", generator=torch.Generator(device="cuda").manual_seed(11)).to(dtype)
    t = torch.arange(N, device="cuda") % 4 - 1                 # every fourth does not count
    leaf = x.detach().requires_grad_()
    found = token_logprobs(leaf, t, 2)
    g, h = torch.linspace(-1, 1, N, device="cuda"), torch.linspace(0, 1, N, device="cuda")
    d, = torch.autograd.grad(found[:2], [leaf], (g, h))
    at = torch.cat([torch.arange(5), torch.arange(N - 9, N)]).cuda()
    want = exact(x[at], t[at], g[at], h[at])
    close(found[0][at], want[0], off(want[0], 3))
    close(found[1][at], want[1], 2 * off(want[1], 3))
    close(d[at], want[2], 2 ** -7 * want[2].abs() + 2.0 ** -18 if dtype == BF16 else torch.full_like(want[2], 2.0 ** -18))
    counts = (t >= 0) & (t < 3)
    order = x.float().sort(dim=-1, descending=True, stable=True)[1][:, :2]
    assert torch.equal(found[3], order.masked_fill(~counts[:, None], -1))
    assert not found[0][~counts].any() and not d[~counts].any()
