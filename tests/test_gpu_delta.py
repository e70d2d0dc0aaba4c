"""chunk_delta and delta_step on the GPU against the recurrence in 64 bits."""
import pytest
import torch

from gla_jax_amd import chunk_delta, delta_step
from tests.delta_reference import check, check_step, inputs, reference, step

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

# B, T, H, HK, DK, DV, dtype, hidden
SIZES = [
    (1, 1, 1, 1, 16, 16, BF16, F32), (1, 2, 2, 1, 32, 16, BF16, F32), (2, 63, 3, 3, 64, 64, BF16, BF16), (1, 64, 2, 2, 128, 128, BF16, F32),
    (2, 65, 4, 2, 64, 48, BF16, F32), (1, 130, 4, 1, 128, 64, BF16, BF16), (2, 200, 2, 2, 96, 96, BF16, F32), (1, 257, 3, 1, 48, 256, BF16, F32),
    (1, 321, 6, 2, 128, 128, BF16, F32), (40, 70, 8, 4, 64, 64, BF16, F32), (20, 66, 8, 8, 128, 128, BF16, F32),
    (1, 1, 1, 1, 16, 16, F32, F32), (2, 31, 2, 2, 32, 48, F32, F32), (1, 33, 4, 2, 64, 64, F32, BF16), (1, 100, 2, 1, 128, 128, F32, F32),
    (2, 65, 3, 3, 80, 32, F32, F32), (20, 40, 8, 2, 128, 128, F32, F32),
]


@pytest.mark.parametrize("case", SIZES, ids=lambda c: "x".join(str(x).replace("torch.", "") for x in c))
def test_sizes(case):
    B, T, H, HK, DK, DV, dtype, hidden = case
    x = inputs(B, T, H, HK, DK, DV, dtype, hidden)
    check_step(step(chunk_delta, *x), *x)
    with torch.no_grad():
        hT, out = chunk_delta(*x[:6])
    exact = reference(*x[:6])
    check("hidden_final", hT, exact[0], dtype, None, -(-T // 64))
    check("out", out, exact[1], dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("decay", ["token", "hard", "mild", "resets", "head"])
@pytest.mark.parametrize("beta", ["token", "ends", "head"])
def test_gates(decay, beta, dtype):
    x = inputs(2, 150, 4, 2, 64, 32, dtype, decay=decay, beta=beta, seed=3)
    check_step(step(chunk_delta, *x), *x)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_keys_that_repeat(dtype):
    """With one key for all tokens and beta 1 the triangular system is as far from the identity as it gets."""
    x = inputs(1, 130, 2, 1, 64, 32, dtype, decay="mild", keys="same", seed=4)
    x[2] = torch.ones_like(x[2])
    check_step(step(chunk_delta, *x), *x)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lengths", [[0, 0, 0], [130, 1, 64], [65, 130, 0], [-3, 500, 63]])
def test_lengths(lengths, dtype):
    x = inputs(3, 130, 4, 2, 64, 32, dtype, seed=5)
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    past = torch.arange(130, device="cuda")[None, :] >= n[:, None]
    for t in (x[1], x[2], x[3], x[4], x[5], x[7]):
        t[past] = float("nan")                       # not read
    got = step(chunk_delta, *x, n)
    clean = [t.clone() for t in x]
    for t in (clean[1], clean[2], clean[3], clean[4], clean[5], clean[7]):
        t[past] = 0
    check_step(got, *clean, n)
    for t in (got[1], *got[3:]):
        assert not t[past].any()
    again = step(chunk_delta, *x, n.long())
    assert all(torch.equal(s, t) for s, t in zip(got, again))


def small(dtype=BF16, T=70, **more):
    return inputs(2, T, 4, 2, 32, 32, dtype, seed=6, **more)


def test_rows_cut_from_one_projection():
    h0, a, b, v, k, q, dh, do = small()
    rows = torch.cat([x.flatten(-2) for x in (q, k, v)], -1)
    cut = [x.unflatten(-1, (-1, 32)) for x in rows.split([64, 64, 128], -1)]
    whole = step(chunk_delta, h0, a, b, v, k, q, dh, do)
    parts = step(chunk_delta, h0, a, b, cut[2], cut[1], cut[0], dh, do)
    assert all(torch.equal(s, t) for s, t in zip(whole, parts))
    with torch.no_grad():
        # rows that begin elsewhere than on 16 bytes, features apart, gates with strides
        odd = torch.empty(2, 70, 4, 33, dtype=BF16, device="cuda")[..., 1:].copy_(v)
        apart = k.repeat_interleave(2, -1)[..., ::2]
        gates = torch.stack([a, b], -1)
        got = chunk_delta(h0, gates[..., 0], gates[..., 1], odd, apart, q)
    assert all(torch.equal(s, t) for s, t in zip(whole, got))


@pytest.mark.parametrize("DK, DV", [(33, 50), (7, 128)])
def test_features_that_16_does_not_divide(DK, DV):
    x = inputs(2, 70, 2, 1, DK, DV, seed=7)
    check_step(step(chunk_delta, *x), *x)


def test_leading_axes_and_other_types():
    h0, a, b, v, k, q, dh, do = small()
    whole = chunk_delta(h0, a, b, v, k, q)
    more = chunk_delta(*(t.unflatten(0, (1, 2)) for t in (h0, a, b, v, k, q)))
    assert all(torch.equal(s, t[0]) for s, t in zip(whole, more))
    one = chunk_delta(*(t[0] for t in (h0, a, b, v, k, q)))
    assert all(torch.equal(s[0], t) for s, t in zip(whole, one))
    double = chunk_delta(h0.double(), a.double(), b.double(), v, k, q)
    assert double[0].dtype == torch.float64 and torch.equal(double[0].float(), whole[0]) and torch.equal(double[1], whole[1])


def test_no_tokens():
    h0, a, b, v, k, q, dh, do = small()
    x = [h0, a[:, :0], b[:, :0], v[:, :0], k[:, :0], q[:, :0]]
    got = step(chunk_delta, *x, dh, do[:, :0])
    assert torch.equal(got[0], h0) and torch.equal(got[2], dh) and got[1].shape == (2, 0, 4, 32) and got[4].shape == (2, 0, 4)
    empty = chunk_delta(h0[:0], a[:0], b[:0], v[:0], k[:0], q[:0])
    assert empty[0].shape == (0, 4, 32, 32) and empty[1].shape == (0, 70, 4, 32)


def test_one_of_two_results_and_one_of_six_gradients():
    x = small()
    dh, do = x[6], x[7]
    zero_dh, zero_do = torch.zeros_like(dh), torch.zeros_like(do)
    for which, cot in ((0, (dh, zero_do)), (1, (zero_dh, do))):
        arrays = [t.detach().clone().requires_grad_() for t in x[:6]]
        got = torch.autograd.grad(chunk_delta(*arrays)[which], arrays, cot[which])
        exact = step(chunk_delta, *x[:6], *cot)[2:]
        assert all(torch.equal(s, t) for s, t in zip(got, exact))
    whole = step(chunk_delta, *x)[2:]
    for i in range(6):
        arrays = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate(x[:6])]
        g, = torch.autograd.grad(chunk_delta(*arrays), [arrays[i]], (dh, do))
        assert torch.equal(g, whole[i])


def test_gradients_against_differences():
    """float32: a step of 2^-6 along a direction, against the gradient's product with it.  With f of four such steps the difference's own error is of the
    fourth power of the step, and a sum of n results rounds to sqrt(n) 2^-24 of their norm, over the step."""
    x = [t.detach() for t in inputs(1, 40, 2, 1, 16, 16, F32, seed=8)]
    dh, do = x[6], x[7]
    grads = step(chunk_delta, *x)[2:]
    g = torch.Generator(device="cuda").manual_seed(9)

    def f(i, t):
        arrays = list(x[:6])
        arrays[i] = t
        hT, out = chunk_delta(*arrays)
        return float((hT.double() * dh).sum() + (out.double() * do).sum())

    for i in range(6):
        d = torch.randn(x[i].shape, device="cuda", generator=g)
        d = d / d.norm()
        e = 2.0 ** -6
        at = [f(i, x[i] + s * e * d) for s in (-2, -1, 1, 2)]
        got = (at[0] - 8 * at[1] + 8 * at[2] - at[3]) / (12 * e)
        want = float((grads[i].double() * d).sum())
        assert abs(got - want) <= 2e-3 * max(abs(want), float(grads[i].norm()) / d.numel() ** 0.5 * 4), (i, got, want)


def test_runs_are_the_same_bits():
    x = inputs(2, 200, 4, 2, 128, 64, seed=10)
    first = step(chunk_delta, *x)
    for _ in range(3):
        assert all(torch.equal(s, t) for s, t in zip(first, step(chunk_delta, *x)))


def test_a_nan_stays_in_its_head_and_behind_its_chunk():
    h0, a, b, v, k, q, dh, do = small()
    clean = chunk_delta(h0, a, b, v, k, q)
    v = v.clone()
    v[0, 66, 1, 3] = float("nan")
    hT, out = chunk_delta(h0, a, b, v, k, q)
    assert torch.isnan(out[0, 67:, 1]).any() and torch.isnan(hT[0, 1]).any()
    assert torch.equal(out[1], clean[1][1]) and torch.equal(out[0, :, [0, 2, 3]], clean[1][0, :, [0, 2, 3]])
    assert torch.equal(out[0, :64], clean[1][0, :64])


def test_graph_of_a_training_step_replays():
    h0, a, b, v, k, q, dh, do = inputs(2, 150, 4, 2, 64, 64, seed=11)
    arrays = [t.detach().clone().requires_grad_() for t in (h0, a, b, v, k, q)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(chunk_delta(*arrays), arrays, (dh, do))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hT, out = chunk_delta(*arrays)
        grads = torch.autograd.grad((hT, out), arrays, (dh, do))
    for seed in range(3):
        new = inputs(2, 150, 4, 2, 64, 64, seed=20 + seed)
        with torch.no_grad():
            for t, s in zip(arrays, new):
                t.copy_(s)
            dh.copy_(new[6])
            do.copy_(new[7])
        graph.replay()
        torch.cuda.synchronize()
        eager = step(chunk_delta, *new)
        assert all(torch.equal(s, t) for s, t in zip((hT, out) + grads, eager))


def test_another_stream():
    x = inputs(2, 200, 4, 2, 64, 64, seed=12)
    first = step(chunk_delta, *x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step(chunk_delta, *x)
    side.synchronize()
    assert all(torch.equal(s, t) for s, t in zip(first, second))


def test_maps_and_second_gradients():
    h0, a, b, v, k, q, dh, do = small()
    whole = chunk_delta(h0, a, b, v, k, q)
    mapped = torch.func.vmap(chunk_delta)(h0, a, b, v, k, q)
    assert all(torch.equal(s, t) for s, t in zip(whole, mapped))

    def loss(*arrays):
        hT, out = chunk_delta(*arrays)
        return (hT * dh).sum() + (out.float() * do.float()).sum()
    got = torch.func.grad(loss, argnums=(0, 1, 2, 3, 4, 5))(h0, a, b, v, k, q)
    assert all(torch.equal(s, t) for s, t in zip(got, step(chunk_delta, h0, a, b, v, k, q, dh, do)[2:]))
    arrays = [t.detach().clone().requires_grad_() for t in (h0, a, b, v, k, q)]
    first = torch.autograd.grad(loss(*arrays), arrays, create_graph=True)
    with pytest.raises(NotImplementedError):
        first[3].float().sum().backward()


# ---- one token ------------------------------------------------------------------------------------
def rows(B, H, HK, DK, DV, dtype=BF16, seed=0):
    h0, a, b, v, k, q, _, _ = inputs(B, 1, H, HK, DK, DV, dtype, seed=seed)
    return h0, a[:, 0], b[:, 0], v[:, 0], k[:, 0], q[:, 0]


def check_states(got, exact, dtype):
    """A state of 32 bits sums DK + 1 products in floats: sqrt(257) 2^-24 of its norm; one of 16 bits is rounded once more."""
    x, y = got.double().cpu(), exact
    bound = 2.0 ** -8 if got.dtype == BF16 else 1e-6
    assert float((x - y).norm()) <= bound * float(y.norm()) and torch.isfinite(x).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("state", [BF16, F32])
@pytest.mark.parametrize("B, H, HK, DK, DV", [(1, 1, 1, 16, 16), (3, 4, 2, 64, 48), (5, 6, 1, 128, 128), (2, 2, 2, 96, 64), (3, 2, 1, 256, 256), (130, 8, 4, 64, 64)])
def test_step(B, H, HK, DK, DV, state, dtype):
    h0, a, b, v, k, q = rows(B, H, HK, DK, DV, dtype)
    states = h0.to(state)
    exact = reference(states, *(t[:, None] for t in (a, b, v, k, q)))
    out = delta_step(states, a, b, v, k, q)
    check_states(states, exact[0], dtype)
    assert out.dtype == dtype and out.shape == (B, H, DV)
    bound = 2.0 ** -8 if dtype == BF16 else 1e-6
    assert float((out.double().cpu() - exact[1][:, 0]).norm()) <= bound * float(exact[1].norm())


def test_step_pool_and_idle_rows():
    h0, a, b, v, k, q = rows(5, 4, 2, 64, 64, seed=1)
    pool = torch.randn(9, 4, 64, 64, device="cuda")
    before = pool.clone()
    for kind in (torch.int32, torch.int64):
        slots = torch.tensor([7, -1, 0, 9, 3], device="cuda", dtype=kind)
        pool.copy_(before)
        out = delta_step(pool, a, b, v, k, q, slots=slots)
        some = before[[7, 0, 3]].contiguous()
        want = delta_step(some, *(t[[0, 2, 4]] for t in (a, b, v, k, q)))
        assert torch.equal(out[[0, 2, 4]], want) and not out[[1, 3]].any()
        assert torch.equal(pool[[7, 0, 3]], some)
        rest = [i for i in range(9) if i not in (7, 0, 3)]
        assert torch.equal(pool[rest], before[rest])


@pytest.mark.parametrize("G, W, DK", [(3, 4, 64), (2, 16, 32), (1, 20, 64), (2, 8, 256)])
def test_step_of_beams(G, W, DK):
    h0, a, b, v, k, q = rows(G * W, 2, 1, DK, 32, seed=2)
    parents = torch.randint(-1, W + 1, (G, W), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    states = h0.clone()
    out = delta_step(states, a, b, v, k, q, parents=parents)
    own = torch.arange(W, device="cuda").expand(G, W)
    source = torch.where((parents < 0) | (parents >= W), own, parents) + torch.arange(G, device="cuda")[:, None] * W
    moved = h0[source.flatten()].contiguous()
    want = delta_step(moved, a, b, v, k, q)
    assert torch.equal(out, want) and torch.equal(states, moved)


def test_step_is_a_chunk_of_one_token():
    h0, a, b, v, k, q = rows(3, 4, 2, 64, 64, F32, seed=4)
    states = h0.clone()
    out = delta_step(states, a, b, v, k, q)
    hT, whole = chunk_delta(h0, *(t[:, None] for t in (a, b, v, k, q)))
    assert float((states - hT).norm()) <= 1e-6 * float(hT.norm()) and float((out - whole[:, 0]).norm()) <= 1e-6 * float(out.norm())


def test_step_from_other_layouts_and_a_graph():
    h0, a, b, v, k, q = rows(6, 4, 2, 64, 64, seed=5)
    want = h0.clone()
    out = delta_step(want, a, b, v, k, q)
    states = h0.clone()
    odd = torch.empty(6, 4, 65, dtype=BF16, device="cuda")[..., 1:].copy_(v)
    got = delta_step(states, a.double(), b.double(), odd, k.transpose(0, 1).contiguous().transpose(0, 1), q)
    assert torch.equal(out, got) and torch.equal(states, want)
    one = torch.full((4,), -0.25, device="cuda")
    each, all_ = h0.clone(), h0.clone()
    assert torch.equal(delta_step(each, one, one.abs(), v, k, q), delta_step(all_, one.expand(6, 4), one.abs().expand(6, 4), v, k, q))
    assert torch.equal(each, all_)
    graph = torch.cuda.CUDAGraph()
    states = h0.clone()
    with torch.cuda.graph(graph):
        got = delta_step(states, a, b, v, k, q)
    for _ in range(3):
        states.copy_(h0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(states, want)


def test_step_counts_as_a_new_version():
    h0, a, b, v, k, q = rows(2, 2, 1, 32, 32, seed=6)
    w = torch.ones_like(h0, requires_grad=True)
    loss = (w * h0).sum()
    delta_step(h0, a, b, v, k, q)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with pytest.raises(RuntimeError, match="no gradient"):
        delta_step(h0, a, b.clone().requires_grad_(), v, k, q)
