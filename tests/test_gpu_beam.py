"""beam_select and reorder_states against the definition in 64 bits.

Places have to be the definition's: inputs whose candidates differ by less than the rounding of a 32-bit score (1e-5 here: scores
are below 64 in size) from another beam's are not drawn.  Scores are sums of three floats and a logarithm of a sum: at most 8 units in the last
place of 64, i.e. 3.1e-5."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _reference(logits, scores, num, finished=None, eos=0):
    """[G][num] of (score, beam * V + token), best first, equal ones by their place."""
    G, W, V = logits.shape
    x = logits.double().cpu()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    lse, scores = torch.logsumexp(x, -1), scores.double().cpu()
    found = []
    for g in range(G):
        cand = []
        for w in range(W):
            if finished is not None and bool(finished[g, w]):
                cand.append((float(scores[g, w]), w * V + eos))
                cand += [(-math.inf, w * V + t) for t in range(min(V, num + 1)) if t != eos][:num - 1]
                continue
            value, token = x[g, w].sort(descending=True, stable=True)
            for v, t in zip(value[:num].tolist(), token[:num].tolist()):
                s = float(scores[g, w]) + (v - float(lse[g, w]))
                cand.append((-math.inf if s != s else s, w * V + t))
        cand.sort(key=lambda c: (-c[0], c[1]))
        found.append(cand[:num])
    return found


def _apart(found):
    """No two candidates of different scores are closer than 32-bit scores tell apart."""
    for cand in found:
        s = [c[0] for c in cand if math.isfinite(c[0])]
        if any(0 < a - b < 1e-5 for a, b in zip(s, s[1:])):
            return False
    return True


def _check(got, found, V):
    scores, parents, tokens = (x.reshape(-1, x.shape[-1]).cpu() for x in got)
    for g, cand in enumerate(found):
        places = (parents[g] * V + tokens[g]).tolist()
        assert places == [c[1] for c in cand], f"search {g}"
        for mine, (s, _) in zip(scores[g].tolist(), cand):
            assert mine == s if math.isinf(s) else abs(mine - s) <= 3.1e-5


def _logits(kind, G, W, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = 3.0 * torch.randn(G, W, V, generator=g)
    beams = 0.37 * torch.arange(W, dtype=torch.float32)[:, None]
    if kind == "equal":                      # ties everywhere, between the beams of equal scores too
        x[:] = 1.5
    elif kind == "banned":
        x[torch.rand(G, W, V, generator=g) < 0.7] = -math.inf
        x[:, -1] = -math.inf                 # a beam without any token
    elif kind == "rising":
        x = (0.001 * torch.arange(V) + beams).expand(G, W, V).clone()
    elif kind == "falling":
        x = (-0.001 * torch.arange(V) + beams).expand(G, W, V).clone()
    elif kind == "nan":
        x[torch.rand(G, W, V, generator=g) < 0.3] = math.nan
    return x.to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["random", "equal", "banned", "rising", "falling", "nan"])
@pytest.mark.parametrize("G, W, V, num", [(1, 1, 1, 1), (2, 3, 7, 3), (3, 4, 5, 20), (2, 2, 4097, 64), (1, 64, 50, 64), (2, 8, 1000, 16),
                                          (4, 5, 8192, 5), (1, 16, 40000, 32), (3, 1, 300, 2), (2, 33, 129, 64)])
def test_candidates(G, W, V, num, kind, dtype):
    from gla_jax_amd import beam_select
    for seed in range(20):
        x = _logits(kind, G, W, V, dtype, 100 * seed + V)
        g = torch.Generator().manual_seed(seed)
        scores = (-5.0 * torch.rand(G, W, generator=g)).cuda() if kind != "equal" else torch.zeros(G, W, device="cuda")
        found = _reference(x, scores, num)
        if kind in ("rising", "falling") or _apart(found):
            break
    if kind in ("rising", "falling") and not _apart(found):
        pytest.skip("these beams' candidates are closer than 32-bit scores tell apart")
    _check(beam_select(x, scores, num), found, V)


@pytest.mark.parametrize("G, W, V, num", [(40, 2, 131072, 5), (70, 2, 131071, 64)])
def test_large_vocabularies(G, W, V, num):
    """Wide stretches, rows that begin on 16 bytes and rows that do not."""
    from gla_jax_amd import beam_select
    x = _logits("random", G, W, V, torch.float32, 1)
    scores = -torch.rand(G, W, device="cuda")
    found = _reference(x, scores, num)
    near = [g for g in range(G) if _apart(found[g:g + 1])]
    assert len(near) > G // 2
    got = beam_select(x, scores, num)
    _check([y[near] for y in got], [found[g] for g in near], V)


@pytest.mark.parametrize("eos", [0, 2, 999])
def test_beams_that_have_ended(eos):
    from gla_jax_amd import beam_select
    x = _logits("random", 3, 4, 1000, torch.bfloat16, 7)
    finished = torch.tensor([[True, False, False, True], [True] * 4, [False] * 4], device="cuda")
    x[finished] = math.nan                   # their logits are not read
    scores = torch.tensor([[-1.0, -2.0, -3.0, -30.0]], device="cuda").repeat(3, 1)
    for num in (4, 8):
        _check(beam_select(x, scores, num, finished, eos), _reference(x, scores, num, finished.cpu(), eos), 1000)


def test_first_step_and_beams_without_a_chance():
    """All beams but one at -inf: the candidates are that one's; where nothing is left, the first places."""
    from gla_jax_amd import beam_select
    x = _logits("random", 2, 4, 100, torch.float32, 8)
    scores = torch.tensor([[0.0, -math.inf, -math.inf, -math.inf], [-math.inf] * 4], device="cuda")
    got = beam_select(x, scores)
    _check(got, _reference(x, scores, 4), 100)
    assert not got[1][0].any() and torch.isinf(got[0][1]).all()
    scores[0, 0] = math.nan
    assert torch.isinf(beam_select(x, scores)[0]).all()


def test_axes_and_strides():
    from gla_jax_amd import beam_select
    x = _logits("random", 6, 3, 500, torch.float32, 9)
    scores = -torch.rand(6, 3, device="cuda")
    want = beam_select(x, scores)
    padded = torch.full((6, 3, 517), math.nan, device="cuda")
    padded[..., :500] = x
    for view, s in ((x.reshape(2, 3, 3, 500), scores.reshape(2, 3, 3)), (padded[..., :500], scores),
                    (x.transpose(0, 1).contiguous().transpose(0, 1), scores), (x.transpose(1, 2).contiguous().transpose(1, 2), scores)):
        for got, y in zip(beam_select(view, s), want):
            assert torch.equal(got.reshape(y.shape), y)
    for got, y in zip(beam_select(x[0], scores[0]), want):
        assert torch.equal(got, y[0])
    assert beam_select(x[:0], scores[:0])[0].shape == (0, 3)
    for got, y in zip(beam_select(x[:, :1], scores[:, :1], 2), beam_select(x[:, :1].contiguous(), scores[:, :1].contiguous(), 2)):
        assert torch.equal(got, y)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("W", [1, 3, 4, 8, 16, 17, 64])
@pytest.mark.parametrize("shape, dtype", [((2, 16, 16), torch.float32), ((3, 8), torch.bfloat16), ((7,), torch.uint8), ((5,), torch.float32),
                                          ((), torch.int64)])
def test_states_in_another_order(shape, dtype, W, index):
    """Rows of any size and type, every one read before any of its search is written."""
    from gla_jax_amd import reorder_states
    G = 3
    gen = torch.Generator().manual_seed(W)
    parents = torch.randint(-1, W + 1, (G, W), generator=gen)
    for pooled in (False, True):
        states = torch.randint(0, 100, (G * W + 5,) + shape, generator=gen).to(dtype)
        slots = torch.randperm(G * W + 5, generator=gen)[:G * W].reshape(G, W) if pooled else torch.arange(G * W).reshape(G, W)
        if pooled:
            slots[1, W // 2] = -1
            slots[2, 0] = 10 ** 6
        want = states.clone()
        for g in range(G):
            for w in range(W):
                p = int(parents[g, w])
                here, there = int(slots[g, w]), int(slots[g, p]) if 0 <= p < W else -1
                if 0 <= here < len(states) and 0 <= there < len(states):
                    want[here] = states[there]
        mine = states.cuda()
        assert reorder_states(mine, parents.to(index).cuda(), slots.to(index).cuda() if pooled else None) is mine
        assert torch.equal(mine.cpu(), want)


def test_rows_that_begin_on_an_odd_address():
    from gla_jax_amd import reorder_states
    x = torch.arange(1 + 4 * 24, device="cuda", dtype=torch.int16)[1:].view(4, 24)
    want = x[[3, 2, 1, 0]].clone()
    assert torch.equal(reorder_states(x, torch.tensor([[3, 2, 1, 0]], device="cuda")), want)


def test_selection_replays_from_a_graph():
    from gla_jax_amd import beam_select, reorder_states
    x = _logits("random", 4, 4, 3001, torch.float32, 12)
    scores, states = torch.zeros(4, 4, device="cuda"), torch.zeros(16, 100, device="cuda")

    def run():
        s, p, t = beam_select(x, scores)
        reorder_states(states, p)
        return s, p, t

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = run()
    for i in range(3):
        x.copy_(_logits("random", 4, 4, 3001, torch.float32, 20 + i))
        scores.copy_(-torch.rand(4, 4))
        states.copy_(torch.rand(16, 100))
        before = states.clone()
        graph.replay()
        torch.cuda.synchronize()
        after = states.clone()
        states.copy_(before)
        for a, b in zip(replayed, run()):
            assert torch.equal(a, b)
        assert torch.equal(after, states)


def test_parents_continue_in_the_next_step():
    """decay_step with parents is reorder_states and decay_step."""
    from gla_jax_amd import decay_step, reorder_states
    G, W, H, D = 2, 4, 3, 32
    g = torch.Generator().manual_seed(3)
    states = torch.randn(G * W, H, D, D, generator=g).cuda()
    a = torch.full((G * W, H), -0.1, device="cuda")
    v, k, q = (torch.randn(G * W, H, D, generator=g).cuda() for _ in range(3))
    parents = torch.randint(W, (G, W), generator=g).cuda()
    other = reorder_states(states.clone(), parents)
    assert torch.equal(decay_step(other, a, v, k, q), decay_step(states, a, v, k, q, parents=parents)) and torch.equal(other, states)
