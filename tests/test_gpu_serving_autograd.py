"""decay_step, beam_select and reorder_states beside autograd and tracers: they have no gradient, and what looks on must not miss them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

B, H, D = 8, 2, 32


def _token(seed, *, batch=B):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    return [torch.nn.functional.logsigmoid(2.0 + r(batch, H)), r(batch, H, D), r(batch, H, D), r(batch, H, D) * D ** -0.5]


def _states(seed):
    return torch.randn(B, H, D, D, generator=torch.Generator().manual_seed(100 + seed)).cuda()


PARENTS = [[1, 0, 0, 3], [2, 2, 2, 1]]


def _updates():
    """Calls that update `states` in place: by the native host side, and as others than it takes (another type of log_decay, indices of
    two widths)."""
    from gla_jax_amd import decay_step, reorder_states
    a, v, k, q = _token(1)
    parents = torch.tensor(PARENTS, device="cuda")
    slots = torch.arange(B, device="cuda", dtype=torch.int32)
    return {"step": lambda s: decay_step(s, a, v, k, q),
            "step_python": lambda s: decay_step(s, a.double(), v, k, q),
            "step_parents": lambda s: decay_step(s, a, v, k, q, parents=parents),
            "reorder": lambda s: reorder_states(s, parents),
            "reorder_python": lambda s: reorder_states(s, parents, slots.view(2, 4))}


UPDATES = ["step", "step_python", "step_parents", "reorder", "reorder_python"]


@pytest.mark.parametrize("name", UPDATES)
def test_saved_states_that_were_updated_are_not_used(name):
    """autograd has saved the final states of a forward for the loss on them; once they are updated in place, its backward raises."""
    from gla_jax_amd import chunk_decay
    update = _updates()[name]
    g = torch.Generator().manual_seed(2)
    rows = [torch.randn(B, 20, H, D, generator=g).cuda() for _ in range(3)]
    for alias in (lambda t: t.detach(), lambda t: t, lambda t: t.detach()[:]):
        h0 = _states(2).requires_grad_()
        hT, _ = chunk_decay(h0, torch.full((H,), -0.1, device="cuda"), *rows)
        loss = (hT * hT).sum()
        with torch.no_grad():
            update(alias(hT))
        with pytest.raises(RuntimeError, match="inplace operation"):
            loss.backward()


@pytest.mark.parametrize("name", UPDATES)
def test_versions(name):
    """A call that updates states counts as one, whatever memory they are a view of; one that is refused does not."""
    from gla_jax_amd import decay_step, reorder_states
    update = _updates()[name]
    pool = torch.zeros(2, B, H, D, D, device="cuda")
    states, before = pool[1], pool._version
    update(states)
    assert pool._version > before and states._version == pool._version
    before = pool._version
    with pytest.raises(AssertionError):
        decay_step(states[:4], *_token(1))
    with pytest.raises(AssertionError):
        reorder_states(states[:4], torch.tensor(PARENTS, device="cuda"))
    assert pool._version == before
    with torch.inference_mode():                 # normal arrays have a version here too, those that are made here none
        update(states)
        made = torch.zeros(B, H, D, D, device="cuda")
        update(made)
    assert pool._version > before
    update(made)
    want = torch.zeros(B, H, D, D, device="cuda")
    update(want)
    update(want)
    assert torch.equal(made, want)


def _serve(states, other, logits, scores, a, v, k, q):
    """A step of a beam search: the candidates, and the states behind them in both ways."""
    from gla_jax_amd import beam_select, decay_step, reorder_states
    scores, parents, tokens = beam_select(logits, scores)
    out = decay_step(states, a, v, k, q, parents=parents)
    reorder_states(other, parents)
    return scores, parents, tokens, out, other.sum(-1)


def _search(seed):
    g = torch.Generator().manual_seed(seed)
    logits, scores = torch.randn(2, 4, 300, generator=g).cuda(), -torch.rand(2, 4, generator=g).cuda()
    return [_states(seed), _states(seed + 1), logits, scores, *_token(seed)]


def test_traced_calls_compute_on_new_inputs():
    """torch.jit.trace records the calls themselves, not the buffers that they fill or the values that they found."""
    traced = torch.jit.trace(_serve, tuple(_search(3)), check_trace=False)
    for seed in (5, 7, 9):
        mine, want = _search(seed), _search(seed)
        for _ in range(3):
            for x, y in zip(traced(*mine), _serve(*want)):
                assert torch.equal(x, y)
            assert torch.equal(mine[0], want[0]) and torch.equal(mine[1], want[1])


@pytest.mark.parametrize("pooled", [False, True])
def test_traced_steps_update_their_states(pooled):
    from gla_jax_amd import decay_step
    slots = torch.tensor([3, -1, 0, 7, 1, 2, 6, 4], device="cuda") if pooled else None
    fn = lambda s, *rows: decay_step(s, *rows, slots)  # noqa: E731
    traced = torch.jit.trace(fn, (_states(1), *_token(1)), check_trace=False)
    mine, want = _states(2), _states(2)
    for seed in (2, 3, 4, 5):
        a, v, k, q = _token(seed)
        # rows in another layout than the traced ones
        spread = torch.stack((v, v), -1)[..., 0]
        assert torch.equal(traced(mine, a, spread, k, q), fn(want, a, v, k, q)) and torch.equal(mine, want)


def test_traced_calls_check_what_they_are_given():
    """States of another shape or layout than the traced ones are refused, as in a plain call."""
    from gla_jax_amd import decay_step, reorder_states
    traced = torch.jit.trace(decay_step, (_states(1), *_token(1)), check_trace=False)
    for other in (_states(1)[:4], _states(1)[:, :, :16].contiguous(), _states(1).transpose(2, 3), _states(1).double()):
        before = other.clone()
        with pytest.raises(Exception, match="states"):
            traced(other, *_token(1))
        assert torch.equal(other, before)
    parents = torch.tensor(PARENTS, device="cuda")
    traced = torch.jit.trace(lambda s, p: reorder_states(s, p), (_states(1), parents), check_trace=False)
    for other in (_states(1)[:4], _states(1).transpose(2, 3)):
        with pytest.raises(Exception, match="states"):
            traced(other, parents)


def test_forward_mode_tangents_are_refused():
    """There is no forward-mode rule: a call on an array with a tangent raises before it updates anything, also where no gradient is
    asked for, instead of returning results without one."""
    import torch.autograd.forward_ad as fwAD
    from gla_jax_amd import beam_select, decay_step, reorder_states
    parents = torch.tensor(PARENTS, device="cuda")
    logits, scores = torch.randn(2, 4, 50, device="cuda"), torch.zeros(2, 4, device="cuda")
    arrays = [_states(1), *_token(1)]
    calls = [(lambda *x: decay_step(*x), arrays), (lambda *x: decay_step(*x, parents=parents), arrays), (lambda s: reorder_states(s, parents), arrays[:1]),
             (beam_select, [logits, scores])]
    with fwAD.dual_level():
        for fn, plain in calls:
            for i, x in enumerate(plain):
                dual = list(plain)
                dual[i] = fwAD.make_dual(x.clone(), torch.ones_like(x))
                before = [t.clone() for t in dual]
                for mode in (torch.enable_grad, torch.no_grad):
                    with mode(), pytest.raises(RuntimeError, match="forward-mode"):
                        fn(*dual)
                for t, y in zip(dual, before):
                    assert torch.equal(t, y)
    for fn, plain in calls:
        before = [t.clone() for t in plain]
        with pytest.raises(RuntimeError):
            torch.func.jvp(fn, tuple(plain), tuple(torch.ones_like(t) for t in plain))
        for t, y in zip(plain, before):
            assert torch.equal(t, y)


@pytest.mark.parametrize("ragged", [False, True])
def test_traced_sequences_check_what_they_are_given(ragged):
    """A recorded chunk_decay computes on other lengths and refuses arrays that do not fit each other."""
    from gla_jax_amd import chunk_decay
    g = torch.Generator().manual_seed(4)
    rows = lambda T, n=B: [torch.randn(n, T, H, D, generator=g).cuda() for _ in range(3)]  # noqa: E731
    fn = lambda h0, a, v, k, q, *n: chunk_decay(h0, a, v, k, q, *n)  # noqa: E731
    lengths = (torch.arange(B, device="cuda", dtype=torch.int32),) if ragged else ()
    head = torch.full((H,), -0.1, device="cuda")
    traced = torch.jit.trace(fn, (_states(1), head, *rows(20), *lengths), check_trace=False)
    new = (_states(2), head, *rows(70), *lengths)
    for x, y in zip(traced(*new), fn(*new)):
        assert torch.equal(x, y)
    h0, a, v, k, q = new[:5]
    for other in ((h0[:4], a, v, k, q), (h0[..., :16].contiguous(), a, v, k, q), (h0, a, v, k[:, :30], q), (h0, a, v, k, q[:, :30]),
                  (h0, a, v, k[:4], q[:4]), (h0, a, v, k.bfloat16(), q)):
        with pytest.raises(Exception, match="chunk_decay"):
            traced(*other, *lengths)
    if ragged:
        for n in (lengths[0][:4], lengths[0].long()):
            with pytest.raises(Exception, match="chunk_decay"):
                traced(*new[:5], n)
