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
