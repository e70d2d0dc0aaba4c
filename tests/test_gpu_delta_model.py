"""chunk_delta, delta_step and token_logprobs as a model uses them: trained on padded rows, prompted, decoded token by token, scored.

All in float32.  Tolerances.  The operators' results are off by 1e-5 of their norm at most (tests/delta_reference.py) and 2^-20 absolutely
(test_gpu_logprobs.py); torch's products of d terms add sqrt(d) 2^-24 each.  A logit sums 128 features of out times weights of their inverse root: 1e-5 of
the logits' norm, and with the projections in front of it three such errors in a row.  Log probabilities move by at most twice as much as the
logits do: bound 1e-4.  Gradients pass through the same products once more: 2e-4 of their norm."""
import math

import pytest
import torch

from gla_jax_amd import chunk_delta, delta_step, token_logprobs
from tests.delta_reference import reference

pytestmark = pytest.mark.gpu
B, T, H, HK, DK, DV, V, D = 3, 90, 4, 2, 16, 32, 501, 32


def weights(seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"embed": r(V, D), "rows": r(D, 2 * HK * DK + H * DV) / math.sqrt(D), "gates": r(D, 2 * H) / math.sqrt(D), "head": r(H * DV, V) / math.sqrt(H * DV)}


def project(w, tokens):
    x = w["embed"][tokens]
    q, k, v = (x @ w["rows"]).split([HK * DK, HK * DK, H * DV], -1)
    a, b = (x @ w["gates"]).split([H, H], -1)
    unit = lambda y: torch.nn.functional.normalize(y.unflatten(-1, (HK, DK)), dim=-1)  # noqa: E731
    return torch.nn.functional.logsigmoid(a + 2), b.sigmoid(), v.unflatten(-1, (H, DV)), unit(k), unit(q)


def forward(w, tokens, lengths, h0, attend):
    hT, out = attend(h0, *project(w, tokens), lengths)
    return hT, out.flatten(-2) @ w["head"]


class Recurrence(torch.autograd.Function):
    """The recurrence of tests/delta_reference.py with its own gradients, in 64 bits."""

    @staticmethod
    def forward(ctx, *x):
        ctx.x = x
        return reference(*x)

    @staticmethod
    def backward(ctx, dh, do):
        return reference(*ctx.x, dh=dh, do=do)[2:8] + (None,)


def data(seed):
    g = torch.Generator().manual_seed(seed)
    tokens, lengths = torch.randint(V, (B, T), generator=g), [T, 41, 64]
    targets = torch.full((B, T), -100)
    for i, n in enumerate(lengths):
        targets[i, :n - 1] = tokens[i, 1:n]
    return tokens, torch.tensor(lengths, dtype=torch.int32), targets, torch.zeros(B, H, DK, DV)


def test_training_step():
    """The cross entropy of padded rows with a bonus for entropy: the loss and the gradient of every weight."""
    tokens, lengths, targets, h0 = data(1)
    w = {n: x.cuda().requires_grad_() for n, x in weights(0).items()}
    _, logits = forward(w, tokens.cuda(), lengths.cuda(), h0.cuda(), chunk_delta)
    given, entropy = token_logprobs(logits, targets.cuda())
    loss = -(given + 0.01 * entropy).sum() / 50
    grads = torch.autograd.grad(loss, list(w.values()))
    exact = {n: x.double().requires_grad_() for n, x in weights(0).items()}
    _, logits = forward(exact, tokens, lengths, h0.double(), lambda *x: Recurrence.apply(*x))
    p = logits.log_softmax(-1)
    counts = (targets >= 0).double()
    want = p.gather(-1, targets.clamp(min=0)[..., None])[..., 0] * counts
    spread = -(p.exp() * p).sum(-1) * counts
    exact_loss = -(want + 0.01 * spread).sum() / 50
    assert float((given.double().cpu() - want).abs().max()) <= 1e-4 and float((entropy.double().cpu() - spread).abs().max()) <= 1e-4
    for n, x, y in zip(w, grads, torch.autograd.grad(exact_loss, list(exact.values()))):
        assert float((x.double().cpu() - y).norm()) <= 2e-4 * float(y.norm()), n


def test_prompts_then_single_tokens():
    """A prompt of ragged rows into a pool of states, 12 tokens one by one, and what they score: as if the whole rows had been given at once."""
    tokens, lengths, _, h0 = data(2)
    w = {n: x.cuda() for n, x in weights(3).items()}
    steps, g = 12, torch.Generator().manual_seed(4)
    more = torch.randint(V, (B, steps), generator=g)
    slots = torch.tensor([4, 0, 2], device="cuda")
    pool = torch.full((6, H, DK, DV), 7.0, device="cuda")
    with torch.no_grad():
        hT, logits = forward(w, tokens.cuda(), lengths.cuda(), h0.cuda(), chunk_delta)
        pool[slots] = hT
        last = logits[torch.arange(B), (lengths - 1).tolist()]
        scores, best = [], []
        for i in range(steps):
            given, _, near, index = token_logprobs(last, more[:, i].cuda(), 5)
            scores.append(given)
            best.append((near, index))
            a, b, v, k, q = project(w, more[:, i].cuda())
            out = delta_step(pool, a, b, v, k, q, slots=slots)
            last = out.flatten(-2) @ w["head"]
        rest = [i for i in range(6) if i not in slots.tolist()]
        assert bool((pool[rest] == 7.0).all())
        for r in range(B):
            whole = torch.cat([tokens[r, :int(lengths[r])], more[r]]).cuda()
            hT, logits = forward(w, whole, None, h0[r].cuda(), chunk_delta)
            n = int(lengths[r])
            given, _, near, index = token_logprobs(logits[n - 1:n - 1 + steps], whole[n:], 5)
            assert float((torch.stack(scores)[:, r] - given).abs().max()) <= 1e-4
            assert float((torch.stack([x[r] for x, _ in best]) - near).abs().max()) <= 1e-4
            assert float((pool[slots[r]] - hT).norm()) <= 1e-4 * float(hT.norm())
