"""chunk_decay where it takes other kernels or cuts sequences: more workgroups than compute units, and ragged sequences as segments."""
import pytest
import torch

from tests.decay_reference import check, check_step, inputs, reference, step

pytestmark = pytest.mark.gpu


def _chunk():
    from gla_jax_amd import chunk_decay
    return chunk_decay


@pytest.mark.parametrize("DK, DV, dtype", [(64, 64, torch.bfloat16), (128, 64, torch.bfloat16), (64, 128, torch.bfloat16), (128, 128, torch.bfloat16),
                                           (96, 112, torch.bfloat16), (64, 64, torch.float32), (128, 64, torch.float32), (128, 128, torch.float32)])
def test_more_workgroups_than_compute_units(DK, DV, dtype):
    x = inputs(20, 70, 14, 7, DK, DV, dtype, seed=DK + DV)
    check_step(step(_chunk(), *x), *x)


@pytest.mark.parametrize("DK, DV, dtype", [(64, 64, torch.bfloat16), (128, 128, torch.bfloat16), (48, 96, torch.float32)])
@pytest.mark.parametrize("lengths", [[1100, 130, 0], [65, 700, 1], [64, 512, 1099], [1, 0, 0]])
def test_ragged_segments(lengths, DK, DV, dtype):
    """Sequences end in the first segment, at a segment's or a chunk's end, before the first token."""
    h0, a, v, k, q, dh, do = inputs(3, 1100, 2, 1, DK, DV, dtype, seed=sum(lengths))
    n = torch.tensor(lengths, device="cuda")
    past = torch.arange(1100, device="cuda")[None, :] >= n[:, None]
    v, k, q, a = v.clone(), k.clone(), q.clone(), a.clone()
    v[past], k[past], q[past], a[past] = float("nan"), float("inf"), -float("inf"), float("nan")
    got = step(_chunk(), h0, a, v, k, q, dh, do, n)
    assert not got[1][past].any() and not any(x[past].any() for x in got[3:])
    # (the rows behind the ends, which are zero, would only dilute the scale that single values are held to)
    exact = reference(h0, torch.where(past[..., None], 0.0, a), *(torch.where(past[..., None, None], 0.0, x) for x in (v, k, q)), n, dh, do)
    live = ~past
    for i, name in enumerate(("hidden_final", "out", "dhidden_init", "dlog_decay", "dvalue", "dkey", "dquery")):
        rows = i not in (0, 2)
        check(name, got[i][live] if rows else got[i], exact[i][live.cpu()] if rows else exact[i])
    for b, length in enumerate(lengths):
        if length == 0:
            assert torch.equal(got[0][b], h0[b]) and torch.equal(got[2][b], dh[b])


@pytest.mark.parametrize("lengths", [[1100, 130, 0, 600], [64, 1, 1100, 65]])
def test_ragged_segments_of_one_constant_a_head(lengths):
    h0, a, v, k, q, dh, do = inputs(4, 1100, 3, 3, 64, 128, decay="head", seed=2)
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    check_step(step(_chunk(), h0, a, v, k, q, dh, do, n), h0, a, v, k, q, dh, do, n)


def test_the_same_from_run_to_run():
    x = inputs(2, 900, 3, 1, 128, 256, seed=9)
    first = step(_chunk(), *x)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, step(_chunk(), *x)))
