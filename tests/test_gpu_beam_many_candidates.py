"""beam_select where the join of a search gets more candidates than its threads hold at once, and more that reach its bound than it has room
for: the largest searches over large vocabularies."""
import math

import pytest
import torch

from tests.test_gpu_beam import _apart, _check, _reference

pytestmark = pytest.mark.gpu

HELD, ROOM = 4096, 2048


def _join(x, scores, num):
    """How many candidates the join gets, and how many of them reach its bound: by stretches of 16384 values and 1024 threads, each of which
    names its largest; a wave's num-th name is a bound."""
    x = x.double().cpu()
    x = (x - torch.logsumexp(x, -1, keepdim=True) + scores.double().cpu()[:, None])
    W, V = x.shape
    splits = -(-V // 16384)
    padded = torch.full((W, splits * 16384), -math.inf, dtype=torch.float64)
    padded[:, :V] = x
    c = padded.view(W * splits, 16384).topk(num, -1)[0].flatten()
    threads = torch.full((-(-c.numel() // 1024) * 1024,), -math.inf, dtype=torch.float64)
    threads[:c.numel()] = c
    names = threads.view(-1, 1024).max(0)[0].view(16, 64)
    return c.numel(), int((c >= names.topk(num, -1)[0][:, -1].max()).sum())


def _problem(W, V, num, dtype):
    for seed in range(20):
        g = torch.Generator().manual_seed(seed)
        x, scores = (3.0 * torch.randn(1, W, V, generator=g)).to(dtype), -5.0 * torch.rand(1, W, generator=g)
        found = _reference(x, scores, num)
        if _apart(found):
            return x.cuda(), scores.cuda(), found
    raise AssertionError("no search whose candidates 32-bit scores tell apart")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("W, V, num", [(48, 40000, 64), (64, 19999, 64), (64, 131072, 32)])
def test_more_than_the_threads_hold(W, V, num, dtype):
    from gla_jax_amd import beam_select
    x, scores, found = _problem(W, V, num, dtype)
    count, reach = _join(x[0], scores[0], num)
    assert count > HELD and reach <= ROOM
    _check(beam_select(x, scores, num), found, V)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("W, V", [(64, 131072), (64, 131071)])
def test_more_than_there_is_room_for(W, V, dtype):
    from gla_jax_amd import beam_select
    x, scores, found = _problem(W, V, 64, dtype)
    count, reach = _join(x[0], scores[0], 64)
    assert count > HELD and reach > ROOM
    _check(beam_select(x, scores, 64), found, V)


def test_beams_that_have_ended_among_many():
    from gla_jax_amd import beam_select
    W, V = 64, 131072
    g = torch.Generator().manual_seed(1)
    x, scores = torch.randn(1, W, V, generator=g), -5.0 * torch.rand(1, W, generator=g)
    finished = torch.rand(1, W, generator=g) < 0.2
    x[finished] = math.nan
    scores[finished] -= 9.0
    found = _reference(x, scores, 64, finished, 7)
    assert _apart(found)
    _check(beam_select(x.cuda(), scores.cuda(), 64, finished.cuda(), 7), found, V)
