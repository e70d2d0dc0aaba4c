"""chunk_delta where the longest sequences are walked first: lengths of at most 64 sequences and more workgroups than compute units (256)."""
import pytest
import torch

from gla_jax_amd import chunk_delta
from tests.delta_reference import check_step, inputs, step

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def lengths_of(B, T, seed):
    """Repeated, none, negative and too large ones among them, in no order."""
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(1, T + 1, (B,), generator=g)
    at = torch.randperm(B, generator=g)
    for i, x in enumerate((0, 0, -5, T, T, T + 100, 17, 17, 17, 64, 64, 1)):
        n[at[i]] = x
    return n.to(torch.int32).cuda()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B, T, H, HK, DK, DV", [(40, 70, 8, 4, 32, 64), (64, 66, 6, 6, 64, 32), (65, 66, 6, 2, 64, 32), (16, 130, 8, 8, 128, 128)])
def test_lengths_in_no_order(B, T, H, HK, DK, DV, dtype):
    x = inputs(B, T, H, HK, DK, DV, dtype, seed=60)
    n = lengths_of(B, T, seed=B)
    past = torch.arange(T, device="cuda")[None, :] >= n[:, None]
    for t in (x[1], x[2], x[3], x[4], x[5], x[7]):
        t[past] = float("nan")                       # not read
    got = step(chunk_delta, *x, n)
    clean = [t.clone() for t in x]
    for t in (clean[1], clean[2], clean[3], clean[4], clean[5], clean[7]):
        t[past] = 0
    check_step(got, *clean, n)
    for t in (got[1], *got[3:]):
        assert not t[past].any()
    with torch.no_grad():
        assert all(torch.equal(s, t) for s, t in zip(got, chunk_delta(*x[:6], n)))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_same_bits_in_every_order(dtype):
    x = inputs(48, 100, 8, 4, 64, 64, dtype, seed=61)
    n = lengths_of(48, 100, seed=1)
    longest_first = torch.argsort(n.clamp(0, 100), descending=True, stable=True)
    sorted_ = step(chunk_delta, *(t[longest_first] for t in x), n[longest_first])
    for got, want in zip(step(chunk_delta, *x, n), sorted_):
        assert torch.equal(got[longest_first], want)


def test_the_same_bits_in_every_order_in_segments():
    """Two sequences of 100 chunks, whose summaries take 512 workgroups."""
    x = inputs(2, 6400, 4, 4, 128, 128, seed=62)
    n = torch.tensor([6400, 2900], device="cuda", dtype=torch.int32)
    one, other = step(chunk_delta, *x, n), step(chunk_delta, *(t.flip(0) for t in x), n.flip(0))
    assert all(torch.equal(s, t.flip(0)) for s, t in zip(one, other))
    whole = step(chunk_delta, *x)                    # (without lengths: no order)
    assert all(torch.equal(s[0], t[0]) for s, t in zip(one, whole))
