"""The order of token_logprobs' alternatives where logits are infinite or not numbers: +inf first, NaN as -inf, equal ones by their tokens."""
import math

import pytest
import torch

from gla_jax_amd import token_logprobs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [40, 5001])
def test_infinities_first_and_nan_last(V, dtype):
    x = torch.randn(6, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    x[0, 30] = math.inf
    x[1, [31, 7]] = math.inf
    x[2, 9], x[2, 3] = math.inf, math.nan
    x[3, ::2] = math.nan
    x[4, 1:] = math.nan
    x[5, :], x[5, 20] = -math.inf, math.inf
    near, index = token_logprobs(x, torch.zeros(6, device="cuda", dtype=torch.int64), 9)[2:]
    order = torch.where(torch.isnan(x), -math.inf, x.float()).sort(dim=-1, descending=True, stable=True)[1][:, :9]
    assert torch.equal(index, order)
    assert torch.isnan(near).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_next_tokens_with_and_without_the_last_position(dtype):
    """Rows that skip the last position of each sequence, which are copied, and all rows with a token there that does not count."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(3, 8, 1001, device="cuda", generator=g).to(dtype)
    labels = torch.randint(1001, (3, 8), device="cuda", generator=g)
    behind = torch.cat([labels[:, 1:], torch.full((3, 1), -100, device="cuda")], 1)
    leaves = [x.detach().clone().requires_grad_() for _ in range(2)]
    short, long = token_logprobs(leaves[0][:, :-1], labels[:, 1:], 4), token_logprobs(leaves[1], behind, 4)
    r = torch.randn(2, 3, 8, device="cuda", generator=g)
    one, = torch.autograd.grad(short[:2], [leaves[0]], tuple(r[:, :, :-1]))
    all_, = torch.autograd.grad(long[:2], [leaves[1]], tuple(r))
    assert torch.equal(short[3], long[3][:, :-1]) and not all_[:, -1].any() and not one[:, -1].any()
    # (rows of odd length begin elsewhere within 16 bytes in a copy, and are summed in another order: 2^-21 + 2^-23 (log 1001 + |log p|) twice)
    for s, t in zip(short[:3], long[:3]):
        assert float((s - t[:, :-1]).abs().max()) <= 2 * (2.0 ** -21 + 2.0 ** -23 * 20)
    share = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18
    assert float((one.float() - all_.float()).abs().max()) <= share * float(all_.float().abs().max())
