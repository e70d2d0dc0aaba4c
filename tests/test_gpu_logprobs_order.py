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
