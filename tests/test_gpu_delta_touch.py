"""chunk_delta's gradients where value columns go 32 to a workgroup and 32 does not divide them: the last workgroup has half of its columns."""
import pytest
import torch

from gla_jax_amd import chunk_delta
from tests.delta_reference import check_step, inputs, step

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("case", [
    # B, T, H, HK, DK, DV, dtype: more than 256 groups of 16 columns, so that they go in pairs
    (12, 32, 8, 8, 128, 48, F32), (24, 20, 4, 4, 112, 48, F32), (12, 70, 8, 4, 128, 48, F32), (12, 64, 8, 8, 128, 48, BF16), (8, 33, 8, 8, 96, 80, BF16),
    (9, 31, 8, 8, 128, 112, F32)],
    ids=lambda c: "x".join(str(x).replace("torch.", "") for x in c))
def test_half_a_workgroup_of_columns(case):
    x = inputs(*case, seed=50)
    check_step(step(chunk_delta, *x), *x)
