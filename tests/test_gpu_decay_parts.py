"""chunk_decay's gradients where several workgroups add to them, at odd sizes: the parts of one array follow each other in memory."""
import pytest
import torch

from tests.decay_reference import check_step, inputs, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B, T, H, HK, DK, DV", [(1, 77, 1, 1, 32, 256), (1, 1, 1, 1, 16, 256), (1, 77, 3, 1, 64, 256), (3, 45, 1, 1, 256, 32), (1, 131, 3, 3, 256, 256),
                                                 (1, 66, 1, 1, 256, 144), (1, 777, 1, 1, 64, 256)])
def test_an_odd_number_of_gates(B, T, H, HK, DK, DV, dtype):
    from gla_jax_amd import chunk_decay
    x = inputs(B, T, H, HK, DK, DV, dtype, seed=T + DK)
    check_step(step(chunk_decay, *x), *x)
