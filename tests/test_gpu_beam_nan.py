"""beam_select on logits that are not numbers, of every bit pattern: they count as -inf."""
import pytest
import torch

from tests.test_gpu_beam import _apart, _check, _reference

pytestmark = pytest.mark.gpu

# quiet and signalling ones, of either sign
PATTERNS = {torch.bfloat16: [0x7fa0, 0xffa0, 0x7f81, 0x7fbf, 0x7fc0, 0xffff],
            torch.float32: [0x7fa00000, 0xffa00000, 0x7f800001, 0x7fbfffff, 0x7fc00000, 0xffffffff]}


def _put(x, where, pattern):
    bits = torch.int16 if x.dtype == torch.bfloat16 else torch.int32
    top = 1 << (15 if x.dtype == torch.bfloat16 else 31)
    x.view(bits)[..., where] = pattern - 2 * top if pattern >= top else pattern
    return x


# one stretch and several, rows that begin on 16 bytes and rows that do not, narrow and wide stretches
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G, W, V, num", [(1, 1, 8, 1), (1, 1, 9, 1), (2, 3, 1000, 1), (2, 3, 1001, 3), (2, 2, 8200, 4), (64, 2, 65536, 1), (64, 2, 65535, 2)])
def test_whatever_is_not_a_number_counts_as_minus_infinity(G, W, V, num, dtype):
    from gla_jax_amd import beam_select
    for seed in range(20):
        g = torch.Generator().manual_seed(seed)
        plain = (3.0 * torch.randn(G, W, V, generator=g)).to(dtype)
        scores = (-5.0 * torch.rand(G, W, generator=g)).cuda()
        # a thread's first places (it holds pieces of 16 bytes), its others, and a row's end
        places = torch.unique(torch.cat([torch.tensor([0, V - 1, V // 2]), 8 * torch.randint(V // 8, (3,), generator=g), torch.randint(V, (V // 20,), generator=g)]))
        plain[..., places] = float("nan")
        found = _reference(plain, scores, num)
        if all(_apart(found[i:i + 1]) for i in range(G)):
            break
    else:
        pytest.skip("candidates closer than 32-bit scores tell apart")
    for pattern in PATTERNS[dtype]:
        _check(beam_select(_put(plain.clone(), places, pattern).cuda(), scores, num), found, V)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 8, 24, 4096, 4097])
def test_beams_without_a_number(V, dtype):
    """Nothing but NaN: the first places, without a chance."""
    from gla_jax_amd import beam_select
    for pattern in PATTERNS[dtype]:
        x = _put(torch.zeros(2, 2, V, dtype=dtype), torch.arange(V), pattern).cuda()
        scores, parents, tokens = beam_select(x, torch.zeros(2, 2, device="cuda"), 1)
        assert torch.equal(scores, torch.full_like(scores, -float("inf"))) and not parents.any() and not tokens.any()
