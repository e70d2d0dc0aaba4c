"""chunk_delta on the GPU within what its results' own rounding leaves: the bounds of delta_precision.py."""
import pytest
import torch

from gla_jax_amd import chunk_delta
from tests.delta_precision import CHANGED, RESULTS, bound_of_floats, changed, off
from tests.delta_reference import inputs, reference, step

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

# B, T, H, HK, DK, DV, and gates; the third in segments, the last two of 32 columns a workgroup
CASES = [
    ((1, 192, 2, 2, 128, 128), dict(decay="token")), ((2, 300, 4, 2, 64, 48), dict(decay="mild", beta="ends")),
    ((1, 4100, 2, 2, 64, 32), dict(decay="token")), ((6, 130, 8, 8, 128, 128), dict(decay="resets")), ((20, 70, 8, 4, 64, 64), dict(decay="head")),
]
ids = lambda c: "x".join(str(x) for x in c) if isinstance(c, tuple) else None  # noqa: E731
_found = {}


def found(sizes, gates, dtype=BF16):
    """Name -> (the kernels' result, the exact one, what its error is a share of), made once for the tests of a case."""
    key = (sizes, tuple(sorted(gates.items())), dtype)
    if key not in _found:
        x = inputs(*sizes, dtype=dtype, seed=40, **gates)
        exact = reference(*x[:6], None, x[6], x[7], 64 if dtype == BF16 else 32)
        got = [t.cpu() for t in step(chunk_delta, *x)]
        _found[key] = {n: (s, t, exact[8] if n == "dlog_decay" else None) for n, s, t in zip(RESULTS, got, exact)}
    return _found[key]


@pytest.mark.parametrize("sizes, gates", CASES, ids=ids)
def test_out(sizes, gates):
    share = changed(*found(sizes, gates)["out"][:2])
    assert share <= CHANGED


@pytest.mark.parametrize("sizes, gates", CASES, ids=ids)
def test_dkey(sizes, gates):
    share = changed(*found(sizes, gates)["dkey"][:2])
    assert share <= CHANGED
