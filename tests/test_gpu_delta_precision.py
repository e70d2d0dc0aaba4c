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
        exact = list(reference(*x[:6], None, x[6], x[7], 64 if dtype == BF16 else 32))
        if gates["decay"] == "head":          # one number a head: the sum over all tokens, whose errors add in quadrature
            exact[3], exact[8] = exact[3].sum((0, 1)), exact[8].square().sum((0, 1)).sqrt()
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


@pytest.mark.parametrize("name", ["dvalue", "dquery"])
@pytest.mark.parametrize("sizes, gates", CASES, ids=ids)
def test_other_16_bit_results(sizes, gates, name):
    share = changed(*found(sizes, gates)[name][:2])
    assert share <= CHANGED


@pytest.mark.parametrize("name", ["hidden_final", "dhidden_init", "dlog_decay", "dbeta"])
@pytest.mark.parametrize("sizes, gates", CASES, ids=ids)
def test_32_bit_results(sizes, gates, name):
    """A third part less is seen: test_delta_precision.py."""
    share = off(*found(sizes, gates)[name])
    assert share <= bound_of_floats(name, -(-sizes[1] // 64))


@pytest.mark.parametrize("name", RESULTS)
@pytest.mark.parametrize("sizes, gates", CASES[:2] + [((1, 2081, 2, 1, 64, 64), dict(decay="token"))] + CASES[3:4], ids=ids)
def test_results_of_32_bit_data(sizes, gates, name):
    share = off(*found(sizes, gates, F32)[name])
    assert share <= bound_of_floats(name, -(-sizes[1] // 32))
