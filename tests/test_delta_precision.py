"""The bounds of delta_precision.py tell one rounding more from none: the chunked rule on the CPU with its operands in as many parts as the kernels hold, and in one
less."""
import pytest
import torch

from tests.delta_precision import CHANGED, RESULTS, bound_of_floats, changed, emulated, off
from tests.delta_reference import inputs, reference

CASES = [dict(decay="token"), dict(decay="mild", beta="ends")]


@pytest.fixture(scope="module", params=range(len(CASES)))
def case(request):
    x = inputs(1, 192, 2, 2, 128, 128, seed=request.param, device="cpu", **CASES[request.param])
    return x, reference(*x[:6], None, x[6], x[7])


def found(got, exact):
    """Name -> by how many times its bound a result is off."""
    r = {}
    for name, x, y in zip(RESULTS, got, exact):
        if x.dtype == torch.bfloat16:
            r[name] = changed(x, y) / CHANGED
        else:
            r[name] = off(x, y, exact[8] if name == "dlog_decay" else None) / bound_of_floats(name, 3)
    return r


def test_parts_as_the_kernels_hold_them(case):
    x, exact = case
    r = found(emulated(*x), exact)
    assert max(r.values()) <= 1.0, r


@pytest.mark.parametrize("planted, seen", [
    (dict(out_scores=1), {"out"}), (dict(dkey_cotangent=1), {"dkey"}),
    (dict(many=2), {"hidden_final", "dhidden_init", "dbeta"})], ids=["scores", "cotangent", "all"])
def test_one_part_less_is_seen(case, planted, seen):
    x, exact = case
    r = found(emulated(*x, **planted), exact)
    assert all(r[name] > 1.0 for name in seen), r
