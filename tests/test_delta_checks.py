"""What chunk_delta, delta_step and token_logprobs refuse before anything is launched: on the host through the C ABI, and in Python on fake arrays
that say they lie on a GPU."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from gla_jax_amd import _lib, chunk_delta, delta_step, token_logprobs

F32, BF16 = _lib.GLA_F32, _lib.GLA_BF16


@pytest.fixture
def zeros():
    with FakeTensorMode():
        yield lambda *shape, device="cuda:0", dtype=torch.float32, **more: torch.zeros(*shape, device=device, dtype=dtype, **more)


def _sequence(zeros, **changed):
    x = {"hidden_init": zeros(2, 4, 32, 16), "log_decay": zeros(2, 10, 4), "beta": zeros(2, 10, 4), "value": zeros(2, 10, 4, 16),
         "key": zeros(2, 10, 2, 32), "query": zeros(2, 10, 2, 32)}
    return {**x, **changed}


def test_sequences_refused(zeros):
    refused = lambda error, match, **x: pytest.raises(error, chunk_delta, **_sequence(zeros, **x)).match(match)  # noqa: E731
    refused(TypeError, "Tensor", beta=0.5)
    refused(ValueError, "GPU", key=torch.zeros(2, 10, 2, 32, device="cpu"))
    for name in ("hidden_init", "log_decay", "beta", "value", "key", "query"):
        refused(ValueError, "device", **{name: zeros(*_sequence(zeros)[name].shape, device="cuda:1")})
    refused(AssertionError, "value", value=zeros(4, 16))
    refused(AssertionError, "key", key=zeros(2, 9, 2, 32), query=zeros(2, 9, 2, 32))
    refused(AssertionError, "query", query=zeros(2, 10, 2, 16))
    refused(AssertionError, "divide", key=zeros(2, 10, 3, 32), query=zeros(2, 10, 3, 32))
    refused(AssertionError, "hidden_init", hidden_init=zeros(2, 4, 16, 32))
    for name in ("log_decay", "beta"):
        refused(AssertionError, name, **{name: zeros(2, 10, 2)})
        refused(AssertionError, name, **{name: zeros(2)})
        refused(TypeError, "floating", **{name: zeros(2, 10, 4, dtype=torch.int32)})
    refused(TypeError, "dtype", key=zeros(2, 10, 2, 32, dtype=torch.bfloat16))
    refused(TypeError, "dtype", **{n: zeros(*_sequence(zeros)[n].shape, dtype=torch.float16) for n in ("value", "key", "query")})
    refused(AssertionError, "128", hidden_init=zeros(2, 4, 144, 16), key=zeros(2, 10, 2, 144), query=zeros(2, 10, 2, 144))
    refused(AssertionError, "256", hidden_init=zeros(2, 4, 32, 272), value=zeros(2, 10, 4, 272))
    refused(AssertionError, "lengths", lengths=zeros(3, dtype=torch.int32))
    refused(AssertionError, "lengths", lengths=zeros(2))


def _token(zeros, **changed):
    x = {"states": zeros(6, 4, 32, 16), "log_decay": zeros(6, 4), "beta": zeros(6, 4), "value": zeros(6, 4, 16), "key": zeros(6, 2, 32),
         "query": zeros(6, 2, 32)}
    return {**x, **changed}


def test_steps_refused(zeros):
    refused = lambda error, match, **x: pytest.raises(error, delta_step, **_token(zeros, **x)).match(match)  # noqa: E731
    refused(ValueError, "GPU", value=torch.zeros(6, 4, 16, device="cpu"))
    refused(ValueError, "device", beta=zeros(6, 4, device="cuda:1"))
    refused(AssertionError, "states", states=zeros(6, 4, 16, 32))
    refused(AssertionError, "6 rows", states=zeros(5, 4, 32, 16))
    refused(AssertionError, "dense", states=zeros(6, 4, 16, 32).transpose(2, 3))
    refused(TypeError, "states", states=zeros(6, 4, 32, 16, dtype=torch.float64))
    refused(AssertionError, "value", value=zeros(6, 1, 4, 16))
    refused(AssertionError, "key", key=zeros(5, 2, 32), query=zeros(5, 2, 32))
    refused(AssertionError, "log_decay", log_decay=zeros(6, 2))
    refused(AssertionError, "beta", beta=zeros(6, 2))
    refused(AssertionError, "multiples of 16", states=zeros(6, 4, 32, 24), value=zeros(6, 4, 24))
    refused(AssertionError, "slots", slots=zeros(5, dtype=torch.int64))
    for name in _token(zeros):
        refused(RuntimeError, "no gradient", **{name: zeros(*_token(zeros)[name].shape, requires_grad=True)})


def test_logprobs_refused(zeros):
    tokens = zeros(6, dtype=torch.int64)
    refused = lambda error, match, *x: pytest.raises(error, token_logprobs, *x).match(match)  # noqa: E731
    refused(TypeError, "Tensor", [[1.0]], tokens)
    refused(ValueError, "GPU", zeros(6, 50), torch.zeros(6, dtype=torch.int64, device="cpu"))
    refused(ValueError, "device", zeros(6, 50), zeros(6, dtype=torch.int64, device="cuda:1"))
    refused(TypeError, "float32 or bfloat16", zeros(6, 50, dtype=torch.float16), tokens)
    refused(TypeError, "int32 or int64", zeros(6, 50), zeros(6))
    refused(AssertionError, "shape", zeros(6, 50), zeros(5, dtype=torch.int64))
    refused(AssertionError, "shape", zeros(2, 3, 50), tokens)
    refused(AssertionError, "V", zeros(6, 0), tokens)
    for top in (-1, 51, 65):
        refused(AssertionError, "alternatives", zeros(6, 50), tokens, top)
    refused(AssertionError, "alternatives", zeros(6, 100), tokens, 65)


def test_entry_points_reject_bad_arguments_without_touching_the_gpu():
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    a = (ctypes.addressof(buf) + 15) & ~15          # a 16-byte aligned, non-null host address (never dereferenced)
    strides = lambda *s: (ctypes.c_int64 * len(s))(*s)  # noqa: E731

    def fwd(B=1, T=8, H=4, HK=2, DK=32, DV=32, dt=BF16, hd=F32, st=None, h0=a, g=a, b=a, v=a, n=None, states=None, ws=None, size=0):
        return lib.gla_delta_fwd(None, B, T, H, HK, DK, DV, dt, hd, st, h0, g, b, v, a, a, n, a, a, states, ws, size)

    assert fwd(h0=None) == -1 and fwd(v=None) == -1 and fwd(g=None) == -1 and fwd(b=None) == -1
    for bad in ({"B": 0}, {"T": -1}, {"H": 0}, {"HK": 3}, {"HK": 0}, {"DK": 40}, {"DK": 144}, {"DV": 8}, {"DV": 272}, {"T": 1 << 31}, {"H": 1 << 20, "HK": 1 << 20}, {"B": 1 << 21, "DV": 256},
                {"B": 1 << 12, "T": 1 << 16}):
        assert fwd(**bad) == -2, bad
    assert fwd(dt=7) == -3 and fwd(hd=7) == -3
    assert fwd(h0=a + 8) == -6 and fwd(v=a + 2) == -6 and fwd(g=a + 2) == -6 and fwd(b=a + 2) == -6 and fwd(n=a + 1) == -6 and fwd(states=a + 8) == -6
    dense = (32, 4, 1, 32, 4, 1, 1024, 128, 32, 512, 64, 32, 512, 64, 32)
    assert fwd(st=strides(*dense[:7], 129, *dense[8:])) == -6                    # rows that do not begin on 16 bytes
    assert fwd(st=strides(*dense[:7], 1 << 23, *dense[8:])) == -2                # and rows too far apart
    need = lib.gla_delta_fwd_workspace_bytes(1, 8, 4, 2, 32, 32, BF16)
    assert need > 0 and fwd() == -5 and fwd(ws=a, size=need - 1) == -5 and fwd(ws=a + 8, size=need) == -6
    assert lib.gla_delta_fwd_workspace_bytes(1, 8, 4, 3, 32, 32, BF16) == 0

    def bwd(T=8, HK=4, DK=32, dt=BF16, states=a, do=a, dv=a, db=a, ws=None, size=0):
        return lib.gla_delta_bwd(None, 1, T, 4, HK, DK, 32, dt, F32, None, a, a, a, a, a, None, states, a, do, a, a, db, dv, a, a, ws, size)

    assert bwd(states=None) == -1 and bwd(do=None) == -1 and bwd(dv=None) == -1 and bwd(db=None) == -1
    assert bwd(DK=33) == -2 and bwd(dt=2) == -3 and bwd(do=a + 8) == -6 and bwd(db=a + 2) == -6
    need = lib.gla_delta_bwd_workspace_bytes(1, 8, 4, 2, 32, 32, BF16)
    # a key head's gradient comes in parts, one of each head that shares it
    assert need >= lib.gla_delta_bwd_workspace_bytes(1, 8, 4, 4, 32, 32, BF16) + 2 * 2 * 8 * 2 * 32 * 4 - 4096
    assert bwd(HK=2) == -5 and bwd(HK=2, ws=a, size=need - 1) == -5

    def step(pool=6, B=6, HK=4, DK=32, beams=0, st=BF16, states=a, slots=None, parents=None, wide=1, b=a, v=a):
        return lib.gla_delta_step(None, pool, B, 4, HK, DK, 32, beams, BF16, st, wide, None, a, b, v, a, a, slots, parents, states, a)

    assert step(states=None) == -1 and step(b=None) == -1 and step(beams=2) == -1
    for bad in ({"pool": 0}, {"B": 0}, {"pool": 5}, {"HK": 3}, {"DK": 8}, {"beams": 4, "parents": a}, {"beams": -1}, {"B": 65, "pool": 65, "beams": 65, "parents": a}):
        assert step(**bad) == -2, bad
    assert step(st=9) == -3 and step(states=a + 8) == -6 and step(slots=a + 4) == -6 and step(v=a + 2) == -6 and step(b=a + 2) == -6

    def logprobs(N=3, V=50, top=0, dt=F32, row=50, wide=1, x=a, t=a, g=a, h=a, s=None, near=None, index=None):
        return lib.gla_token_logprobs(None, N, V, top, dt, row, wide, x, t, g, h, s, near, index)

    assert logprobs(x=None) == -1 and logprobs(t=None) == -1 and logprobs(g=None) == -1 and logprobs(h=None) == -1 and logprobs(top=1) == -1
    for bad in ({"N": -1}, {"N": 1 << 31}, {"V": 0}, {"V": 1 << 31, "row": 1 << 31}, {"row": 49}, {"top": -1}, {"top": 51}, {"top": 65, "V": 100, "row": 100}):
        assert logprobs(**bad) == -2, bad
    assert logprobs(N=0, x=None) == 0 and logprobs(dt=5) == -3
    assert logprobs(x=a + 2) == -6 and logprobs(t=a + 4) == -6 and logprobs(t=a + 2, wide=0) == -6 and logprobs(s=a + 2) == -6
    assert logprobs(top=1, near=a, index=a + 4) == -6

    def gradient(N=3, V=50, dt=F32, row=50, to=50, x=a, d=a, s=a, g=None):
        return lib.gla_token_logprobs_bwd(None, N, V, dt, row, to, 1, x, a, s, a, g, None, d)

    assert gradient(x=None) == -1 and gradient(d=None) == -1 and gradient(s=None) == -1 and gradient(dt=9) == -3
    for bad in ({"V": 0}, {"row": 49}, {"to": 49}, {"N": 1 << 31}):
        assert gradient(**bad) == -2, bad
    # rows of the gradient begin where those of the logits do, within 16 bytes
    assert gradient(d=a + 4) == -6 and gradient(to=51) == -6 and gradient(g=a + 1) == -6


def test_sizes_of_what_the_forward_leaves():
    lib = _lib.load()
    # the states before the chunks of 64 tokens (float data 32) and at the end, features in pairs of tiles, and what the tokens miss, in 32 bits
    assert lib.gla_delta_states_bytes(2, 130, 4, 2, 32, 48, BF16) == 2 * 4 * (4 * 32 * 48 + 3 * 64 * 48) * 4
    assert lib.gla_delta_states_bytes(2, 130, 4, 2, 48, 48, F32) == 2 * 4 * (6 * 64 * 48 + 5 * 32 * 48) * 4
    assert lib.gla_delta_states_bytes(2, 0, 4, 2, 32, 48, BF16) == 2 * 4 * 32 * 48 * 4
    # few long sequences run as segments, which leave summaries
    whole = lib.gla_delta_fwd_workspace_bytes(64, 4096, 8, 8, 64, 64, BF16)
    long = lib.gla_delta_fwd_workspace_bytes(1, 64 * 4096, 8, 8, 64, 64, BF16)
    assert long >= whole + 8 * 7 * 2 * 64 * 64 * 4
