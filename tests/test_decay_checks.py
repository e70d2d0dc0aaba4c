"""What chunk_decay, decay_step, beam_select and reorder_states refuse before anything is launched: on the host through the C ABI, and in
Python on fake arrays that say they lie on a GPU."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from gla_jax_amd import _lib, beam_select, chunk_decay, decay_step, reorder_states

F32, BF16 = _lib.GLA_F32, _lib.GLA_BF16


@pytest.fixture
def zeros():
    with FakeTensorMode():
        yield lambda *shape, device="cuda:0", dtype=torch.float32, **more: torch.zeros(*shape, device=device, dtype=dtype, **more)


def _sequence(zeros, **changed):
    x = {"hidden_init": zeros(2, 4, 32, 16), "log_decay": zeros(2, 10, 4), "value": zeros(2, 10, 4, 16), "key": zeros(2, 10, 2, 32),
         "query": zeros(2, 10, 2, 32)}
    return {**x, **changed}


def test_sequences_refused(zeros):
    refused = lambda error, match, **x: pytest.raises(error, chunk_decay, **_sequence(zeros, **x)).match(match)  # noqa: E731
    refused(TypeError, "Tensor", value=[1.0])
    refused(ValueError, "GPU", key=torch.zeros(2, 10, 2, 32, device="cpu"))
    for name in ("hidden_init", "log_decay", "value", "key", "query"):
        refused(ValueError, "device", **{name: zeros(*_sequence(zeros)[name].shape, device="cuda:1")})
    refused(AssertionError, "key", key=zeros(2, 9, 2, 32), query=zeros(2, 9, 2, 32))
    refused(AssertionError, "query", query=zeros(2, 10, 2, 16))
    refused(AssertionError, "divide", key=zeros(2, 10, 3, 32), query=zeros(2, 10, 3, 32))
    refused(AssertionError, "hidden_init", hidden_init=zeros(2, 4, 16, 32))
    refused(AssertionError, "log_decay", log_decay=zeros(2, 10, 2))
    refused(AssertionError, "log_decay", log_decay=zeros(2))
    refused(TypeError, "dtype", key=zeros(2, 10, 2, 32, dtype=torch.bfloat16))
    refused(TypeError, "dtype", **{n: zeros(*_sequence(zeros)[n].shape, dtype=torch.float16) for n in ("value", "key", "query")})
    refused(TypeError, "floating", log_decay=zeros(2, 10, 4, dtype=torch.int32))
    refused(AssertionError, "256", hidden_init=zeros(2, 4, 264, 16), key=zeros(2, 10, 2, 264), query=zeros(2, 10, 2, 264))
    refused(AssertionError, "lengths", lengths=zeros(3, dtype=torch.int32))
    refused(AssertionError, "lengths", lengths=zeros(2))


def _token(zeros, **changed):
    x = {"states": zeros(6, 4, 32, 16), "log_decay": zeros(6, 4), "value": zeros(6, 4, 16), "key": zeros(6, 2, 32), "query": zeros(6, 2, 32)}
    return {**x, **changed}


def test_steps_refused(zeros):
    refused = lambda error, match, **x: pytest.raises(error, decay_step, **_token(zeros, **x)).match(match)  # noqa: E731
    refused(ValueError, "GPU", value=torch.zeros(6, 4, 16, device="cpu"))
    refused(AssertionError, "states", states=zeros(6, 4, 16, 32))
    refused(AssertionError, "6 rows", states=zeros(5, 4, 32, 16))
    refused(AssertionError, "dense", states=zeros(6, 4, 16, 32).transpose(2, 3))
    refused(TypeError, "states", states=zeros(6, 4, 32, 16, dtype=torch.float64))
    refused(AssertionError, "value", value=zeros(6, 1, 4, 16))
    refused(AssertionError, "key", key=zeros(5, 2, 32), query=zeros(5, 2, 32))
    refused(AssertionError, "log_decay", log_decay=zeros(6, 2))
    refused(AssertionError, "slots", slots=zeros(5, dtype=torch.int64))
    refused(TypeError, "slots", slots=zeros(6))
    refused(AssertionError, "parents", parents=zeros(2, 2, dtype=torch.int64))
    refused(AssertionError, "65 beams", states=zeros(65, 4, 32, 16), log_decay=zeros(4), value=zeros(65, 4, 16), key=zeros(65, 2, 32),
            query=zeros(65, 2, 32), parents=zeros(1, 65, dtype=torch.int64))
    refused(RuntimeError, "no gradient", value=zeros(6, 4, 16, requires_grad=True))


def test_selections_refused(zeros):
    def refused(error, match, logits, scores, *more):
        with pytest.raises(error, match=match):
            beam_select(logits, scores, *more)

    x, s = zeros(2, 3, 100), zeros(2, 3)
    refused(ValueError, "GPU", torch.zeros(2, 3, 100, device="cpu"), s)
    refused(ValueError, "device", x, zeros(2, 3, device="cuda:1"))
    refused(AssertionError, "logits", zeros(100), zeros(1))
    refused(AssertionError, "scores", x, zeros(2, 2))
    refused(TypeError, "logits", zeros(2, 3, 100, dtype=torch.float16), s)
    for num in (0, -1, 65, 301):
        refused(AssertionError, "candidates", x, s, num)
    refused(AssertionError, "candidates", zeros(2, 3, 2), s, 7)
    refused(AssertionError, "candidates", zeros(2, 65, 100), zeros(2, 65))
    refused(AssertionError, "finished", x, s, 3, zeros(2, 2, dtype=torch.bool))
    refused(AssertionError, "finished", x, s, 3, zeros(2, 3))
    refused(AssertionError, "eos", x, s, 3, zeros(2, 3, dtype=torch.bool), 100)
    refused(AssertionError, "eos", x, s, 3, zeros(2, 3, dtype=torch.bool), -1)


def test_orders_refused(zeros):
    def refused(error, match, *args):
        with pytest.raises(error, match=match):
            reorder_states(*args)

    states, parents = zeros(6, 4, 8), zeros(2, 3, dtype=torch.int64)
    refused(ValueError, "GPU", torch.zeros(6, 4, device="cpu"), parents)
    refused(AssertionError, "parents", states, zeros(6, dtype=torch.int64))
    refused(TypeError, "parents", states, zeros(2, 3))
    refused(AssertionError, "5 states", zeros(5, 4), parents)
    refused(AssertionError, "dense", zeros(4, 6).t(), parents)
    refused(AssertionError, "slots", states, parents, zeros(6, dtype=torch.int64))
    refused(AssertionError, "65 beams", zeros(65, 4), zeros(1, 65, dtype=torch.int64))
    refused(RuntimeError, "no gradient", zeros(6, 4, requires_grad=True), parents)


def test_entry_points_reject_bad_arguments_without_touching_the_gpu():
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    a = (ctypes.addressof(buf) + 15) & ~15          # a 16-byte aligned, non-null host address (never dereferenced)
    strides = lambda *s: (ctypes.c_int64 * len(s))(*s)  # noqa: E731

    def fwd(B=1, T=8, H=4, HK=2, DK=32, DV=32, dt=BF16, hd=F32, st=None, h0=a, g=a, v=a, n=None, ws=None, size=0):
        return lib.gla_decay_fwd(None, B, T, H, HK, DK, DV, dt, hd, st, h0, g, v, a, a, n, a, a, None, ws, size)

    assert fwd(h0=None) == -1 and fwd(v=None) == -1 and fwd(g=None) == -1
    for bad in ({"B": 0}, {"T": -1}, {"H": 0}, {"HK": 3}, {"HK": 0}, {"DK": 40}, {"DK": 272}, {"DV": 8}, {"DV": 512}, {"T": 1 << 31}, {"H": 1 << 20, "HK": 1 << 20}):
        assert fwd(**bad) == -2, bad
    assert fwd(dt=7) == -3 and fwd(hd=7) == -3
    assert fwd(h0=a + 8) == -6 and fwd(v=a + 2) == -6 and fwd(g=a + 2) == -6 and fwd(n=a + 1) == -6
    dense = (32, 4, 1, 1024, 128, 32, 512, 64, 32, 512, 64, 32)
    assert fwd(st=strides(*dense[:4], 129, *dense[5:])) == -6                    # rows that do not begin on 16 bytes
    assert fwd(st=strides(*dense[:4], 1 << 23, *dense[5:])) == -2                # and rows too far apart
    need = lib.gla_decay_fwd_workspace_bytes(1, 8192, 4, 2, 32, 32, BF16, 0)
    assert need > 0 and fwd(T=8192) == -5 and fwd(T=8192, ws=a, size=need - 1) == -5 and fwd(T=8192, ws=a + 8, size=need) == -6
    assert lib.gla_decay_fwd_workspace_bytes(1, 8192, 4, 3, 32, 32, BF16, 0) == 0

    def bwd(T=8, HK=4, DK=32, dt=BF16, states=a, do=a, dv=a, ws=None, size=0):
        return lib.gla_decay_bwd(None, 1, T, 4, HK, DK, 32, dt, F32, 0, None, a, a, a, a, None, states, a, do, a, a, dv, a, a, ws, size)

    assert bwd(states=None) == -1 and bwd(do=None) == -1 and bwd(dv=None) == -1 and bwd(DK=33) == -2 and bwd(dt=2) == -3 and bwd(do=a + 8) == -6
    # a key head's gradient comes in parts, one of each head that shares it
    need = lib.gla_decay_bwd_workspace_bytes(1, 8, 4, 2, 32, 32, BF16, 0, 0)
    assert need >= 2 * 2 * 8 * 2 * 32 * 4 and bwd(HK=2) == -5 and bwd(HK=2, ws=a, size=need - 1) == -5
    assert lib.gla_decay_bwd_workspace_bytes(1, 8, 4, 4, 32, 32, BF16, 0, 0) == 0 < lib.gla_decay_bwd_workspace_bytes(1, 8, 4, 4, 32, 32, BF16, 1, 0)

    def step(pool=6, B=6, HK=4, DK=32, beams=0, st=BF16, states=a, slots=None, parents=None, wide=1, v=a, strides=None):
        return lib.gla_decay_step(None, pool, B, 4, HK, DK, 32, beams, BF16, st, wide, strides, a, v, a, a, slots, parents, states, a)

    assert step(states=None) == -1 and step(beams=2) == -1
    for bad in ({"pool": 0}, {"B": 0}, {"pool": 5}, {"HK": 3}, {"DK": 8}, {"beams": 4, "parents": a}, {"beams": -1}, {"B": 65, "pool": 65, "beams": 65, "parents": a}):
        assert step(**bad) == -2, bad
    assert step(st=9) == -3 and step(states=a + 8) == -6 and step(slots=a + 4) == -6 and step(v=a + 2) == -6
    assert step(strides=strides(4, 1, 129, 32, 128, 32, 128, 32)) == -6

    def select(G=2, W=3, V=100, num=3, dt=F32, row=100, logits=a, finished=None, eos=0, ws=a, size=1 << 20):
        return lib.gla_beam_select(None, G, W, V, num, dt, row, logits, a, finished, eos, a, a, a, ws, size)

    assert select(logits=None) == -1 and select(dt=4) == -3 and select(logits=a + 2) == -6
    for bad in ({"G": 0}, {"W": 0}, {"W": 65}, {"V": 0}, {"num": 0}, {"num": 65}, {"V": 1, "num": 4, "row": 1}, {"row": 99}, {"finished": a, "eos": 100},
                {"finished": a, "eos": -1}, {"G": 65536}, {"V": 1 << 30, "row": 1 << 30}):
        assert select(**bad) == -2, bad
    need = lib.gla_beam_select_workspace_bytes(2, 3, 100, 3)
    assert need > 0 and select(ws=None) == -5 and select(size=need - 1) == -5 and lib.gla_beam_select_workspace_bytes(2, 65, 100, 3) == 0

    def order(pool=6, G=2, W=3, size=16, parents=a, slots=None, states=a, wide=1):
        return lib.gla_reorder_states(None, pool, G, W, size, wide, parents, slots, states)

    assert order(parents=None) == -1 and order(states=None) == -1 and order(parents=a + 4) == -6 and order(slots=a + 2, wide=0) == -6
    for bad in ({"pool": 5}, {"G": 0}, {"W": 65}, {"size": 0}):
        assert order(**bad) == -2, bad


def test_sizes_of_what_the_forward_leaves():
    lib = _lib.load()
    # the state before every chunk of 64 tokens (float data 32), in 32 bits
    assert lib.gla_decay_states_bytes(2, 130, 4, 2, 32, 48, BF16) == 2 * 4 * 3 * 32 * 48 * 4
    assert lib.gla_decay_states_bytes(2, 130, 4, 2, 32, 48, F32) == 2 * 4 * 5 * 32 * 48 * 4
    assert lib.gla_decay_states_bytes(2, 0, 4, 2, 32, 48, BF16) == 0
    # sequences enough to fill the GPU run whole, few long ones as segments
    assert lib.gla_decay_fwd_workspace_bytes(64, 4096, 8, 8, 64, 64, BF16, 0) == 0
    assert lib.gla_decay_fwd_workspace_bytes(1, 32768, 8, 8, 128, 128, BF16, 0) >= 8 * 32 * 128 * 128 * 4
