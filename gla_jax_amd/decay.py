"""Linear attention with one decay a head on MI355X: `chunk_decay` for whole sequences, `decay_step` for single tokens.

    S_t = exp(a_t) S_{t-1} + k_t v_t^T,   o_t = S_t^T q_t      (a_t: one number for each head and token)

the recurrence of `chunk_gla` with a gate that all key features of a head share, or that is one constant a head.  A pair's
weight is then a number, so scores need no rescaled operands, and heads may share their keys and queries.  The reference
has no counterpart; names, argument order and layouts follow `chunk_gla`:

    hidden_init [H,DK,DV];  log_decay [T,H] or [H];  value [T,H,DV];  key, query [T,HK,DK], HK divides H
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .gla import (_DT, _apply, _as, _merge_mapped, _native, _no_double_backward, _plain_call, _ptr, _split_mapped, _stream,
                  _transforms_active, _twin)


def _rows(t, dtype):
    """`t` [B,T,heads,features] as the kernels take it: features side by side, rows on 16 bytes, batch, token and head strides
    as they are (a projection's output cut into its parts stays where it lies)."""
    t = t.to(dtype)
    piece = 16 // t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
            s % piece == 0 and s < 1 << 23 or n == 1 for s, n in zip(t.stride()[1:-1], t.shape[1:])) and t.stride(0) % piece == 0:
        return t
    return _dense(t)


def _dense(t):
    """`t` without gaps, on 16 bytes."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _strides(*rows):
    """The host array of strides that the C ABI takes: all axes but the features' (of an axis of one, any will do)."""
    s = [x if m > 1 else 0 for t, n in rows for x, m in zip(t.stride()[:n], t.shape)]
    return (ctypes.c_int64 * len(s))(*s)


def _decay_forward(h0, a, v, k, q, lengths, residual):
    B, T, H, DV = v.shape
    HK, DK = k.shape[2:]
    # (chunk_decay has checked its own arguments; a call that a tracer has recorded may be given others)
    if tuple(h0.shape) != (B, H, DK, DV) or tuple(k.shape[:2]) != (B, T) or q.shape != k.shape or k.dtype != v.dtype or q.dtype != v.dtype:
        raise ValueError("chunk_decay: arrays that do not fit each other")
    if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype != torch.int32 or not lengths.is_contiguous()):
        raise ValueError("chunk_decay: lengths of another type or number than the sequences")
    lib, dt = _lib.load(), _DT[v.dtype]
    h0, v, k, q = _dense(h0), _rows(v, v.dtype), _rows(k, k.dtype), _rows(q, q.dtype)
    at = a.expand(B, T, H)
    with torch.cuda.device(v.device):
        hT, out = torch.empty_like(h0), torch.empty(v.shape, dtype=v.dtype, device=v.device)
        n = lib.gla_decay_fwd_workspace_bytes(B, T, H, HK, DK, DV, dt, int(lengths is not None))
        ws = torch.empty(n, dtype=torch.uint8, device=v.device) if n else None
        # cut into B rows of bytes it maps over the batch axis as arrays do
        kept = lib.gla_decay_states_bytes(B, T, H, HK, DK, DV, dt) if residual else 0
        states = torch.empty(B, kept // B, dtype=torch.uint8, device=v.device) if residual else None
        rc = lib.gla_decay_fwd(_stream(), B, T, H, HK, DK, DV, dt, _DT[h0.dtype], _strides((at, 3), (v, 3), (k, 3), (q, 3)), _ptr(h0),
                               _ptr(at), _ptr(v), _ptr(k), _ptr(q), _ptr(lengths), _ptr(hT), _ptr(out), _ptr(states) if kept else None,
                               _ptr(ws), n)
    _lib.check("gla_decay_fwd", rc)
    return hT, out, states


class _ChunkDecay(torch.autograd.Function):
    """Arguments are the canonical arrays of `chunk_decay`: h0 [B,H,DK,DV], a [B,T,H] or [H] float32, v, k, q [B,T,...],
    lengths [B] int32 or None."""

    @staticmethod
    def forward(h0, a, v, k, q, lengths):
        return _decay_forward(h0, a, v, k, q, lengths, True)

    @staticmethod
    def setup_context(ctx, inputs, output):
        h0, a, v, k, q, lengths = inputs
        ctx.save_for_backward(output[2], a, v, k, q, lengths)
        ctx.hidden = (tuple(h0.shape), h0.dtype)
        ctx.mark_non_differentiable(output[2])
        ctx.set_materialize_grads(False)

    @staticmethod
    def backward(ctx, dhT, dout, dstates=None):
        states, a, v, k, q, lengths = ctx.saved_tensors
        shape, dtype = ctx.hidden
        dhT = torch.zeros(shape, dtype=dtype, device=v.device) if dhT is None else dhT
        dout = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if dout is None else dout
        return _apply(_ChunkDecayBwd, states, a, v, k, q, lengths, dhT, dout) + (None,)

    @staticmethod
    def vmap(info, in_dims, h0, a, v, k, q, lengths):
        outs = _ChunkDecay.apply(*_merge_mapped(info, in_dims[:5], (h0, a, v, k, q)), _merge_lengths(info, in_dims[5], lengths))
        return _split_mapped(info, outs), (0, 0, 0)


def _merge_lengths(info, dim, lengths):
    return None if lengths is None else _merge_mapped(info, (dim,), (lengths,))[0]


class _ChunkDecayBwd(torch.autograd.Function):
    """The backward rule as a function of its own (see gla._ChunkGLABwd)."""

    @staticmethod
    def forward(states, a, v, k, q, lengths, dhT, dout):
        B, T, H, DV = v.shape
        HK, DK = k.shape[2:]
        lib, dt = _lib.load(), _DT[v.dtype]
        states, v, k, q = states.contiguous(), _rows(v, v.dtype), _rows(k, k.dtype), _rows(q, q.dtype)
        dhT, dout = _dense(dhT.to(dhT.dtype if dhT.dtype in _DT else torch.float32)), _dense(dout.to(v.dtype))
        constant = a.ndim == 1
        at = a.expand(B, T, H)
        with torch.cuda.device(v.device):
            new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
            dh0, da, dv, dk, dq = new(dhT), new(a), new(v), new(k), new(q)
            n = lib.gla_decay_bwd_workspace_bytes(B, T, H, HK, DK, DV, dt, int(constant), int(lengths is not None))
            ws = torch.empty(n, dtype=torch.uint8, device=v.device) if n else None
            rc = lib.gla_decay_bwd(_stream(), B, T, H, HK, DK, DV, dt, _DT[dhT.dtype], int(constant),
                                   _strides((at, 3), (v, 3), (k, 3), (q, 3)), _ptr(at), _ptr(v), _ptr(k), _ptr(q), _ptr(lengths),
                                   _ptr(states), _ptr(dhT), _ptr(dout), _ptr(dh0), _ptr(da), _ptr(dv), _ptr(dk), _ptr(dq), _ptr(ws), n)
        _lib.check("gla_decay_bwd", rc)
        return dh0, da, dv, dk, dq

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *grads):
        _no_double_backward("chunk_decay")

    @staticmethod
    def vmap(info, in_dims, states, a, v, k, q, lengths, dhT, dout):
        if in_dims[0] is not None:      # the forward was mapped as well: its states are those of the merged batch
            merged = _merge_mapped(info, in_dims[:5] + in_dims[6:], (states, a, v, k, q, dhT, dout))
            outs = _ChunkDecayBwd.apply(*merged[:5], _merge_lengths(info, in_dims[5], lengths), *merged[5:])
            return _split_mapped(info, outs), (0,) * 5
        if any(d is not None for d in in_dims[1:6]):
            raise RuntimeError("chunk_decay: the rows are mapped and the states of their forward are not")
        outs = [_ChunkDecayBwd.apply(states, a, v, k, q, lengths,
                                     *(x if d is None else x.select(d, i) for x, d in zip((dhT, dout), in_dims[6:])))
                for i in range(info.batch_size)]
        return tuple(torch.stack(o) for o in zip(*outs)), (0,) * 5


def _check(named, device):
    for name, t in named:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise ValueError(f"{name} must live on the GPU; gla_jax_amd has no CPU path")
        if t.device != device:
            raise ValueError(f"{name} lies on another device ({t.device}) than the states ({device})")


def _check_heads(value, key, query, HK, H):
    if HK < 1 or H % HK:
        raise AssertionError(f"{HK} key heads do not divide {H} heads")
    if value.dtype not in _DT or key.dtype != value.dtype or query.dtype != value.dtype:
        raise TypeError("value, key, query must share one dtype (float32 or bfloat16)")
    if not (1 <= key.shape[-1] <= 256 and 1 <= value.shape[-1] <= 256):
        raise AssertionError("head dimensions from 1 to 256 are built")


def chunk_decay(hidden_init, log_decay, value, key, query, lengths=None):
    """Linear attention with one decay a head over whole sequences, chunk by chunk on the matrix cores.

    Shapes as in the module's head, with any leading batch axes in front of all arrays ([H] for log_decay is one constant for
    each head everywhere); T is any length, 0 among them.  `value`, `key`, `query` share one dtype (float32 or bfloat16) and may be
    views with strides, such as the parts of one projection.  log_decay is taken in float32; -inf forgets everything before its token.  `lengths`
    (integers, shaped as the leading axes) ends sequences early: what lies behind is not read (it may be NaN), `out` is zero there
    and hidden_final is the state at the end.

    Returns (hidden_final [..,H,DK,DV] in hidden_init.dtype, out [..,T,H,DV] in value.dtype).  Differentiable in all five arrays;
    heads that share a key head add up to its gradient, tokens to that of a constant decay."""
    done = _native("decay", (hidden_init, log_decay, value, key, query), lengths)
    if done is not None:
        return tuple(done)
    arrays = (("hidden_init", hidden_init), ("log_decay", log_decay), ("value", value), ("key", key), ("query", query))
    _check(arrays, hidden_init.device if isinstance(hidden_init, torch.Tensor) else None)
    if value.ndim < 3:
        raise AssertionError("value must be [..., T, H, DV]")
    lead = tuple(value.shape[:-3])
    T, H, DV = value.shape[-3:]
    if key.ndim != value.ndim or tuple(key.shape[:-2]) != lead + (T,) or query.shape != key.shape:
        raise AssertionError(f"key {tuple(key.shape)} and query {tuple(query.shape)} must be {lead + (T, 'HK', 'DK')}")
    HK, DK = key.shape[-2:]
    _check_heads(value, key, query, HK, H)
    if tuple(hidden_init.shape) != lead + (H, DK, DV):
        raise AssertionError(f"hidden_init shape {tuple(hidden_init.shape)} != {lead + (H, DK, DV)}")
    if tuple(log_decay.shape) not in (lead + (T, H), (H,)):
        raise AssertionError(f"log_decay shape {tuple(log_decay.shape)} is neither {lead + (T, H)} nor {(H,)}")
    if not hidden_init.dtype.is_floating_point or not log_decay.dtype.is_floating_point:
        raise TypeError("hidden_init and log_decay must be floating-point tensors")
    B = 1
    for s in lead:
        B *= s
    if lengths is not None:
        _check((("lengths", lengths),), hidden_init.device)
        if tuple(lengths.shape) != lead or lengths.dtype not in (torch.int32, torch.int64):
            raise AssertionError(f"lengths must be integers of shape {lead}")
        lengths = lengths.reshape(B).clamp(0, T).to(torch.int32) if lengths.dtype == torch.int64 else lengths.reshape(B).contiguous()
    if B == 0 or H == 0:
        return hidden_init.clone(), value.clone()
    h0 = _as(hidden_init, (B, H, DK, DV), hidden_init.dtype if hidden_init.dtype in _DT else torch.float32)
    a = log_decay.to(torch.float32)
    if a.ndim > 1 or _transforms_active():
        a = a.expand(lead + (T, H)).reshape(B, T, H)
    v, k, q = value.reshape(B, T, H, DV), key.reshape(B, T, HK, DK), query.reshape(B, T, HK, DK)
    pk, pv = -DK % 16, -DV % 16
    if pk or pv:
        # The kernels take 16 features at a time.  A zero feature adds nothing to a score or to the rest of the state.
        F = torch.nn.functional
        h0, v, k, q = F.pad(h0, (0, pv, 0, pk)), F.pad(v, (0, pv)), F.pad(k, (0, pk)), F.pad(q, (0, pk))
    if _plain_call():
        hT, out = _native("decay", (_dense(h0), a, *(_rows(t, t.dtype) for t in (v, k, q))), lengths)
    else:
        hT, out = _apply(_ChunkDecay, h0, a, v, k, q, lengths)[:2]
    if pk or pv:
        hT, out = hT[..., :DK, :DV], out[..., :DV]
    return _as(hT, lead + (H, DK, DV), hidden_init.dtype), _as(out, lead + (T, H, DV), out.dtype)


def _indices(name, t, shape, device):
    _check(((name, t),), device)
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64")
    if tuple(t.shape) != shape:
        raise AssertionError(f"{name} shape {tuple(t.shape)} != {shape}")
    return t.contiguous()


def _same_width(*indices):
    """Indices of one call share a width."""
    wide = any(t is not None and t.dtype == torch.int64 for t in indices)
    return int(wide), [t if t is None or not wide else t.to(torch.int64) for t in indices]


def _no_gradient(name):
    raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad()")


def _refuse_gradients(name, *arrays):
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in arrays):
        _no_gradient(name)


def _refuse_tangents(name, *arrays):
    """There is no forward-mode rule, and a result without its tangent would be a wrong one.  (An autograd function refuses them as well, but
    after its forward, which updates states in place.)"""
    if any(isinstance(t, torch.Tensor) and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in arrays):
        raise RuntimeError(f"{name} has no forward-mode rule: an array carries a tangent")


def _step(entry, states, gates, value, key, query, slots, parents):
    """One launch of `entry` with all of its checks; `gates`: pairs of a name and an array [B,H] or [H]."""
    _check((("states", states), *gates, ("value", value), ("key", key), ("query", query)),
           states.device if isinstance(states, torch.Tensor) else None)
    if value.ndim != 3 or key.ndim != 3 or query.shape != key.shape or key.shape[0] != value.shape[0]:
        raise AssertionError("value must be [B, H, DV], key and query [B, HK, DK]")
    B, H, DV = value.shape
    HK, DK = key.shape[1:]
    _check_heads(value, key, query, HK, H)
    if states.ndim != 4 or tuple(states.shape[1:]) != (H, DK, DV):
        raise AssertionError(f"states shape {tuple(states.shape)} != {('N', H, DK, DV)}")
    if states.dtype not in _DT:
        raise TypeError("states must be float32 or bfloat16")
    if not states.is_contiguous() or states.data_ptr() % 16 or DK % 16 or DV % 16:
        raise AssertionError("states are updated where they lie: dense, on 16 bytes, DK and DV multiples of 16")
    for name, t in gates:
        if tuple(t.shape) not in ((B, H), (H,)):
            raise AssertionError(f"{name} shape {tuple(t.shape)} is neither {(B, H)} nor {(H,)}")
    if slots is None and states.shape[0] < B:
        raise AssertionError(f"{states.shape[0]} states for {B} rows")
    if slots is not None:
        slots = _indices("slots", slots, (B,), states.device)
    W = 0
    if parents is not None:
        if parents.ndim != 2 or parents.shape[0] * parents.shape[1] != B:
            raise AssertionError(f"parents shape {tuple(parents.shape)} does not hold {B} rows")
        W = parents.shape[1]
        if W > _lib.GLA_MOST_BEAMS:
            raise AssertionError(f"{W} beams: at most {_lib.GLA_MOST_BEAMS} are built")
        parents = _indices("parents", parents, tuple(parents.shape), states.device)
    if B == 0 or H == 0 or states.shape[0] == 0:
        return torch.zeros_like(value)
    wide, (slots, parents) = _same_width(slots, parents)
    v, k, q = (_rows(t, value.dtype) for t in (value, key, query))
    gates = [t.to(torch.float32).expand(B, H) for _, t in gates]
    with torch.cuda.device(states.device):
        out = torch.empty(B, H, DV, dtype=v.dtype, device=v.device)
        rc = getattr(_lib.load(), entry)(_stream(), states.shape[0], B, H, HK, DK, DV, W, _DT[v.dtype], _DT[states.dtype], wide,
                                         _strides(*((t, 2) for t in (*gates, v, k, q))), *(_ptr(t) for t in gates), _ptr(v), _ptr(k),
                                         _ptr(q), _ptr(slots), _ptr(parents), _ptr(states), _ptr(out))
    _lib.check(entry, rc)
    torch.autograd.graph.increment_version(states)
    return out


class _DecayStep(torch.autograd.Function):
    """decay_step for arrays that are not as the native host side takes them, and under a tracer, which records a Function as a call of
    it.  So all checks are here, where a recorded call makes them again.  There is no gradient."""

    @staticmethod
    def forward(states, log_decay, value, key, query, slots, parents):
        return _step("gla_decay_step", states, (("log_decay", log_decay),), value, key, query, slots, parents)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *grads):
        _no_gradient("decay_step")


def decay_step(states, log_decay, value, key, query, slots=None, parents=None):
    """One token for each row of a batch: the recurrent form for decoding.  `states` [N,H,DK,DV] (float32 or bfloat16, dense) is
    updated in place and is a pool: row b's state is states[slots[b]] (slots None: states[b]); a slot outside 0..N-1 (-1) marks a row without a
    sequence, whose output is zero.  No two rows may name the same slot.

    log_decay [B,H] or [H];  value [B,H,DV];  key, query [B,HK,DK], HK divides H.  Returns out [B,H,DV] in value.dtype.

    `parents` [G,W] with G * W = B takes the rows as G beam searches of W beams: row w of a search continues from the state that row
    parents[g,w] had before the call (`beam_select` returns them), which saves `reorder_states` its pass.  A parent outside
    0..W-1 counts as w.  W is at most 64.

    States are updated in place: nothing here is differentiable, and arrays that require a gradient are refused.  The update counts as a
    new version of `states`: a backward that has saved them raises instead of using them."""
    done = _native("decay_step", (states, log_decay, value, key, query), slots, parents)
    if done is not None:
        return done
    _refuse_gradients("decay_step", states, log_decay, value, key, query)
    _refuse_tangents("decay_step", states, log_decay, value, key, query)
    return _apply(_DecayStep, states, log_decay, value, key, query, slots, parents)


for _cls in (_ChunkDecay, _ChunkDecayBwd, _DecayStep):
    _cls._twin = _twin(_cls)
