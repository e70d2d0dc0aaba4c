"""Linear attention by the gated delta rule on MI355X: `chunk_delta` for whole sequences, `delta_step` for single tokens.

    S_t = (1 - b_t k_t k_t^T) exp(a_t) S_{t-1} + b_t k_t v_t^T,   o_t = S_t^T q_t      (a_t, b_t: one number for each head and token)

chunk_decay's recurrence with a state that, before it takes a value in, forgets what it would have answered the key with: a share b_t of it is
replaced, where chunk_decay adds.  With keys of length one and b_t = 1 the state answers k_t with v_t exactly.  The reference has no counterpart;
names, argument order and layouts follow `chunk_decay`:

    hidden_init [H,DK,DV];  log_decay, beta [T,H] or [H];  value [T,H,DV];  key, query [T,HK,DK], HK divides H
"""
from __future__ import annotations

import torch

from . import _lib
from .decay import (_check, _check_heads, _dense, _merge_lengths, _no_gradient, _refuse_gradients, _refuse_tangents, _rows, _step,
                    _strides)
from .gla import _DT, _apply, _as, _merge_mapped, _native, _no_double_backward, _plain_call, _ptr, _split_mapped, _stream, _twin


def _delta_forward(h0, a, b, v, k, q, lengths, residual):
    B, T, H, DV = v.shape
    HK, DK = k.shape[2:]
    # (chunk_delta has checked its own arguments; a call that a tracer has recorded may be given others)
    if (tuple(h0.shape) != (B, H, DK, DV) or tuple(k.shape[:2]) != (B, T) or q.shape != k.shape or k.dtype != v.dtype or q.dtype != v.dtype
            or tuple(a.shape) != (B, T, H) or tuple(b.shape) != (B, T, H)):
        raise ValueError("chunk_delta: arrays that do not fit each other")
    if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype != torch.int32 or not lengths.is_contiguous()):
        raise ValueError("chunk_delta: lengths of another type or number than the sequences")
    lib, dt = _lib.load(), _DT[v.dtype]
    h0, v, k, q = _dense(h0), _rows(v, v.dtype), _rows(k, k.dtype), _rows(q, q.dtype)
    with torch.cuda.device(v.device):
        hT, out = torch.empty_like(h0), torch.empty(v.shape, dtype=v.dtype, device=v.device)
        n = lib.gla_delta_fwd_workspace_bytes(B, T, H, HK, DK, DV, dt)
        ws = torch.empty(n, dtype=torch.uint8, device=v.device) if n else None
        # cut into B rows of bytes it maps over the batch axis as arrays do
        kept = lib.gla_delta_states_bytes(B, T, H, HK, DK, DV, dt) if residual else 0
        states = torch.empty(B, kept // B, dtype=torch.uint8, device=v.device) if residual else None
        rc = lib.gla_delta_fwd(_stream(), B, T, H, HK, DK, DV, dt, _DT[h0.dtype], _strides((a, 3), (b, 3), (v, 3), (k, 3), (q, 3)), _ptr(h0),
                               _ptr(a), _ptr(b), _ptr(v), _ptr(k), _ptr(q), _ptr(lengths), _ptr(hT), _ptr(out),
                               _ptr(states) if kept else None, _ptr(ws), n)
    _lib.check("gla_delta_fwd", rc)
    return hT, out, states


class _ChunkDelta(torch.autograd.Function):
    """Arguments are the canonical arrays of `chunk_delta`: h0 [B,H,DK,DV], a and b [B,T,H] float32, v, k, q [B,T,...], lengths [B] int32 or None."""

    @staticmethod
    def forward(h0, a, b, v, k, q, lengths):
        return _delta_forward(h0, a, b, v, k, q, lengths, True)

    @staticmethod
    def setup_context(ctx, inputs, output):
        h0, a, b, v, k, q, lengths = inputs
        ctx.save_for_backward(output[2], a, b, v, k, q, lengths)
        ctx.hidden = (tuple(h0.shape), h0.dtype)
        ctx.mark_non_differentiable(output[2])
        ctx.set_materialize_grads(False)

    @staticmethod
    def backward(ctx, dhT, dout, dstates=None):
        states, a, b, v, k, q, lengths = ctx.saved_tensors
        _lib.binding().refuse_capture_for_eager_leaves("chunk_delta", v)
        shape, dtype = ctx.hidden
        dhT = torch.zeros(shape, dtype=dtype, device=v.device) if dhT is None else dhT
        dout = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if dout is None else dout
        return _apply(_ChunkDeltaBwd, states, a, b, v, k, q, lengths, dhT, dout) + (None,)

    @staticmethod
    def vmap(info, in_dims, h0, a, b, v, k, q, lengths):
        outs = _ChunkDelta.apply(*_merge_mapped(info, in_dims[:6], (h0, a, b, v, k, q)), _merge_lengths(info, in_dims[6], lengths))
        return _split_mapped(info, outs), (0, 0, 0)


class _ChunkDeltaBwd(torch.autograd.Function):
    """The backward rule as a function of its own (see gla._ChunkGLABwd)."""

    @staticmethod
    def forward(states, a, b, v, k, q, lengths, dhT, dout):
        B, T, H, DV = v.shape
        HK, DK = k.shape[2:]
        lib, dt = _lib.load(), _DT[v.dtype]
        states, v, k, q = states.contiguous(), _rows(v, v.dtype), _rows(k, k.dtype), _rows(q, q.dtype)
        dhT, dout = _dense(dhT.to(dhT.dtype if dhT.dtype in _DT else torch.float32)), _dense(dout.to(v.dtype))
        with torch.cuda.device(v.device):
            new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
            dh0, da, db, dv, dk, dq = new(dhT), new(a), new(b), new(v), new(k), new(q)
            n = lib.gla_delta_bwd_workspace_bytes(B, T, H, HK, DK, DV, dt)
            ws = torch.empty(n, dtype=torch.uint8, device=v.device) if n else None
            rc = lib.gla_delta_bwd(_stream(), B, T, H, HK, DK, DV, dt, _DT[dhT.dtype], _strides((a, 3), (b, 3), (v, 3), (k, 3), (q, 3)),
                                   _ptr(a), _ptr(b), _ptr(v), _ptr(k), _ptr(q), _ptr(lengths), _ptr(states), _ptr(dhT), _ptr(dout),
                                   _ptr(dh0), _ptr(da), _ptr(db), _ptr(dv), _ptr(dk), _ptr(dq), _ptr(ws), n)
        _lib.check("gla_delta_bwd", rc)
        return dh0, da, db, dv, dk, dq

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *grads):
        _no_double_backward("chunk_delta")

    @staticmethod
    def vmap(info, in_dims, states, a, b, v, k, q, lengths, dhT, dout):
        if in_dims[0] is not None:      # the forward was mapped as well: its states are those of the merged batch
            merged = _merge_mapped(info, in_dims[:6] + in_dims[7:], (states, a, b, v, k, q, dhT, dout))
            outs = _ChunkDeltaBwd.apply(*merged[:6], _merge_lengths(info, in_dims[6], lengths), *merged[6:])
            return _split_mapped(info, outs), (0,) * 6
        if any(d is not None for d in in_dims[1:7]):
            raise RuntimeError("chunk_delta: the rows are mapped and the states of their forward are not")
        outs = [_ChunkDeltaBwd.apply(states, a, b, v, k, q, lengths,
                                     *(x if d is None else x.select(d, i) for x, d in zip((dhT, dout), in_dims[7:])))
                for i in range(info.batch_size)]
        return tuple(torch.stack(o) for o in zip(*outs)), (0,) * 6


def chunk_delta(hidden_init, log_decay, beta, value, key, query, lengths=None):
    """Linear attention by the gated delta rule over whole sequences, chunk by chunk on the matrix cores.

    Shapes as in the module's head, with any leading batch axes in front of all arrays ([H] for log_decay or beta is one constant for each head
    everywhere); T is any length, 0 among them; DK is at most 128, DV 256.  `value`, `key`, `query` share one dtype (float32 or bfloat16) and may
    be views with strides, such as the parts of one projection.  log_decay and beta are taken in float32; a log_decay of -inf forgets everything before its
    token.  Keys are taken as they are: with b_t |k_t|^2 above 2 the states grow without bound.  `lengths` (integers, shaped as the leading
    axes) ends sequences early: what lies behind is not read (it may be NaN), `out` is zero there and hidden_final is the state at the end.

    Returns (hidden_final [..,H,DK,DV] in hidden_init.dtype, out [..,T,H,DV] in value.dtype).  Differentiable in all six arrays; heads that
    share a key head add up to its gradient.  A backward pass is captured into a graph only while no graph of the same leaves from the default
    stream is alive (RuntimeError)."""
    done = _native("delta", (hidden_init, log_decay, beta, value, key, query), lengths)
    if done is not None:
        return tuple(done)
    arrays = (("hidden_init", hidden_init), ("log_decay", log_decay), ("beta", beta), ("value", value), ("key", key), ("query", query))
    _check(arrays, hidden_init.device if isinstance(hidden_init, torch.Tensor) else None)
    if value.ndim < 3:
        raise AssertionError("value must be [..., T, H, DV]")
    lead = tuple(value.shape[:-3])
    T, H, DV = value.shape[-3:]
    if key.ndim != value.ndim or tuple(key.shape[:-2]) != lead + (T,) or query.shape != key.shape:
        raise AssertionError(f"key {tuple(key.shape)} and query {tuple(query.shape)} must be {lead + (T, 'HK', 'DK')}")
    HK, DK = key.shape[-2:]
    _check_heads(value, key, query, HK, H)
    if DK > _lib.GLA_MOST_DELTA_KEYS:
        raise AssertionError(f"{DK} key features: at most {_lib.GLA_MOST_DELTA_KEYS} are built")
    if tuple(hidden_init.shape) != lead + (H, DK, DV):
        raise AssertionError(f"hidden_init shape {tuple(hidden_init.shape)} != {lead + (H, DK, DV)}")
    for name, t in arrays[1:3]:
        if tuple(t.shape) not in (lead + (T, H), (H,)):
            raise AssertionError(f"{name} shape {tuple(t.shape)} is neither {lead + (T, H)} nor {(H,)}")
    if not all(t.dtype.is_floating_point for _, t in arrays[:3]):
        raise TypeError("hidden_init, log_decay and beta must be floating-point tensors")
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
    a, b = (t.to(torch.float32).expand(lead + (T, H)).reshape(B, T, H) for t in (log_decay, beta))
    v, k, q = value.reshape(B, T, H, DV), key.reshape(B, T, HK, DK), query.reshape(B, T, HK, DK)
    pk, pv = -DK % 16, -DV % 16
    if pk or pv:
        # The kernels take 16 features at a time.  A zero feature adds nothing to a score or to the rest of the state.
        F = torch.nn.functional
        h0, v, k, q = F.pad(h0, (0, pv, 0, pk)), F.pad(v, (0, pv)), F.pad(k, (0, pk)), F.pad(q, (0, pk))
    if _plain_call():
        hT, out = _native("delta", (_dense(h0), a, b, *(_rows(t, t.dtype) for t in (v, k, q))), lengths)
    else:
        hT, out = _apply(_ChunkDelta, h0, a, b, v, k, q, lengths)[:2]
    if pk or pv:
        hT, out = hT[..., :DK, :DV], out[..., :DV]
    return _as(hT, lead + (H, DK, DV), hidden_init.dtype), _as(out, lead + (T, H, DV), out.dtype)


class _DeltaStep(torch.autograd.Function):
    """delta_step for arrays that are not as the native host side takes them, and under a tracer (see decay._DecayStep)."""

    @staticmethod
    def forward(states, log_decay, beta, value, key, query, slots, parents):
        return _step("gla_delta_step", states, (("log_decay", log_decay), ("beta", beta)), value, key, query, slots, parents)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *grads):
        _no_gradient("delta_step")


def delta_step(states, log_decay, beta, value, key, query, slots=None, parents=None):
    """One token for each row of a batch: the recurrent form for decoding.  `states` [N,H,DK,DV] (float32 or bfloat16, dense) is a pool that is
    updated in place, with `slots` and `parents` as in `decay_step`: row b's state is states[slots[b]], and with `parents` [G,W] it continues from
    the state that its parent beam had before the call.

    log_decay, beta [B,H] or [H];  value [B,H,DV];  key, query [B,HK,DK], HK divides H, DK and DV multiples of 16 up to 256
    (chunk_delta pads others; states are updated where they lie).  Returns out [B,H,DV] in value.dtype.

    States are updated in place: nothing here is differentiable, and arrays that require a gradient are refused.  The update counts as a
    new version of `states`."""
    done = _native("delta_step", (states, log_decay, beta, value, key, query), slots, parents)
    if done is not None:
        return done
    _refuse_gradients("delta_step", states, log_decay, beta, value, key, query)
    _refuse_tangents("delta_step", states, log_decay, beta, value, key, query)
    return _apply(_DeltaStep, states, log_decay, beta, value, key, query, slots, parents)


for _cls in (_ChunkDelta, _ChunkDeltaBwd, _DeltaStep):
    _cls._twin = _twin(_cls)
