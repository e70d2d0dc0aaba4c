"""What a model's logits say of given tokens: log probabilities, entropies and alternatives, and the gradient of the first two.  The reference has
no counterpart."""
from __future__ import annotations

import torch

from . import _lib
from .decay import _check
from .gla import _DT, _apply, _native, _no_double_backward, _ptr, _stream, _twin


def _logit_rows(logits):
    """`logits` as rows [N,V] one distance apart, features side by side: a view where it can be one."""
    V = logits.shape[-1]
    rows = logits.reshape(-1, V)
    if V > 1 and rows.stride(1) != 1 or rows.shape[0] > 1 and rows.stride(0) < V:
        rows = rows.contiguous()
    return rows, rows.stride(0) if rows.shape[0] > 1 else V


class _TokenLogprobs(torch.autograd.Function):
    """token_logprobs for arrays that are not as the native host side takes them, and under a transform or a tracer.  All checks are here, where a
    recorded call makes them again."""

    @staticmethod
    def forward(logits, tokens, top):
        _check((("logits", logits), ("tokens", tokens)), logits.device if isinstance(logits, torch.Tensor) else None)
        if logits.ndim < 1 or logits.shape[-1] < 1:
            raise AssertionError("logits must be [..., V], V at least 1")
        if logits.dtype not in _DT:
            raise TypeError("logits must be float32 or bfloat16")
        if tokens.dtype not in (torch.int32, torch.int64):
            raise TypeError("tokens must be int32 or int64")
        lead, V = tuple(logits.shape[:-1]), logits.shape[-1]
        if tuple(tokens.shape) != lead:
            raise AssertionError(f"tokens shape {tuple(tokens.shape)} != {lead}")
        if not 0 <= top <= min(_lib.GLA_MOST_ALTERNATIVES, V):
            raise AssertionError(f"{top} alternatives of {V} tokens: 0 to {_lib.GLA_MOST_ALTERNATIVES} are built")
        rows, step = _logit_rows(logits)
        tokens, N = tokens.contiguous(), rows.shape[0]
        with torch.cuda.device(logits.device):
            new = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device=logits.device)  # noqa: E731
            given, entropy, stats = new(lead), new(lead), new(lead + (2,))
            near, index = new(lead + (top,)), new(lead + (top,), dtype=torch.int64)
            rc = _lib.load().gla_token_logprobs(_stream(), N, V, top, _DT[logits.dtype], step, int(tokens.dtype == torch.int64), _ptr(rows),
                                                _ptr(tokens), _ptr(given), _ptr(entropy), _ptr(stats), _ptr(near) if top else None,
                                                _ptr(index) if top else None)
        _lib.check("gla_token_logprobs", rc)
        return given, entropy, near, index, stats

    @staticmethod
    def setup_context(ctx, inputs, output):
        logits, tokens, _ = inputs
        ctx.save_for_backward(logits, tokens, output[4], output[1])
        ctx.mark_non_differentiable(*output[2:])
        ctx.set_materialize_grads(False)

    @staticmethod
    def backward(ctx, dgiven, dentropy, *others):
        logits, tokens, stats, entropy = ctx.saved_tensors
        _lib.binding().refuse_capture_for_eager_leaves("token_logprobs", logits)
        zero = lambda d: torch.zeros_like(entropy) if d is None else d  # noqa: E731
        return _apply(_TokenLogprobsBwd, logits, tokens, stats, entropy, zero(dgiven), zero(dentropy))[0], None, None

    @staticmethod
    def vmap(info, in_dims, logits, tokens, top):
        front = [t.movedim(d, 0) if d is not None else t.unsqueeze(0).expand(info.batch_size, *t.shape) for t, d in zip((logits, tokens), in_dims)]
        return _TokenLogprobs.apply(*front, top), (0,) * 5


class _TokenLogprobsBwd(torch.autograd.Function):
    """The backward rule as a function of its own (see gla._ChunkGLABwd)."""

    @staticmethod
    def forward(logits, tokens, stats, entropy, dgiven, dentropy):
        rows, step = _logit_rows(logits)
        tokens, stats, entropy = tokens.contiguous(), stats.contiguous(), entropy.contiguous()
        dgiven, dentropy = (d.to(torch.float32).contiguous() for d in (dgiven, dentropy))
        V, piece = logits.shape[-1], 16 // logits.element_size()
        # rows that begin at the same place within 16 bytes as those of the logits
        ahead, row = rows.data_ptr() % 16 // logits.element_size(), V + (step - V) % piece
        with torch.cuda.device(logits.device):
            d = torch.empty(ahead + rows.shape[0] * row, dtype=logits.dtype, device=logits.device)
            to = d.as_strided(rows.shape, (row, 1), ahead)
            rc = _lib.load().gla_token_logprobs_bwd(_stream(), rows.shape[0], V, _DT[logits.dtype], step, row, int(tokens.dtype == torch.int64),
                                                    _ptr(rows), _ptr(tokens), _ptr(stats), _ptr(entropy), _ptr(dgiven), _ptr(dentropy), _ptr(to))
        _lib.check("gla_token_logprobs_bwd", rc)
        return (to.view(logits.shape),)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *grads):
        _no_double_backward("token_logprobs")

    @staticmethod
    def vmap(info, in_dims, *arrays):
        front = [t.movedim(d, 0) if d is not None else t.unsqueeze(0).expand(info.batch_size, *t.shape) for t, d in zip(arrays, in_dims)]
        return _TokenLogprobsBwd.apply(*front), (0,)


def token_logprobs(logits, tokens, top=0):
    """What logits say of given tokens: logits [..,V] (float32 or bfloat16), tokens [..] (int32 or int64).

    Rows that are one distance apart, whatever axes lie in front, are read where they lie, at any distance and alignment.  Others are copied first, in the
    forward and again in the backward pass: features that lie apart, and rows such as logits[:, :-1] of several sequences, which skip one at
    each sequence's end.  (All positions at once, with -100 for the token behind the last, take no copy.)

    Returns (logprobs [..], entropy [..]), float32: the log softmax at each token, and the entropy of each distribution in nats; with `top`
    (at most 64) also (top_logprobs [..,top], top_tokens [..,top] int64): the largest log probabilities, of equal ones the lower token first.  A token
    outside 0..V-1 (-100, say) marks a position that does not count: its logits are not read, logprobs and entropy are 0 there and its
    alternatives -inf and -1.  A logit of -inf has probability 0; a row with a NaN, or a +inf, or nothing above -inf, has NaN results.  In the order of the
    alternatives NaN counts as -inf, and +inf comes first.

    Differentiable in logits through logprobs and entropy: -logprobs.sum() is the cross entropy.  Positions that do not count get a gradient of 0.
    A backward pass is captured into a graph only while no graph of the same leaves from the default stream is alive (RuntimeError)."""
    top = int(top)
    done = _native("token_logprobs", (logits, tokens), top)
    if done is None:
        done = _apply(_TokenLogprobs, logits, tokens, top)[:4]
    return tuple(done[:4] if top else done[:2])


for _cls in (_TokenLogprobs, _TokenLogprobsBwd):
    _cls._twin = _twin(_cls)
