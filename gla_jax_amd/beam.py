"""Beam search over models whose memory is a state for each sequence: the selection of the next candidates, and the states behind
them.  The reference has no counterpart."""
from __future__ import annotations

import torch

from . import _lib
from .decay import _check, _indices, _no_gradient, _refuse_gradients, _refuse_tangents, _same_width
from .gla import _DT, _apply, _native, _ptr, _stream, _twin


class _BeamSelect(torch.autograd.Function):
    """beam_select for arrays that are not as the native host side takes them, and under a tracer (see decay._DecayStep)."""

    @staticmethod
    def forward(logits, scores, num, finished, eos):
        _check((("logits", logits), ("scores", scores)), logits.device if isinstance(logits, torch.Tensor) else None)
        if logits.ndim < 2:
            raise AssertionError("logits must be [..., W, V]")
        lead = tuple(logits.shape[:-2])
        W, V = logits.shape[-2:]
        if tuple(scores.shape) != lead + (W,):
            raise AssertionError(f"scores shape {tuple(scores.shape)} != {lead + (W,)}")
        if logits.dtype not in _DT or not scores.dtype.is_floating_point:
            raise TypeError("logits must be float32 or bfloat16, scores floating-point")
        num = int(W if num is None else num)
        if not 1 <= W <= _lib.GLA_MOST_BEAMS or not 1 <= num <= min(_lib.GLA_MOST_CANDIDATES, W * V):
            raise AssertionError(f"{num} candidates of {W} beams over {V} tokens: 1 to {_lib.GLA_MOST_CANDIDATES} of at most "
                                 f"{_lib.GLA_MOST_BEAMS} beams are built")
        eos = int(eos)
        if finished is not None:
            _check((("finished", finished),), logits.device)
            if tuple(finished.shape) != lead + (W,) or finished.dtype != torch.bool:
                raise AssertionError(f"finished must be bool of shape {lead + (W,)}")
            if not 0 <= eos < V:
                raise AssertionError(f"eos {eos} lies outside the vocabulary of {V}")
            finished = finished.contiguous()
        G = 1
        for s in lead:
            G *= s
        scores = scores.to(torch.float32).contiguous()
        rows = logits.reshape(G * W, V) if not logits.ndim == 2 else logits
        if rows.stride(1) != 1 or (G * W > 1 and rows.stride(0) < V):
            rows = rows.contiguous()
        step = rows.stride(0) if G * W > 1 else V
        with torch.cuda.device(logits.device):
            best = torch.empty(lead + (num,), dtype=torch.float32, device=logits.device)
            parents, tokens = (torch.empty(lead + (num,), dtype=torch.int64, device=logits.device) for _ in range(2))
            if G == 0:
                return best, parents, tokens
            lib = _lib.load()
            n = lib.gla_beam_select_workspace_bytes(G, W, V, num)
            if n == 0:
                _lib.check("gla_beam_select", -2)
            ws = torch.empty(n, dtype=torch.uint8, device=logits.device)
            rc = lib.gla_beam_select(_stream(), G, W, V, num, _DT[logits.dtype], step, _ptr(rows), _ptr(scores), _ptr(finished), eos,
                                     _ptr(best), _ptr(parents), _ptr(tokens), _ptr(ws), n)
        _lib.check("gla_beam_select", rc)
        return best, parents, tokens

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *grads):
        _no_gradient("beam_select")


def beam_select(logits, scores, num=None, finished=None, eos=0):
    """The `num` best continuations of every search's beams, best first.

    logits [..,W,V] (float32 or bfloat16, any distance between rows), scores [..,W] (taken in float32): what every beam has so
    far.  A candidate's score is its beam's score plus the log softmax of its logit.  Each beam offers its `num` largest logits, and
    of equal scores the lower (beam, token) comes first.  A logit that is not a number counts as -inf, and so does a score that comes out as none
    (a beam whose logits are all -inf).  `finished` [..,W] bool: such a beam offers `eos` at the score that it has and nothing else.
    num: at most 64, W (the default) or, for searches that put finished beams aside, 2 W.

    Returns (scores [..,num] float32, parents [..,num] int64, tokens [..,num] int64): candidate i is tokens[i] behind beam
    parents[i].  Nothing here is differentiable."""
    done = _native("beam_select", (logits, scores), num, finished, eos)
    if done is not None:
        return tuple(done)
    _refuse_tangents("beam_select", logits, scores)
    logits, scores = (t.detach() if isinstance(t, torch.Tensor) else t for t in (logits, scores))
    return _apply(_BeamSelect, logits, scores, num, finished, eos)


class _ReorderStates(torch.autograd.Function):
    """reorder_states for arrays that are not as the native host side takes them, and under a tracer (see decay._DecayStep)."""

    @staticmethod
    def forward(states, parents, slots):
        _check((("states", states), ("parents", parents)), states.device if isinstance(states, torch.Tensor) else None)
        if parents.ndim != 2:
            raise AssertionError("parents must be [G, W]")
        G, W = parents.shape
        if W > _lib.GLA_MOST_BEAMS:
            raise AssertionError(f"{W} beams: at most {_lib.GLA_MOST_BEAMS} are built")
        if states.ndim < 1 or not states.is_contiguous():
            raise AssertionError("states are reordered where they lie: they must be dense")
        if slots is None and states.shape[0] < G * W:
            raise AssertionError(f"{states.shape[0]} states for {G * W} beams")
        parents = _indices("parents", parents, (G, W), states.device)
        if slots is not None:
            slots = _indices("slots", slots, (G, W), states.device)
        if G * W == 0 or states.numel() == 0:
            return states
        wide, (slots, parents) = _same_width(slots, parents)
        with torch.cuda.device(states.device):
            rc = _lib.load().gla_reorder_states(_stream(), states.shape[0], G, W, states[0].numel() * states.element_size(), wide,
                                                _ptr(parents), _ptr(slots), _ptr(states))
        _lib.check("gla_reorder_states", rc)
        torch.autograd.graph.increment_version(states)
        return states

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *grads):
        _no_gradient("reorder_states")


def reorder_states(states, parents, slots=None):
    """states[g*W + w] <- states[g*W + parents[g,w]] in place, for every search g and its W beams: the states follow the beams that
    `beam_select` keeps.  `states` [N, ..] is dense, of any element type and shape behind its first axis (the states of chunk_decay and decay_step as
    those of recurrent_gla); `slots` [G,W] says where a beam's state lies when they do not lie in order, one outside 0..N-1 marks a
    beam without one.  A parent outside 0..W-1 counts as w.  W is at most 64.  Returns `states`, which count as a new version to autograd, as after
    any operation in place."""
    if _native("reorder", (states, parents), slots):
        return states
    _refuse_gradients("reorder_states", states)
    _refuse_tangents("reorder_states", states)
    _apply(_ReorderStates, states, parents, slots)
    return states


for _cls in (_BeamSelect, _ReorderStates):
    _cls._twin = _twin(_cls)
