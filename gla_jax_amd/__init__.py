"""gla_jax_amd — Gated Linear Attention (zhixuan-lin/gla-jax's hot path) for AMD MI355X / gfx950.

Public surface, mirroring the reference's modules:
    gla.py : chunk_gla, recurrent_gla, recurrent_gla_naive
    ops.py : cumsum_recursive, rnn_recursive
and, for models whose heads have one decay each and for serving them:
    decay.py : chunk_decay (prompts, training), decay_step (single tokens)
    beam.py : beam_select, reorder_states (beam search)
All of them run hand-written HIP kernels from libgla_hip.so; there is no CPU or eager fallback.
"""
from . import _lib
from .beam import beam_select, reorder_states
from .decay import chunk_decay, decay_step
from .gla import chunk_gla, recurrent_gla, recurrent_gla_naive
from .ops import cumsum_recursive, rnn_recursive

__all__ = ["chunk_gla", "recurrent_gla", "recurrent_gla_naive", "cumsum_recursive", "rnn_recursive",
           "chunk_decay", "decay_step", "beam_select", "reorder_states"]
