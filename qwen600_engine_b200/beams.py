"""Beam search on the GPU, over the C ABI (its torch binding, csrc/qs_torch.cpp,
checks the tensors and makes the buffers).

``beam_select`` takes one step of a search: of all continuations of an entry's
beams, the best by their sums of log-probabilities.  ``beam_reorder`` then moves
what the program keeps of each beam (caches of keys and values, token lists) to
the beams that go on, in place; ``Sampler.reorder_history`` does so for a
sampler's own windows and counts.  include/qwen600_sampler.h gives the meaning
of every field.

Row ``b * beams + i`` of the logits, and of every state, belongs to beam ``i`` of
entry ``b``.  Calls run on the current stream of the tensors' device, or on
``stream``; errors raise ``SamplerError``.  What the functions return has no
autograd history.  The reference has no counterpart (it draws one token of one
sequence).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib  # noqa: F401  (loads the library)
from .losses import _on, _torch


class BeamStep(NamedTuple):
    scores: torch.Tensor    # fp32 [batch, n]
    parents: torch.Tensor   # int32 [batch, n]: the beam that each one continues, -1: none
    tokens: torch.Tensor    # int32 [batch, n], -1: none (not a token to look up)
    finished: torch.Tensor  # bool [batch, n]


def beam_select(logits, scores, *, n: Optional[int] = None, finished=None, eos_token: int = -1, pad_token: Optional[int] = None,
                temperature: float = 1.0, keep_slots: bool = False, stream=None) -> BeamStep:
    """The ``n`` best continuations (default: as many as beams) of each entry's
    beams, the best first.  ``logits`` [batch * beams, vocab] fp32 or bf16,
    ``scores`` fp32 [batch, beams]: each beam's sum of log-probabilities so far
    (-inf: a beam that is not there; a search begins with one beam at 0 and the
    others at -inf).  A beam that ``finished`` (bool [batch, beams]) marks goes on
    with ``pad_token`` (default: ``eos_token``) and its own score.
    ``keep_slots``: each beam's best child stays in its parent's place, so that
    ``beam_reorder`` has only the places of beams that end to write; scores are
    then in no order."""
    if pad_token is None:
        pad_token = eos_token
    return tuple.__new__(BeamStep, _on(stream, _torch.beam_select, logits, scores, n, finished, eos_token, pad_token, temperature,
                                       keep_slots))


def beam_reorder(states, parents, *, dim: int = 0, lengths=None, length_dim: int = -2, stream=None) -> None:
    """Row ``b * beams + i`` of each state becomes what row ``b * beams +
    parents[b, i]`` was, in place.  ``states``: a tensor or a list of tensors of
    any type whose dimension ``dim`` holds the rows (a cache of all layers at
    once, or one tensor per layer); ``parents`` int32 [batch, beams], one outside
    [0, beams) leaves its row as it is.  ``lengths`` int32 [batch]: the positions
    in use of each entry, along ``length_dim``, with those that the step's model
    call has written; what lies behind them is left as it is.  Tensors that need
    a gradient are refused while autograd records: the move has no backward."""
    states = (states,) if isinstance(states, torch.Tensor) else tuple(states)
    _on(stream, _torch.beam_reorder, parents, states, dim, lengths, length_dim)


__all__ = ["BeamStep", "beam_select", "beam_reorder"]
