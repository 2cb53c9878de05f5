"""Scoring and training on sampled tokens, over the C ABI (its torch binding,
csrc/qs_torch.cpp, checks the tensors and makes the buffers).

``token_logprobs`` gives the log-probability of one token per row of logits
(the old and reference log-probabilities of the losses, or what a server
returns beside a sampled token), ``token_logprobs_backward`` takes a gradient of
those back to the logits.  ``policy_loss`` (clipped, with a KL term) and
``preference_loss`` (paired log ratios) return their loss and the gradient of
the logits in one call.  The formulas stand in include/qwen600_sampler.h.

Nothing these functions return has an autograd history, also where the logits
require a gradient: ``loss.backward()`` raises, and in a sum with other losses
this one's part would be missing without an error.  ``logits.backward(result.grad)``
hands the gradient on; beside other losses over the same graph, use
``torch.autograd.backward([logits, other], [result.grad, None])``.

Tensors are on one GPU: logits [rows, vocab] fp32 or bf16 whose columns are
contiguous (any row stride of at least vocab), tokens int32 [rows].  A token
outside [0, vocab) marks a row that scores nothing (a prompt's, padding): its
log-probability is 0 and its gradient zero.  Row i scores ``tokens[i]``: shift
the tokens, not the logits, and mark each sequence's last row.  Calls run on the
current stream of the tensors' device, or on ``stream``; errors raise
``SamplerError``.  The reference has no counterpart (it only samples).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib  # noqa: F401  (loads the library)
try:
    from . import _torch
except ImportError as e:
    raise ImportError("qwen600_engine_b200/_torch.so is missing or was built for another torch; build it with "
                      "`python -m qwen600_engine_b200.build` (or __graft_entry__.build())") from e
from ._lib import QS_ERR_INVALID, SamplerError


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor  # fp32 [rows]
    stats: torch.Tensor     # fp32 [rows, 2]: row maximum, sum of exp((x - maximum) / T) - 1


class PolicyLoss(NamedTuple):
    loss: torch.Tensor            # fp32 scalar
    logprobs: torch.Tensor        # fp32 [rows]
    grad: Optional[torch.Tensor]  # [rows, vocab] in the logits' type


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor            # fp32 scalar
    seq_logprobs: torch.Tensor    # fp32 [2 * pairs]
    grad: Optional[torch.Tensor]  # [rows, vocab] in the logits' type


def _on(stream, call, *args):
    """call(*args) on the current stream of the tensors' device, or on `stream`:
    buffers made by the call belong to it, and tensors used on it from another
    stream are kept until it is done with them."""
    if stream is None:
        return call(*args)
    device = args[0].device
    if device.type == "cuda":
        if stream.device != device:
            raise SamplerError(QS_ERR_INVALID, f"stream of {stream.device} for tensors on {device}")
        if stream != torch.cuda.current_stream(device):
            for t in args:
                if isinstance(t, torch.Tensor) and t.is_cuda:
                    t.record_stream(stream)
    with torch.cuda.stream(stream):
        return call(*args)


def token_logprobs(logits, tokens, *, temperature: float = 1.0, stream=None) -> TokenLogprobs:
    """log softmax(logits / temperature) of each row's token, and the row
    statistics that ``token_logprobs_backward`` takes."""
    return tuple.__new__(TokenLogprobs, _on(stream, _torch.token_logprobs, logits, tokens, temperature))


def token_logprobs_backward(logits, tokens, stats, grad_logprobs, *, temperature: float = 1.0, out=None, stream=None):
    """The gradient of the logits from that of the log-probabilities; ``stats``
    are the forward call's, on the same logits and temperature.  ``out`` may be
    ``logits`` (the gradient then replaces them)."""
    return _on(stream, _torch.token_logprobs_backward, logits, tokens, stats, grad_logprobs, temperature, out)


def policy_loss(logits, tokens, old_logprobs, advantages, *, ref_logprobs=None, weights=None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0, grad: bool = True, out=None,
                stream=None) -> PolicyLoss:
    """Clipped policy loss with a KL term, summed over the rows with
    ``weights`` (default 1 / rows; 0 leaves a row out), and the gradient of the
    logits (``grad=False``: the loss alone).  ``ref_logprobs`` is needed where
    ``kl_coef`` is above 0.  ``out`` takes the gradient and may be ``logits``."""
    return tuple.__new__(PolicyLoss, _on(stream, _torch.policy_loss, logits, tokens, old_logprobs, advantages, ref_logprobs,
                                         weights, clip_low, clip_high, kl_coef, temperature, grad, out))


def preference_loss(logits, tokens, seq_offsets, ref_logprobs, *, beta: float = 0.1, label_smoothing: float = 0.0,
                    weights=None, grad: bool = True, out=None, stream=None) -> PreferenceLoss:
    """Paired log-ratio loss over sequences packed along the rows, and the
    gradient of the logits (``grad=False``: the loss alone).  Sequence q holds
    rows ``seq_offsets[q]`` to ``seq_offsets[q + 1]`` (int32 [2 * pairs + 1]);
    sequence p is chosen over sequence pairs + p.  ``ref_logprobs`` fp32
    [2 * pairs]: each sequence's log-probability under the reference model.
    ``weights`` fp32 [pairs] (default 1 / pairs).  ``out`` takes the gradient
    and may be ``logits``.  Offsets that fall anywhere make the loss and every
    sum NaN, without a gradient."""
    return tuple.__new__(PreferenceLoss, _on(stream, _torch.preference_loss, logits, tokens, seq_offsets, ref_logprobs,
                                             weights, beta, label_smoothing, grad, out))


__all__ = ["TokenLogprobs", "PolicyLoss", "PreferenceLoss", "token_logprobs", "token_logprobs_backward", "policy_loss",
           "preference_loss"]
