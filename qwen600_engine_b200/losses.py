"""Scoring and training on sampled tokens, over the C ABI.

``token_logprobs`` gives the log-probability of one token per row of logits
(the old and reference log-probabilities of the losses, or what a server
returns beside a sampled token), ``token_logprobs_backward`` takes a gradient of
those back to the logits.  ``policy_loss`` (clipped, with a KL term) and
``preference_loss`` (paired log ratios) return their loss and the gradient of
the logits in one call; ``logits.backward(result.grad)`` hands it to autograd.
The formulas stand in include/qwen600_sampler.h.

Tensors are on one GPU: logits [rows, vocab] fp32 or bf16 whose columns are
contiguous (any row stride of at least vocab), tokens int32 [rows].  A token
outside [0, vocab) marks a row that scores nothing (a prompt's, padding): its
log-probability is 0 and its gradient zero.  Row i scores ``tokens[i]``: shift
the tokens, not the logits, and mark each sequence's last row.  Buffers are made on the stream that
runs the call; errors raise ``SamplerError``.  The reference has no counterpart
(it only samples).
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import PolicyParams, PreferenceParams, QS_BF16, QS_ERR_INVALID, QS_F32, SamplerError, check

_DTYPES = {torch.float32: QS_F32, torch.bfloat16: QS_BF16}


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


def _invalid(msg: str) -> SamplerError:
    return SamplerError(QS_ERR_INVALID, msg)


_current_device = torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream


def _on_stream(device, stream, inputs, run):
    """run(stream handle) on the device and stream of one call.  Buffers made
    by run belong to the stream that uses them, and inputs used on another
    stream than the current one are kept until it is done with them."""
    if device.type != "cuda":
        raise _invalid("the tensors must be on a GPU")
    if stream is None:
        if _current_device() == device.index:
            return run(_raw_stream(device.index))
        with torch.cuda.device(device):
            return run(_raw_stream(device.index))
    if stream.device != device:
        raise _invalid(f"stream of {stream.device} for tensors on {device}")
    if stream != torch.cuda.current_stream(device):
        for t in inputs:
            if t is not None:
                t.record_stream(stream)
    with torch.cuda.stream(stream):
        return run(stream.cuda_stream)


def _matrix(name: str, t):
    """(rows, vocab, row stride, dtype code) of a [rows, vocab] tensor."""
    if t.dim() != 2:
        raise _invalid(f"{name} must be [rows, vocab], got {tuple(t.shape)}")
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise _invalid(f"{name} dtype {t.dtype} (want float32 or bfloat16)")
    rows, vocab = t.shape
    ld, step = t.stride()
    if vocab > 1 and step != 1 or rows > 1 and ld < vocab:
        raise _invalid(f"{name} columns must be contiguous and its rows apart, got strides {(ld, step)}")
    return rows, vocab, max(ld, vocab), code


def _vector(name: str, t, dtype, n: int, device) -> int:
    if t.dtype is dtype and t.dim() == 1 and t.numel() == n and t.is_contiguous() and t.device == device:
        return t.data_ptr()
    raise _invalid(f"{name} must be a contiguous {dtype} tensor [{n}] on {device}, got {t.dtype} {tuple(t.shape)} "
                   f"on {t.device}")


def _grad_stride(out, logits) -> int:
    """The row stride of the caller's buffer for the gradient, or of a new one."""
    if out is None:
        return logits.shape[1]
    if out.dtype != logits.dtype or out.shape != logits.shape or out.device != logits.device:
        raise _invalid(f"the gradient's buffer must be {logits.dtype} {tuple(logits.shape)} on {logits.device}")
    return _matrix("the gradient's buffer", out)[2]


def _new_grad(logits):
    return torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty(logits.shape)


def token_logprobs(logits, tokens, *, temperature: float = 1.0, stream=None) -> TokenLogprobs:
    """log softmax(logits / temperature) of each row's token, and the row
    statistics that ``token_logprobs_backward`` takes."""
    rows, vocab, ld, code = _matrix("logits", logits)
    dev = logits.device
    tok = _vector("tokens", tokens, torch.int32, rows, dev)

    def run(st):
        lp = torch.empty(rows, dtype=torch.float32, device=dev)
        stats = torch.empty((rows, 2), dtype=torch.float32, device=dev)
        size = _lib.lib.qs_token_logprobs_workspace(code, rows, vocab)
        work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        check(_lib.lib.qs_token_logprobs(logits.data_ptr(), code, rows, vocab, ld, tok, temperature, lp.data_ptr(),
                                         stats.data_ptr(), work.data_ptr() if size else None, size, st))
        return TokenLogprobs(lp, stats)

    return _on_stream(dev, stream, (logits, tokens), run)


def token_logprobs_backward(logits, tokens, stats, grad_logprobs, *, temperature: float = 1.0, out=None, stream=None):
    """The gradient of the logits from that of the log-probabilities; ``stats``
    are the forward call's, on the same logits and temperature.  ``out`` may be
    ``logits`` (the gradient then replaces them)."""
    rows, vocab, ld, code = _matrix("logits", logits)
    dev = logits.device
    tok = _vector("tokens", tokens, torch.int32, rows, dev)
    if stats.dtype != torch.float32 or stats.shape != (rows, 2) or not stats.is_contiguous() or stats.device != dev:
        raise _invalid(f"stats must be a contiguous float32 tensor [{rows}, 2] on {dev}")
    g = _vector("grad_logprobs", grad_logprobs, torch.float32, rows, dev)
    gld = _grad_stride(out, logits)

    def run(st):
        buf = _new_grad(logits) if out is None else out
        check(_lib.lib.qs_token_logprobs_backward(logits.data_ptr(), code, rows, vocab, ld, tok, stats.data_ptr(), g,
                                                  temperature, buf.data_ptr(), gld, st))
        return buf

    return _on_stream(dev, stream, (logits, tokens, stats, grad_logprobs, out), run)


def policy_loss(logits, tokens, old_logprobs, advantages, *, ref_logprobs=None, weights=None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0, grad: bool = True, out=None,
                stream=None) -> PolicyLoss:
    """Clipped policy loss with a KL term, summed over the rows with
    ``weights`` (default 1 / rows; 0 leaves a row out), and the gradient of the
    logits (``grad=False``: the loss alone).  ``ref_logprobs`` is needed where
    ``kl_coef`` is above 0.  ``out`` takes the gradient and may be ``logits``."""
    rows, vocab, ld, code = _matrix("logits", logits)
    dev = logits.device
    tok = _vector("tokens", tokens, torch.int32, rows, dev)
    old = _vector("old_logprobs", old_logprobs, torch.float32, rows, dev)
    adv = _vector("advantages", advantages, torch.float32, rows, dev)
    ref = None if ref_logprobs is None else _vector("ref_logprobs", ref_logprobs, torch.float32, rows, dev)
    w = None if weights is None else _vector("weights", weights, torch.float32, rows, dev)
    if out is not None and not grad:
        raise _invalid("a buffer for the gradient without a gradient")
    gld = _grad_stride(out, logits)
    params = PolicyParams(clip_low, clip_high, kl_coef, temperature)

    def run(st):
        buf = _new_grad(logits) if grad and out is None else out
        size = _lib.lib.qs_policy_loss_workspace(rows)
        work = torch.empty(size // 4 + 1 + rows, dtype=torch.float32, device=dev)  # and the small outputs behind it
        loss, lp = work[size // 4], work[size // 4 + 1:]
        check(_lib.lib.qs_policy_loss(logits.data_ptr(), code, rows, vocab, ld, tok, old, ref, adv, w, C.byref(params),
                                      loss.data_ptr(), lp.data_ptr(), buf.data_ptr() if grad else None, gld,
                                      work.data_ptr(), size, st))
        return PolicyLoss(loss, lp, buf)

    return _on_stream(dev, stream, (logits, tokens, old_logprobs, advantages, ref_logprobs, weights, out), run)


def preference_loss(logits, tokens, seq_offsets, ref_logprobs, *, beta: float = 0.1, label_smoothing: float = 0.0,
                    weights=None, grad: bool = True, out=None, stream=None) -> PreferenceLoss:
    """Paired log-ratio loss over sequences packed along the rows, and the
    gradient of the logits (``grad=False``: the loss alone).  Sequence q holds
    rows ``seq_offsets[q]`` to ``seq_offsets[q + 1]`` (int32 [2 * pairs + 1]);
    sequence p is chosen over sequence pairs + p.  ``ref_logprobs`` fp32
    [2 * pairs]: each sequence's log-probability under the reference model.
    ``weights`` fp32 [pairs] (default 1 / pairs).  ``out`` takes the gradient
    and may be ``logits``."""
    rows, vocab, ld, code = _matrix("logits", logits)
    dev = logits.device
    tok = _vector("tokens", tokens, torch.int32, rows, dev)
    if seq_offsets.dim() != 1 or seq_offsets.shape[0] % 2 != 1:
        raise _invalid(f"seq_offsets must be [2 * pairs + 1], got {tuple(seq_offsets.shape)}")
    pairs = seq_offsets.shape[0] // 2
    off = _vector("seq_offsets", seq_offsets, torch.int32, 2 * pairs + 1, dev)
    ref = _vector("ref_logprobs", ref_logprobs, torch.float32, 2 * pairs, dev)
    w = None if weights is None else _vector("weights", weights, torch.float32, pairs, dev)
    if out is not None and not grad:
        raise _invalid("a buffer for the gradient without a gradient")
    gld = _grad_stride(out, logits)
    params = PreferenceParams(beta, label_smoothing)

    def run(st):
        buf = _new_grad(logits) if grad and out is None else out
        small = torch.empty(1 + 2 * pairs, dtype=torch.float32, device=dev)
        loss, seq = small[0], small[1:]
        size = _lib.lib.qs_preference_loss_workspace(code, rows, vocab)
        work = torch.empty(size, dtype=torch.uint8, device=dev)
        check(_lib.lib.qs_preference_loss(logits.data_ptr(), code, rows, vocab, ld, tok, off, pairs, ref, w,
                                          C.byref(params), loss.data_ptr(), seq.data_ptr(),
                                          buf.data_ptr() if grad else None, gld, work.data_ptr(), size, st))
        return PreferenceLoss(loss, seq, buf)

    return _on_stream(dev, stream, (logits, tokens, seq_offsets, ref_logprobs, weights, out), run)


__all__ = ["TokenLogprobs", "PolicyLoss", "PreferenceLoss", "token_logprobs", "token_logprobs_backward", "policy_loss",
           "preference_loss"]
