"""The lm_head with its weight held in 4 bits, over the C ABI.

``W4Weight`` holds a weight in the order the kernel reads it, made once when a
program loads its weights: from codes, scales and zero points
(``W4Weight.pack``) or from a bf16 weight (``W4Weight.quantize``).
``lm_head_w4`` is ``sampler.lm_head`` with such a weight, and
``Sampler.lm_head_sample`` takes one in place of the bf16 weight.  The formulas
stand in include/qwen600_sampler.h; the reference has no counterpart (its
weights are bf16).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import QS_BF16, QS_ERR_INVALID, QS_F16, SamplerError, check
from .losses import _on, _torch  # the binding, with what to do where it does not load

_SCALES = {torch.bfloat16: QS_BF16, torch.float16: QS_F16}


def _invalid(msg: str) -> SamplerError:
    return SamplerError(QS_ERR_INVALID, msg)


def _on_stream(device, stream, inputs, run):
    """run(stream handle) on the device and stream of one call.  Buffers made
    by run belong to the stream that uses them, and inputs used on another
    stream than the current one are kept until it is done with them."""
    if device.type != "cuda":
        raise _invalid("the tensors must be on a GPU")
    with torch.cuda.device(device):
        if stream is None:
            return run(torch.cuda.current_stream().cuda_stream)
        if stream.device != device:
            raise _invalid(f"stream of {stream.device} for tensors on {device}")
        if stream != torch.cuda.current_stream():
            for t in inputs:
                if t is not None:
                    t.record_stream(stream)
        with torch.cuda.stream(stream):
            return run(stream.cuda_stream)


class W4Weight:
    """A packed weight [vocab, hidden_dim] on one GPU: 4-bit codes, a scale and
    a zero point for each ``group`` columns of a row.  The constructor takes
    buffers that ``pack`` laid out (another weight's ``codes``, ``scales`` and
    ``zeros``)."""

    def __init__(self, codes, scales, zeros, vocab: int, hidden_dim: int, group: int, scale_dtype: int):
        L = _lib.lib
        if hidden_dim % 64 or group not in (32, 64, 128) or hidden_dim % group or scale_dtype not in _SCALES.values():
            raise _invalid(f"hidden_dim {hidden_dim}, group {group} or scale dtype {scale_dtype} outside the library's limits")
        for name, t, size in (("codes", codes, L.qs_w4_codes_bytes(vocab, hidden_dim)),
                              ("scales", scales, L.qs_w4_scales_bytes(vocab, hidden_dim, group)),
                              ("zeros", zeros, L.qs_w4_zeros_bytes(vocab, hidden_dim, group))):
            if t is None and name == "zeros":
                continue
            if not size or t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() != size or t.device != codes.device:
                raise _invalid(f"{name} must be {size} contiguous bytes on {codes.device} for [{vocab}, {hidden_dim}] in groups "
                               f"of {group}, got {t.dtype} {tuple(t.shape)} on {t.device}")
        self.codes, self.scales, self.zeros = codes, scales, zeros
        self.vocab, self.hidden_dim, self.group = vocab, hidden_dim, group
        self.device = codes.device
        self._w4_desc = _lib.W4Desc(codes.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(),
                                    vocab, hidden_dim, group, scale_dtype)
        self._parts = (codes, scales, zeros, vocab, hidden_dim, group, scale_dtype)

    @classmethod
    def pack(cls, codes, scales, zeros=None, *, stream=None) -> "W4Weight":
        """codes uint8 [vocab, hidden_dim / 2], the even column in the low half
        of a byte; scales bf16 or fp16 [vocab, hidden_dim / group], which gives
        the group (32, 64 or 128); zeros uint8 of the scales' shape, in 0..15,
        or None (all 8).  The weight is scale * (code - zero)."""
        if codes.dim() != 2 or codes.dtype != torch.uint8:
            raise _invalid(f"codes must be uint8 [vocab, hidden_dim / 2], got {codes.dtype} {tuple(codes.shape)}")
        vocab, hidden = int(codes.shape[0]), 2 * int(codes.shape[1])
        if scales.dim() != 2 or scales.shape[0] != vocab or scales.shape[1] < 1 or hidden % scales.shape[1] \
                or scales.dtype not in _SCALES:
            raise _invalid(f"scales must be bf16 or fp16 [{vocab}, {hidden} / group], got {scales.dtype} "
                           f"{tuple(scales.shape)}")
        group = hidden // int(scales.shape[1])
        if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
            raise _invalid(f"zeros must be uint8 {tuple(scales.shape)}, got {zeros.dtype} {tuple(zeros.shape)}")
        for t in (codes, scales, zeros):
            if t is not None and (not t.is_contiguous() or t.device != codes.device):
                raise _invalid("codes, scales and zeros must be contiguous and on one device")
        dev, code = codes.device, _SCALES[scales.dtype]
        L = _lib.lib

        def run(st):
            pc = torch.empty(L.qs_w4_codes_bytes(vocab, hidden), dtype=torch.uint8, device=dev)
            ps = torch.empty(L.qs_w4_scales_bytes(vocab, hidden, group), dtype=torch.uint8, device=dev)
            pz = None if zeros is None else torch.empty(L.qs_w4_zeros_bytes(vocab, hidden, group), dtype=torch.uint8,
                                                        device=dev)
            check(L.qs_w4_pack(codes.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(), vocab,
                               hidden, group, code, pc.data_ptr(), ps.data_ptr(), None if pz is None else pz.data_ptr(),
                               st))
            return pc, ps, pz

        if not L.qs_w4_codes_bytes(vocab, hidden):
            raise _invalid(f"vocab {vocab} or hidden_dim {hidden} outside the library's limits")
        if group not in (32, 64, 128):
            raise _invalid(f"scales make a group of {group} columns (want 32, 64 or 128)")
        pc, ps, pz = _on_stream(dev, stream, (codes, scales, zeros), run)
        return cls(pc, ps, pz, vocab, hidden, group, code)

    @classmethod
    def quantize(cls, weight, group: int = 128, *, stream=None) -> "W4Weight":
        """Rounds a bf16 weight [vocab, hidden_dim] to 4 bits: per group a bf16
        scale of a fifteenth of the range that holds the group and zero, and
        the nearest codes."""
        return cls.pack(*quantize_w4(weight, group, stream=stream), stream=stream)


def quantize_w4(weight, group: int = 128, *, stream=None):
    """(codes, scales, zeros) of a bf16 weight in the plain form that
    ``W4Weight.pack`` takes."""
    if weight.dim() != 2 or weight.dtype != torch.bfloat16 or not weight.is_contiguous():
        raise _invalid("weight must be a contiguous bf16 tensor [vocab, hidden_dim]")
    vocab, hidden = int(weight.shape[0]), int(weight.shape[1])
    if group not in (32, 64, 128) or hidden % group:
        raise _invalid(f"group {group} must be 32, 64 or 128 and divide hidden_dim {hidden}")
    if not _lib.lib.qs_w4_codes_bytes(vocab, hidden):
        raise _invalid(f"vocab {vocab} or hidden_dim {hidden} outside the library's limits")
    dev = weight.device

    def run(st):
        codes = torch.empty((vocab, hidden // 2), dtype=torch.uint8, device=dev)
        scales = torch.empty((vocab, hidden // group), dtype=torch.bfloat16, device=dev)
        zeros = torch.empty((vocab, hidden // group), dtype=torch.uint8, device=dev)
        check(_lib.lib.qs_w4_quantize(weight.data_ptr(), vocab, hidden, group, codes.data_ptr(), scales.data_ptr(),
                                      zeros.data_ptr(), st))
        return codes, scales, zeros

    return _on_stream(dev, stream, (weight,), run)


def _check_rows(hidden, weight: W4Weight, norm_weight):
    h = hidden if hidden.dim() == 2 else hidden.view(1, -1)
    for t in (h, norm_weight):
        if t is not None and (t.dtype != torch.bfloat16 or not t.is_contiguous() or t.device != weight.device):
            raise _invalid(f"hidden and norm_weight must be contiguous bf16 tensors on {weight.device}")
    if h.shape[1] != weight.hidden_dim:
        raise _invalid(f"hidden has {h.shape[1]} columns, the weight {weight.hidden_dim}")
    if norm_weight is not None and norm_weight.numel() != weight.hidden_dim:
        raise _invalid(f"norm_weight has {norm_weight.numel()} values, the weight {weight.hidden_dim} columns")
    return h


def lm_head_w4(hidden, weight: W4Weight, norm_weight=None, *, stream=None):
    """Final RMSNorm + lm_head with a 4-bit weight, for bf16 rows
    [B, hidden_dim]; returns (normed [B, hidden_dim], logits [B, vocab]) bf16,
    as ``sampler.lm_head`` does."""
    h = _check_rows(hidden, weight, norm_weight)
    return _on(stream, _torch.lm_head_w4, h, norm_weight, *weight._parts)


__all__ = ["W4Weight", "quantize_w4", "lm_head_w4"]
