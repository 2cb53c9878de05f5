"""Calls of the scoring, loss and 4-bit lm_head entries that are refused:
argument checks of the C ABI (no pointer is followed, so no GPU is needed) and
of the Python functions (on CPU tensors, refused at the latest for not being on
a GPU)."""
import ctypes as C

import pytest
import torch

from qwen600_engine_b200 import _lib, losses, w4
from qwen600_engine_b200._lib import QS_BF16, QS_ERR_INVALID, QS_ERR_UNSUPPORTED, QS_F16, QS_F32, SamplerError

L = _lib.lib
P = 0x10000  # a 16-byte aligned address that no refused call follows
FAR = 0x7F0000000000


def logprobs(logits=P, dtype=QS_BF16, rows=4, vocab=1000, ld=1000, tokens=P, T=1.0, lp=P, stats=P, ws=P, size=1 << 30):
    return L.qs_token_logprobs(logits, dtype, rows, vocab, ld, tokens, T, lp, stats, ws, size, None)


def backward(logits=P, dtype=QS_BF16, rows=4, vocab=1000, ld=1000, tokens=P, stats=P, g=P, T=1.0, grad=FAR, gld=1000):
    return L.qs_token_logprobs_backward(logits, dtype, rows, vocab, ld, tokens, stats, g, T, grad, gld, None)


def policy(logits=P, dtype=QS_BF16, rows=4, vocab=1000, ld=1000, tokens=P, old=P, ref=None, adv=P, w=None, lo=0.2,
           hi=0.2, kl=0.0, T=1.0, loss=P, lp=P, grad=FAR, gld=1000, ws=P, size=1 << 20, params=True):
    p = _lib.PolicyParams(lo, hi, kl, T)
    return L.qs_policy_loss(logits, dtype, rows, vocab, ld, tokens, old, ref, adv, w, C.byref(p) if params else None,
                            loss, lp, grad, gld, ws, size, None)


def preference(logits=P, dtype=QS_BF16, rows=4, vocab=1000, ld=1000, tokens=P, off=P, pairs=2, ref=P, w=None, beta=0.1,
               eps=0.0, loss=P, seq=P, grad=FAR, gld=1000, ws=P, size=1 << 20, params=True):
    p = _lib.PreferenceParams(beta, eps)
    return L.qs_preference_loss(logits, dtype, rows, vocab, ld, tokens, off, pairs, ref, w, C.byref(p) if params else None,
                                loss, seq, grad, gld, ws, size, None)


NAN, INF = float("nan"), float("inf")
ROWS = [dict(dtype=QS_F16), dict(dtype=7), dict(rows=-1), dict(logits=None), dict(tokens=None), dict(ld=999),
        dict(logits=P + 1), dict(dtype=QS_F32, logits=P + 2)]
LIMITS = [dict(rows=(1 << 27) + 1), dict(vocab=0), dict(vocab=-5), dict(vocab=1 << 20, ld=1 << 20)]
TEMPS = [dict(T=0.0), dict(T=1e-7), dict(T=-1.0), dict(T=NAN), dict(T=INF), dict(T=1e7)]
GRADS = [dict(grad=P + 2), dict(grad=P + 2000), dict(grad=P, gld=1008), dict(grad=P - 16), dict(gld=999), dict(grad=FAR + 1)]


@pytest.mark.parametrize("call,bad", [(logprobs, b) for b in ROWS + TEMPS + [
                             dict(lp=None), dict(stats=None), dict(rows=100000, ws=None), dict(rows=100000, ws=P + 4),
                             dict(rows=100000, size=1000)]]
                         + [(backward, b) for b in ROWS + TEMPS + GRADS + [dict(stats=None), dict(g=None), dict(grad=None)]]
                         + [(policy, b) for b in ROWS + TEMPS + GRADS + [
                             dict(old=None), dict(adv=None), dict(loss=None), dict(params=False), dict(kl=0.1, ref=None),
                             dict(kl=-0.1), dict(kl=NAN), dict(kl=INF), dict(lo=-0.1), dict(lo=1.5), dict(lo=NAN),
                             dict(hi=-0.1), dict(hi=INF), dict(hi=NAN), dict(ws=None), dict(ws=P + 8), dict(size=8)]]
                         + [(preference, b) for b in ROWS + GRADS + [
                             dict(off=None), dict(ref=None), dict(loss=None), dict(params=False), dict(pairs=-1),
                             dict(beta=0.0), dict(beta=-1.0), dict(beta=NAN), dict(beta=INF), dict(eps=-0.1),
                             dict(eps=0.5), dict(eps=NAN), dict(ws=None), dict(ws=P + 4), dict(size=8)]])
def test_c_abi_refuses(call, bad):
    assert call(**bad) == QS_ERR_INVALID, bad
    assert L.qs_last_error()


@pytest.mark.parametrize("call", [logprobs, backward, policy, preference])
@pytest.mark.parametrize("bad", LIMITS)
def test_c_abi_limits(call, bad):
    assert call(**bad) == QS_ERR_UNSUPPORTED
    assert L.qs_last_error()


def test_empty_batches_need_no_buffers():
    assert L.qs_token_logprobs(None, QS_BF16, 0, 1000, 1000, None, 1.0, None, None, None, 0, None) == _lib.QS_OK
    assert L.qs_token_logprobs_backward(None, QS_F32, 0, 1000, 1000, None, None, None, 1.0, None, 0, None) == _lib.QS_OK


def weight(vocab=1000, hidden=1024, group=128, dtype=QS_BF16, codes=P, scales=P, zeros=None):
    return _lib.W4Desc(codes, scales, zeros, vocab, hidden, group, dtype)


BAD_WEIGHTS = [(dict(vocab=0), QS_ERR_UNSUPPORTED), (dict(vocab=1 << 20), QS_ERR_UNSUPPORTED),
               (dict(hidden=0), QS_ERR_UNSUPPORTED), (dict(hidden=100), QS_ERR_UNSUPPORTED),
               (dict(hidden=16384), QS_ERR_UNSUPPORTED), (dict(group=16), QS_ERR_UNSUPPORTED),
               (dict(group=0), QS_ERR_UNSUPPORTED), (dict(group=-32), QS_ERR_UNSUPPORTED),
               (dict(hidden=192, group=128), QS_ERR_UNSUPPORTED), (dict(dtype=QS_F32), QS_ERR_INVALID),
               (dict(codes=None), QS_ERR_INVALID), (dict(scales=None), QS_ERR_INVALID),
               (dict(codes=P + 8), QS_ERR_INVALID), (dict(scales=P + 2), QS_ERR_INVALID), (dict(zeros=P + 1), QS_ERR_INVALID)]


@pytest.mark.parametrize("bad,code", BAD_WEIGHTS)
def test_w4_weight_refused(bad, code):
    w = weight(**bad)
    assert L.qs_lm_head_w4(P, None, C.byref(w), 1, P, P, P, 1 << 20, None) == code
    assert L.qs_last_error()


def test_sizes_outside_the_limits_are_0_bytes():
    for vocab, hidden, group in ((0, 1024, 128), (-1, 1024, 128), (1000, 0, 64), (1 << 30, 1024, 64), (1000, 1 << 20, 32)):
        assert L.qs_w4_codes_bytes(vocab, hidden) == 0
        assert L.qs_w4_scales_bytes(vocab, hidden, group) == 0 and L.qs_w4_zeros_bytes(vocab, hidden, group) == 0
    for group in (0, -32, 48, 1 << 30):
        assert L.qs_w4_scales_bytes(1000, 1024, group) == 0 and L.qs_w4_zeros_bytes(1000, 1024, group) == 0
    assert L.qs_lm_head_w4_workspace(-1, 1024) == 0 and L.qs_lm_head_w4_workspace(4, 1 << 20) == 0
    assert L.qs_policy_loss_workspace(-5) > 0 and L.qs_preference_loss_workspace(QS_F32, -5, 1000) == 0
    assert L.qs_token_logprobs_workspace(9, 10, 1000) == 0 and L.qs_token_logprobs_workspace(QS_F32, 10, -1) == 0


def test_w4_calls_refused():
    w = weight()
    r = C.byref(w)
    assert L.qs_lm_head_w4(P, None, None, 1, P, P, P, 1 << 20, None) == QS_ERR_INVALID
    assert L.qs_lm_head_w4(None, None, r, 1, P, P, P, 1 << 20, None) == QS_ERR_INVALID
    assert L.qs_lm_head_w4(P + 4, None, r, 1, P, P, P, 1 << 20, None) == QS_ERR_INVALID
    assert L.qs_lm_head_w4(P, None, r, -1, P, P, P, 1 << 20, None) == QS_ERR_INVALID
    assert L.qs_lm_head_w4(P, None, r, 1, None, P, P, 1 << 20, None) == QS_ERR_INVALID
    assert L.qs_lm_head_w4(P, None, r, 1, P, P + 2, P, 1 << 20, None) == QS_ERR_INVALID
    assert L.qs_lm_head_w4(P, P + 2, r, 1, P, P, P, 1 << 20, None) == QS_ERR_INVALID
    assert L.qs_lm_head_w4(P, None, r, 1, P, P, None, 1 << 20, None) == QS_ERR_INVALID
    assert L.qs_lm_head_w4(P, None, r, 1, P, P, P + 8, 1 << 20, None) == QS_ERR_INVALID
    assert L.qs_lm_head_w4(P, None, r, 1, P, P, P, 64, None) == QS_ERR_INVALID
    assert L.qs_lm_head_w4_sample(None, P, None, r, 1, P, None, 0) == QS_ERR_INVALID
    assert L.qs_w4_pack(P, P, None, 1000, 1024, 128, QS_F32, P, P, None, None) == QS_ERR_INVALID
    assert L.qs_w4_pack(P, P, P, 1000, 1024, 128, QS_BF16, P, P, None, None) == QS_ERR_INVALID
    assert L.qs_w4_pack(P, P, None, 1000, 1024, 128, QS_BF16, P + 8, P, None, None) == QS_ERR_INVALID
    assert L.qs_w4_pack(P, P + 1, None, 1000, 1024, 128, QS_BF16, P, P, None, None) == QS_ERR_INVALID
    assert L.qs_w4_pack(P, P, None, 1000, 1024, 48, QS_BF16, P, P, None, None) == QS_ERR_UNSUPPORTED
    assert L.qs_w4_quantize(None, 1000, 1024, 128, P, P, P, None) == QS_ERR_INVALID
    assert L.qs_w4_quantize(P, 1000, 1024, 128, P, P, None, None) == QS_ERR_INVALID
    assert L.qs_w4_quantize(P, 1000, 100, 128, P, P, P, None) == QS_ERR_UNSUPPORTED


X = torch.zeros((4, 10))
TOK = torch.zeros(4, dtype=torch.int32)
F = torch.zeros(4)


@pytest.mark.parametrize("call,match", [
    (lambda: losses.token_logprobs(X[0], TOK), "must be \\[rows, vocab\\]"),
    (lambda: losses.token_logprobs(X.half(), TOK), "dtype"),
    (lambda: losses.token_logprobs(X.t(), TOK), "strides"),
    (lambda: losses.token_logprobs(X[:1].expand(4, 10), TOK), "strides"),
    (lambda: losses.token_logprobs(X, TOK.long()), "tokens must be"),
    (lambda: losses.token_logprobs(X, TOK[:3]), "tokens must be"),
    (lambda: losses.token_logprobs(X, torch.zeros(8, dtype=torch.int32)[::2]), "tokens must be"),
    (lambda: losses.token_logprobs(X, TOK), "on a GPU"),
    (lambda: losses.token_logprobs_backward(X, TOK, torch.zeros((4, 3)), F), "stats must be"),
    (lambda: losses.token_logprobs_backward(X, TOK, torch.zeros((4, 2)), F[:2]), "grad_logprobs must be"),
    (lambda: losses.token_logprobs_backward(X, TOK, torch.zeros((4, 2)), F, out=X.bfloat16()), "buffer must be"),
    (lambda: losses.token_logprobs_backward(X, TOK, torch.zeros((4, 2)), F, out=torch.zeros((10, 4)).t()), "strides"),
    (lambda: losses.policy_loss(X, TOK, F.double(), F), "old_logprobs must be"),
    (lambda: losses.policy_loss(X, TOK, F, F[:1]), "advantages must be"),
    (lambda: losses.policy_loss(X, TOK, F, F, weights=F.bool()), "weights must be"),
    (lambda: losses.policy_loss(X, TOK, F, F, ref_logprobs=F[:1]), "ref_logprobs must be"),
    (lambda: losses.policy_loss(X, TOK, F, F, grad=False, out=X), "without a gradient"),
    (lambda: losses.policy_loss(X, TOK, F, F), "on a GPU"),
    (lambda: losses.preference_loss(X, TOK, torch.zeros(4, dtype=torch.int32), F), "seq_offsets must be"),
    (lambda: losses.preference_loss(X, TOK, torch.zeros(5), F), "seq_offsets must be"),
    (lambda: losses.preference_loss(X, TOK, torch.zeros(5, dtype=torch.int32), F[:2]), "ref_logprobs must be"),
    (lambda: losses.preference_loss(X, TOK, torch.zeros(5, dtype=torch.int32), F, weights=F), "weights must be"),
    (lambda: losses.preference_loss(X, TOK, torch.zeros(5, dtype=torch.int32), F), "on a GPU"),
    (lambda: w4.W4Weight.pack(torch.zeros((4, 64)), F), "codes must be"),
    (lambda: w4.W4Weight.pack(torch.zeros((4, 64), dtype=torch.uint8), torch.zeros((4, 1))), "scales must be"),
    (lambda: w4.W4Weight.pack(torch.zeros((4, 64), dtype=torch.uint8), torch.zeros((4, 3), dtype=torch.half)), "scales must be"),
    (lambda: w4.W4Weight.pack(torch.zeros((4, 64), dtype=torch.uint8), torch.zeros((4, 1), dtype=torch.half),
                              torch.zeros((4, 2), dtype=torch.uint8)), "zeros must be"),
    (lambda: w4.W4Weight.pack(torch.zeros((64, 4), dtype=torch.uint8).t(), torch.zeros((4, 1), dtype=torch.half)), "contiguous"),
    (lambda: w4.W4Weight.pack(torch.zeros((4, 64), dtype=torch.uint8), torch.zeros((4, 1), dtype=torch.half)), "on a GPU"),
    (lambda: w4.quantize_w4(torch.zeros((4, 128))), "bf16"),
    (lambda: w4.quantize_w4(torch.zeros((4, 128), dtype=torch.bfloat16), 48), "group"),
])
def test_python_refuses(call, match):
    with pytest.raises(SamplerError, match=match):
        call()


def test_package_names():
    import qwen600_engine_b200 as q
    assert q.policy_loss is losses.policy_loss and q.preference_loss is losses.preference_loss
    assert q.token_logprobs is losses.token_logprobs and q.token_logprobs_backward is losses.token_logprobs_backward
    assert q.W4Weight is w4.W4Weight and q.lm_head_w4 is w4.lm_head_w4


def w4_parts(vocab=100, hidden=256, group=64):
    return (torch.zeros(L.qs_w4_codes_bytes(vocab, hidden), dtype=torch.uint8),
            torch.zeros(L.qs_w4_scales_bytes(vocab, hidden, group), dtype=torch.uint8),
            torch.zeros(L.qs_w4_zeros_bytes(vocab, hidden, group), dtype=torch.uint8))


def test_w4_weight_of_packed_buffers():
    codes, scales, zeros = w4_parts()
    w = w4.W4Weight(codes, scales, zeros, 100, 256, 64, QS_F16)
    assert (w.vocab, w.hidden_dim, w.group) == (100, 256, 64)
    assert w4.W4Weight(codes, scales, None, 100, 256, 64, QS_BF16).zeros is None


@pytest.mark.parametrize("bad", [
    dict(codes=w4_parts()[0][1:]), dict(codes=w4_parts()[0][:-1]), dict(codes=w4_parts()[0].view(torch.int8)),
    dict(codes=torch.zeros(2 * w4_parts()[0].numel(), dtype=torch.uint8)[::2]), dict(scales=w4_parts()[1][:-2]),
    dict(scales=w4_parts()[1].view(torch.float16)), dict(zeros=w4_parts()[2][:-1]), dict(zeros=w4_parts()[1]),
    dict(scales=w4_parts()[1].to("meta")), dict(vocab=101 + 32), dict(vocab=0), dict(vocab=-1), dict(vocab=1 << 20),
    dict(hidden_dim=512), dict(hidden_dim=0), dict(hidden_dim=200), dict(group=32), dict(group=48), dict(group=0),
    dict(scale_dtype=QS_F32), dict(scale_dtype=9)])
def test_w4_weight_of_other_buffers_refused(bad):
    """Sizes that do not fit the shape would be read out of range."""
    codes, scales, zeros = w4_parts()
    kw = dict(codes=codes, scales=scales, zeros=zeros, vocab=100, hidden_dim=256, group=64, scale_dtype=QS_F16) | bad
    with pytest.raises(SamplerError):
        w4.W4Weight(**kw)
