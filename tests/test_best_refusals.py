"""Calls of the entries for rows' best tokens that are refused: argument checks of
the C ABI (no pointer is followed, so no GPU is needed) and of the Python
functions (on CPU tensors, refused at the latest for not being on a GPU)."""
import ctypes as C

import pytest
import torch

from qwen600_engine_b200 import _lib, beams, losses
from qwen600_engine_b200._lib import QS_BF16, QS_ERR_INVALID, QS_ERR_UNSUPPORTED, QS_F16, QS_F32, QS_OK, SamplerError

L = _lib.lib
P = 0x10000  # a 16-byte aligned address that no refused call follows
FAR = 0x7F0000000000
NAN, INF = float("nan"), float("inf")


def top(logits=P, dtype=QS_BF16, rows=4, vocab=1000, ld=1000, k=5, T=1.0, lp=P, tok=P, ws=P, size=1 << 30):
    return L.qs_top_logprobs(logits, dtype, rows, vocab, ld, k, T, lp, tok, ws, size, None)


def select(logits=P, dtype=QS_BF16, batch=2, width=2, vocab=1000, ld=1000, scores=P, finished=None, n=2, T=1.0, eos=-1, pad=-1, keep=0,
           out=FAR, parents=FAR + 64, tok=FAR + 128, done=FAR + 192, ws=P, size=1 << 30, params=True):
    p = _lib.BeamParams(T, eos, pad, keep)
    return L.qs_beam_select(logits, dtype, batch, width, vocab, ld, scores, finished, n, C.byref(p) if params else None, out, parents,
                            tok, done, ws, size, None)


def distill(logits=P, dtype=QS_BF16, rows=4, vocab=1000, ld=1000, tokens=P, lps=P, k=5, w=None, T=1.0, rest=1, loss=P, each=P, grad=FAR,
            gld=1000, ws=P, size=1 << 20, params=True):
    p = _lib.DistillParams(T, rest)
    return L.qs_distill_loss(logits, dtype, rows, vocab, ld, tokens, lps, k, w, C.byref(p) if params else None, loss, each, grad, gld,
                             ws, size, None)


ROWS = [dict(dtype=QS_F16), dict(dtype=7), dict(logits=None), dict(ld=999), dict(logits=P + 1), dict(dtype=QS_F32, logits=P + 2)]
TEMPS = [dict(T=0.0), dict(T=1e-7), dict(T=-1.0), dict(T=NAN), dict(T=INF), dict(T=1e7)]
GRADS = [dict(grad=P + 2), dict(grad=P + 2000), dict(grad=P, gld=1008), dict(grad=P - 16), dict(gld=999), dict(grad=FAR + 1)]
WORK = [dict(ws=None), dict(ws=P + 4), dict(size=8)]


@pytest.mark.parametrize("call,bad", [(top, b) for b in ROWS + TEMPS + WORK + [dict(rows=-1), dict(lp=None), dict(tok=None)]]
                         + [(select, b) for b in ROWS + TEMPS + WORK + [
                             dict(batch=-1), dict(scores=None), dict(out=None), dict(parents=None), dict(tok=None), dict(params=False),
                             dict(eos=1000), dict(eos=-2), dict(keep=1, n=3), dict(keep=1, n=1),
                             dict(out=P), dict(parents=P + 12), dict(tok=P - 12), dict(done=P + 3), dict(finished=FAR + 128), dict(finished=FAR - 3)]]
                         + [(distill, b) for b in ROWS + TEMPS + GRADS + WORK + [
                             dict(rows=-1), dict(tokens=None), dict(lps=None), dict(loss=None), dict(params=False)]])
def test_c_abi_refuses(call, bad):
    assert call(**bad) == QS_ERR_INVALID, bad
    assert L.qs_last_error()


@pytest.mark.parametrize("call,bad", [(f, b) for f in (top, select, distill) for b in (dict(vocab=0), dict(vocab=-5), dict(vocab=1 << 20, ld=1 << 20))]
                         + [(top, dict(k=0)), (top, dict(k=257)), (top, dict(k=-1)), (top, dict(rows=(1 << 27) + 1)),
                            (select, dict(n=0)), (select, dict(n=257)), (select, dict(width=0)), (select, dict(width=65)),
                            (select, dict(batch=1 << 30)), (distill, dict(k=0)), (distill, dict(k=257)), (distill, dict(rows=(1 << 27) + 1))])
def test_c_abi_limits(call, bad):
    assert call(**bad) == QS_ERR_UNSUPPORTED, bad
    assert L.qs_last_error()


def test_empty_calls_need_no_buffers():
    assert top(rows=0, logits=None, lp=None, tok=None, ws=None, size=0) == QS_OK
    assert select(batch=0, logits=None, scores=None, out=None, parents=None, tok=None, done=None, ws=None, size=0) == QS_OK
    assert L.qs_beam_reorder(None, 0, None, 3, 4, None, None) == QS_OK
    assert L.qs_beam_reorder(None, 5, None, 0, 4, None, None) == QS_OK


def test_sizes_outside_the_limits_are_0_bytes():
    for bad in ((9, 4, 1000, 5), (QS_F32, 0, 1000, 5), (QS_F32, -4, 1000, 5), (QS_F32, 4, 0, 5), (QS_F32, 4, 1 << 20, 5), (QS_F32, 4, 1000, 0),
                (QS_F32, 4, 1000, 257)):
        assert L.qs_top_logprobs_workspace(*bad) == 0
    for bad in ((QS_F32, 2, 65, 1000, 5), (QS_F32, 0, 4, 1000, 5), (QS_F32, 1 << 30, 4, 1000, 5), (QS_F32, 2, -1, 1000, 5)):
        assert L.qs_beam_select_workspace(*bad) == 0
    assert L.qs_top_logprobs_workspace(QS_BF16, 4, 151936, 20) > 0 and L.qs_beam_select_workspace(QS_F32, 2, 4, 151936, 8) > 0
    assert L.qs_distill_loss_workspace(-3, 5) > 0 and L.qs_distill_loss_workspace(4, 0) == 0 and L.qs_distill_loss_workspace(4, 257) == 0


def state(base=FAR, row=1000, outer=(1, 1), outer_stride=(0, 0), positions=1, stride=0, unit=1000):
    s = _lib.States()
    s.d_base, s.row_stride, s.unit, s.positions, s.position_stride = base, row, unit, positions, stride
    s.outer[0], s.outer[1] = outer
    s.outer_stride[0], s.outer_stride[1] = outer_stride
    return s


def reorder(*states, parents=P, batch=2, width=3, count=None):
    a = (_lib.States * max(1, len(states)))(*states)
    return L.qs_beam_reorder(a, len(states) if count is None else count, parents, batch, width, None, None)


LAYERS = dict(row=100, unit=10, positions=10, stride=10, outer=(1, 4), outer_stride=(0, 600))  # 4 layers of 6 rows


@pytest.mark.parametrize("states", [
    [state(base=None)], [state(unit=0)], [state(unit=-1)], [state(positions=0)], [state(outer=(0, 1))], [state(outer=(1, -1))],
    [state(row=999)], [state(row=0)], [state(row=-1000)], [state(unit=10, positions=5, stride=9)], [state(unit=10, positions=5, stride=0)],
    [state(unit=10, positions=5, stride=-10)], [state(unit=10, positions=101, stride=10)],
    [state(unit=10, outer=(2, 2), outer_stride=(10, 10))], [state(unit=10, outer=(2, 3), outer_stride=(25, 10))],
    [state(**(LAYERS | dict(outer_stride=(0, 599))))], [state(**(LAYERS | dict(outer_stride=(0, 500))))],
    [state(**(LAYERS | dict(outer=(2, 4), outer_stride=(2399, 600))))],
    [state(unit=1 << 50, row=1 << 50)], [state(row=1 << 50)],
    [state(), state()], [state(), state(base=FAR + 999)], [state(base=FAR + 5999), state()], [state(unit=500), state(base=FAR + 499, unit=500)],
    [state(unit=500), state(base=FAR + 501, unit=500)], [state(unit=400), state(base=FAR + 500, unit=400, row=1001)],
    [state(**LAYERS), state(**(LAYERS | dict(base=FAR + 600)))], [state(**LAYERS), state(**(LAYERS | dict(base=FAR + 350)))]])
def test_states_refused(states):
    assert reorder(*states) == QS_ERR_INVALID
    assert L.qs_last_error()


def test_reorder_calls_refused():
    assert reorder(state(), parents=None) == QS_ERR_INVALID
    assert L.qs_beam_reorder(None, 1, P, 2, 3, None, None) == QS_ERR_INVALID
    assert reorder(state(), batch=-1) == QS_ERR_INVALID and reorder(state(), count=-1) == QS_ERR_INVALID
    assert reorder(state(), width=0) == QS_ERR_UNSUPPORTED and reorder(state(), width=1025) == QS_ERR_UNSUPPORTED
    assert reorder(state(), batch=1 << 30) == QS_ERR_UNSUPPORTED
    assert reorder(state(unit=1, positions=1 << 30, stride=3, outer=(1, 4), outer_stride=(0, 1 << 33), row=1 << 40)) == QS_ERR_UNSUPPORTED
    assert L.qs_reorder_history(None, P, 2, 3, None) == QS_ERR_INVALID
    for at in (P, P + 20, P - 5999):  # a state that holds the parents, or the lengths
        assert reorder(state(base=at)) == QS_ERR_INVALID
        a = (_lib.States * 1)(state(base=at))
        assert L.qs_beam_reorder(a, 1, FAR, 2, 3, P if at != P + 20 else P + 15, None) == QS_ERR_INVALID


X = torch.zeros((4, 10))
S = torch.zeros((2, 2))
TOK = torch.zeros((4, 3), dtype=torch.int32)
LP = torch.zeros((4, 3))
PAR = torch.zeros((2, 2), dtype=torch.int32)


@pytest.mark.parametrize("call,match", [
    (lambda: losses.top_logprobs(X[0], 2), "must be \\[rows, vocab\\]"),
    (lambda: losses.top_logprobs(X.half(), 2), "dtype"),
    (lambda: losses.top_logprobs(X.t(), 2), "strides"),
    (lambda: losses.top_logprobs(X, 0), "outside \\[1, 256\\]"),
    (lambda: losses.top_logprobs(X, 1 << 40), "outside \\[1, 256\\]"),
    (lambda: losses.top_logprobs(X, 2), "on a GPU"),
    (lambda: losses.distill_loss(X, TOK[0], LP), "must be \\[rows, k\\]"),
    (lambda: losses.distill_loss(X, TOK.long(), LP), "teacher_tokens must be"),
    (lambda: losses.distill_loss(X, TOK[:3], LP), "teacher_tokens must be"),
    (lambda: losses.distill_loss(X, TOK[:, ::2], LP[:, ::2]), "teacher_tokens must be"),
    (lambda: losses.distill_loss(X, TOK, LP[:, :2]), "teacher_logprobs must be"),
    (lambda: losses.distill_loss(X, TOK, LP.bfloat16()), "teacher_logprobs must be"),
    (lambda: losses.distill_loss(X, TOK[:, :0].contiguous(), LP[:, :0].contiguous()), "outside \\[1, 256\\]"),
    (lambda: losses.distill_loss(X, TOK, LP, weights=torch.zeros(3)), "weights must be"),
    (lambda: losses.distill_loss(X, TOK, LP, grad=False, out=X), "without a gradient"),
    (lambda: losses.distill_loss(X, TOK, LP, out=X.bfloat16()), "buffer must be"),
    (lambda: losses.distill_loss(X, TOK, LP), "on a GPU"),
    (lambda: beams.beam_select(X, S[0], n=2), "scores must be"),
    (lambda: beams.beam_select(X, S.double()), "scores must be"),
    (lambda: beams.beam_select(X, torch.zeros((2, 3))), "a row for each"),
    (lambda: beams.beam_select(X, S, n=0), "outside \\[1, 256\\]"),
    (lambda: beams.beam_select(X, S, finished=S), "finished must be"),
    (lambda: beams.beam_select(X, S, finished=S.bool().t()[:1]), "finished must be"),
    (lambda: beams.beam_select(X, S, eos_token=1 << 40), "32-bit"),
    (lambda: beams.beam_select(X, S), "on a GPU"),
    (lambda: beams.beam_reorder(X, PAR[0]), "parents must be"),
    (lambda: beams.beam_reorder(X, PAR.long()), "parents must be"),
    (lambda: beams.beam_reorder(X, PAR.t()), "parents must be"),
    (lambda: beams.beam_reorder(X[:3], PAR), "rows in dimension"),
    (lambda: beams.beam_reorder(X, PAR, dim=1), "rows in dimension"),
    (lambda: beams.beam_reorder(X, PAR, dim=5), "rows in dimension"),
    (lambda: beams.beam_reorder(X, PAR, lengths=PAR[0]), "positions must be"),
    (lambda: beams.beam_reorder(torch.zeros((4, 5, 6)), PAR, lengths=PAR[0].long()), "lengths must be"),
    (lambda: beams.beam_reorder(torch.zeros((4, 5, 6)), PAR, lengths=PAR.view(-1)), "lengths must be"),
    (lambda: beams.beam_reorder(torch.zeros((4, 5, 6)), PAR, lengths=PAR[0].contiguous(), length_dim=4), "positions must be"),
    (lambda: beams.beam_reorder(torch.zeros((9, 4, 8, 7, 6, 5))[::2, :, ::2, ::2, ::2, ::2], PAR, dim=1), "too many levels"),
    (lambda: beams.beam_reorder([X.to_sparse()], PAR), "dense"),
    (lambda: beams.beam_reorder([X, 3], PAR), "must be a tensor"),
    (lambda: beams.beam_reorder(X, PAR), "on a GPU"),
])
def test_python_refuses(call, match):
    with pytest.raises(SamplerError, match=match):
        call()


def test_package_names():
    import qwen600_engine_b200 as q
    assert q.top_logprobs is losses.top_logprobs and q.distill_loss is losses.distill_loss
    assert q.beam_select is beams.beam_select and q.beam_reorder is beams.beam_reorder
