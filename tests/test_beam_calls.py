"""Refusals of the beam calls that need no GPU: layouts whose extent passes 64
bits, tensors that need a gradient, and scores of no shape to count beams by."""
import pytest
import torch

from qwen600_engine_b200 import _lib, beams
from qwen600_engine_b200._lib import QS_ERR_INVALID, QS_ERR_UNSUPPORTED, SamplerError

L = _lib.lib
BASE = 0x7F0000000000


def state(row, outer=(1, 1), outer_stride=(0, 0), positions=1, stride=0, unit=16, base=BASE):
    s = _lib.States()
    s.d_base, s.row_stride, s.unit, s.positions, s.position_stride = base, row, unit, positions, stride
    s.outer[0], s.outer[1] = outer
    s.outer_stride[0], s.outer_stride[1] = outer_stride
    return s


# (count - 1) * stride of one level is 2^64 or near it: as a 64-bit number small or negative
@pytest.mark.parametrize("wide", [
    dict(row=1 << 40, positions=(1 << 29) + 1, stride=1 << 35), dict(row=16, positions=(1 << 30) + 1, stride=1 << 34),
    dict(row=16, outer=(1, (1 << 29) + 1), outer_stride=(0, 1 << 35)), dict(row=16, outer=((1 << 30) + 1, 1), outer_stride=(1 << 34, 0)),
    dict(row=16, positions=1 << 30, stride=1 << 34), dict(row=1 << 44, positions=(1 << 20) + 1, stride=1 << 43)])
def test_states_wider_than_64_bits_refused(wide):
    states = (_lib.States * 1)(state(**wide))
    assert L.qs_beam_reorder(states, 1, 0x10000, 2, 3, None, None) == QS_ERR_INVALID
    assert b"nested blocks" in L.qs_last_error()
    both = (_lib.States * 2)(state(row=1000, unit=1000, base=BASE - (1 << 20)), state(**wide))
    assert L.qs_beam_reorder(both, 2, 0x10000, 2, 3, None, None) == QS_ERR_INVALID
    assert b"state 1" in L.qs_last_error()


PARENTS = torch.zeros((2, 2), dtype=torch.int32)


@pytest.mark.parametrize("make", [lambda w: w, lambda w: w * 2, lambda w: (w * 2).view(4, 5, 2), lambda w: w[:, :4]])
def test_states_that_need_a_gradient_refused(make):
    """A leaf (a parameter given by mistake), a result of one, and views of both."""
    w = torch.ones((4, 10), requires_grad=True)
    for states in (make(w), [torch.zeros((4, 3)), make(w)]):
        with pytest.raises(SamplerError, match="needs a gradient"):
            beams.beam_reorder(states, PARENTS)
    # what autograd does not record goes on to the next check
    for t in (make(w).detach(), make(w.detach())):
        with pytest.raises(SamplerError, match="on a GPU"):
            beams.beam_reorder(t, PARENTS)
    for mode in (torch.no_grad(), torch.inference_mode()):
        with mode, pytest.raises(SamplerError, match="on a GPU"):
            beams.beam_reorder(make(w), PARENTS)


@pytest.mark.parametrize("scores,match", [(torch.zeros(4), "scores must be"), (torch.tensor(0.0), "scores must be"), ([[0.0, 0.0]], "must be a tensor"),
                                          (None, "must be a tensor"), (torch.zeros((4, 1, 1)), "scores must be")])
def test_scores_that_give_no_number_of_beams_refused(scores, match):
    """`n` is as many as beams where it is not given: what the scores are is looked at first."""
    for n in ({}, {"n": 2}):
        with pytest.raises(SamplerError, match=match) as e:
            beams.beam_select(torch.zeros((4, 10)), scores, **n)
        assert e.value.code == QS_ERR_INVALID


def test_beams_above_the_list_refused():
    with pytest.raises(SamplerError, match="300 outside \\[1, 256\\]") as e:
        beams.beam_select(torch.zeros((300, 10)), torch.zeros((1, 300)))
    assert e.value.code == QS_ERR_UNSUPPORTED
    with pytest.raises(SamplerError, match="outside"):
        beams.beam_select(torch.zeros((0, 10)), torch.zeros((2, 0)))
