"""Token log-probabilities and the losses over them against the formulas in 64
bits.

Tolerances.  u = 2^-24 is half a step of fp32 relative to the value.  A term
exp((x - m) / T) is computed as 2^a with a rounded three times (difference,
constant, product: 3 u relative, so 3 u |x - m| / T on the term) and an
exponential good to 2^-22 = 4 u; a thread adds at most V / 256 + 16 terms in
fp32 (u each), warps 5 more, the rest is 64-bit.  Terms' own weights average
their |x - m| / T to at most the row's entropy plus log of the sum, below
2 log V.  So a row's sum of exponentials is good to
  REL = (4 + 6 log V + V / 256 + 21) u
relative, apart from the maximum's own term, which is exact.  Outputs add half
a step of their type: eps / 2 relative."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = 2.0 ** -126  # exponentials below it are 0


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def L():
    from qwen600_engine_b200 import losses
    return losses


def rel_sum(V):
    return (4 + 6 * math.log(max(V, 2)) + V / 256 + 21) * U


def half_step(t):
    return torch.finfo(t).eps / 2


def rows_of(N, V, dtype, seed, kind="mixed", pad=0, shift=0):
    """[N, V] logits on the GPU; pad: extra columns between rows; shift: elements before the first."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn((N, V), generator=g, device="cuda") * (0.5 + 4 * torch.rand((N, 1), generator=g, device="cuda"))
    x += 20 * torch.rand((N, 1), generator=g, device="cuda") - 10
    if kind == "peaked":
        x[torch.arange(N), torch.randint(0, V, (N,), generator=g, device="cuda")] += 40
    if kind == "equal":
        x[:] = 3.0
    buf = torch.full((N * (V + pad) + shift,), 77.0, dtype=dtype, device="cuda")
    view = buf[shift:].view(N, V + pad)[:, :V]
    view.copy_(x)
    tok = torch.randint(0, V, (N,), generator=g, device="cuda", dtype=torch.int32)
    return view, tok, g


def exact(x, tok, T=1.0):
    """(logprob, probabilities, excess, max) in 64 bits, and the tolerance of the logprob."""
    V = x.shape[1]
    d = x.double()
    m = d.amax(1)
    e = ((d - m[:, None]) / T).exp()
    n = (d == m[:, None]).sum(1)
    excess = torch.where(d == m[:, None], torch.zeros_like(e), e).sum(1) + (n - 1)
    total = 1 + excess
    fine = (tok >= 0) & (tok < V)
    at = tok.long().clamp(0, V - 1)[:, None]
    lp = (d.gather(1, at)[:, 0] - m) / T - torch.log1p(excess)
    lp = torch.where(fine, lp, torch.zeros_like(lp))
    tol = rel_sum(V) * excess / total + U * lp.abs() + 1e-12
    return lp, e / total[:, None], excess, m, torch.where(fine, tol, torch.zeros_like(tol))


def grad_of(x, tok, coef, T=1.0):
    """coef * (one-hot - p) / T in 64 bits and its tolerance for fp32 arithmetic, before the output's own rounding."""
    lp, p, excess, m, _ = exact(x, tok, T)
    V = x.shape[1]
    fine = ((tok >= 0) & (tok < V) & (coef != 0))[:, None]
    hot = torch.zeros_like(p)
    hot.scatter_(1, tok.long().clamp(0, V - 1)[:, None], 1.0)
    p_target = p.gather(1, tok.long().clamp(0, V - 1)[:, None])
    q = torch.where(hot > 0, 1 - p, -p)
    # 1 - p of a target that holds nearly everything, without cancellation
    only = (x.double().gather(1, tok.long().clamp(0, V - 1)[:, None])[:, 0] == m)
    q = torch.where((hot > 0) & only[:, None], (excess / (1 + excess))[:, None].expand_as(p), q)
    c = (coef.double() / T)[:, None]
    away = ((m[:, None] - x.double()) / T).clamp(max=100)
    tol = c.abs() * (q.abs() * (rel_sum(V) + 8 * U) + p * (3 * U * away + 4 * U) * (hot == 0)
                     + hot * p_target * rel_sum(V) * (~only)[:, None] + TINY)
    z = torch.zeros_like(p)
    return torch.where(fine, c * q, z), torch.where(fine, tol, z)


def check(got, ref, tol, what):
    got, bad = got.double(), ~torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaNs differ"
    assert torch.equal(got[bad & ~torch.isnan(ref)], ref[bad & ~torch.isnan(ref)]), f"{what}: infinities differ"
    diff, lim = (got - ref).abs()[~bad], tol[~bad] if tol.shape == ref.shape else tol
    assert (diff <= lim).all(), f"{what}: off by {float((diff / lim.clamp(min=1e-300)).max()):.3g} tolerances"


def check_grad(got, ref, tol, what="gradient"):
    h = half_step(got.dtype)
    # half a step of the output's type (of its smallest numbers: half their spacing)
    check(got, ref, tol * (1 + h) + h * ref.abs() + torch.finfo(got.dtype).smallest_normal * 2 * h, what)


SHAPES = [(1, 1), (1, 2), (3, 7), (5, 33), (2, 1000), (4, 1003), (2, 8192), (3, 50021), (3, 151936), (1, 262144), (37, 4099)]
DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V", SHAPES)
@pytest.mark.parametrize("T", [1.0, 0.7])
def test_logprobs_and_backward(dtype, N, V, T):
    x, tok, g = rows_of(N, V, dtype, seed=N * 1000 + V)
    r = L().token_logprobs(x, tok, temperature=T)
    lp, _, excess, m, tol = exact(x, tok, T)
    check(r.logprobs, lp, tol, "logprobs")
    assert torch.equal(r.stats[:, 0].double(), m)
    check(r.stats[:, 1], excess, (rel_sum(V) + U) * excess + 1e-30, "excess")
    gl = torch.randn((N,), generator=g, device="cuda")
    out = L().token_logprobs_backward(x, tok, r.stats, gl, temperature=T)
    assert out.dtype == dtype and out.shape == x.shape
    check_grad(out, *grad_of(x, tok, gl, T))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["peaked", "equal"])
@pytest.mark.parametrize("T", [1e-6, 1.0, 50.0])
def test_logprobs_of_peaked_and_equal_rows(dtype, kind, T):
    N, V = 4, 5003
    x, tok, g = rows_of(N, V, dtype, seed=11, kind=kind)
    tok[:3] = x[:3].argmax(1).to(torch.int32)
    r = L().token_logprobs(x, tok, temperature=T)
    lp, _, excess, _, tol = exact(x, tok, T)
    # a log-probability near 0 keeps its relative precision
    check(r.logprobs, lp, torch.where(lp.abs() < 0.5, (rel_sum(V) + 4 * U) * lp.abs() + 1e-30, tol), "logprobs")
    gl = torch.randn((N,), generator=g, device="cuda")
    check_grad(L().token_logprobs_backward(x, tok, r.stats, gl, temperature=T), *grad_of(x, tok, gl, T))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,pad,shift", [(1000, 24, 0), (1000, 3, 0), (1003, 0, 1), (4099, 5, 3), (151936, 64, 8), (50021, 0, 5)])
def test_strides_and_alignment(dtype, V, pad, shift):
    """Rows at any element alignment; the gradient's buffer at another; elements between rows stay as they were."""
    N = 5
    x, tok, g = rows_of(N, V, dtype, seed=V + pad, pad=pad, shift=shift)
    r = L().token_logprobs(x, tok)
    lp, _, _, _, tol = exact(x, tok)
    check(r.logprobs, lp, tol, "logprobs")
    gl = torch.randn((N,), generator=g, device="cuda")
    ref = grad_of(x, tok, gl)
    for gpad, gshift in ((pad, shift), (pad + 1, shift + 1), (0, 0)):
        buf = torch.full((N * (V + gpad) + gshift,), 55.0, dtype=dtype, device="cuda")
        out = buf[gshift:].view(N, V + gpad)[:, :V]
        L().token_logprobs_backward(x, tok, r.stats, gl, out=out)
        check_grad(out, *ref)
        assert (buf[:gshift] == 55).all() and (buf[gshift:].view(N, V + gpad)[:, V:] == 55).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_and_special_logits(dtype):
    V = 2003
    x, tok, _ = rows_of(12, V, dtype, seed=5)
    low = torch.finfo(dtype).min
    x[0, 1::2] = -math.inf                    # masked tokens
    x[1, :] = -math.inf
    x[1, 17] = 2.5                            # one token left
    x[2, :] = -math.inf                       # nothing left
    x[3, :] = low                             # the type's lowest value everywhere: uniform
    x[4, 500:] = low                          # masked with it
    x[5, 9] = math.nan
    x[6, 9] = math.inf
    x[7, :1990] = -math.inf                   # only a tail left
    x[8, :] = torch.finfo(dtype).max
    x[9, 3] = torch.finfo(dtype).max          # and the others far below
    x[10, :] = math.nan
    x[11, :1000] = math.nan
    x[11, 1000:] = -math.inf
    tok[0], tok[1], tok[4], tok[7], tok[9] = 2, 17, 3, 2001, 3
    r = L().token_logprobs(x, tok)
    lp = torch.log_softmax(x.double(), 1).gather(1, tok.long()[:, None])[:, 0]
    lp[3] = -math.log(V)
    lp[8] = -math.log(V)
    check(r.logprobs, lp, rel_sum(V) + U * lp.abs().nan_to_num(0, 0, 0) + 1e-12, "logprobs")
    assert torch.isnan(r.logprobs).nonzero()[:, 0].tolist() == [2, 5, 6, 10, 11]
    tok[0] = 3                                # a masked token
    r = L().token_logprobs(x, tok)
    assert float(r.logprobs[0]) == -math.inf
    gl = torch.full((12,), 0.5, device="cuda")
    out = L().token_logprobs_backward(x, tok, r.stats, gl).double()
    p = torch.softmax(x.double(), 1)
    p[3], p[8] = 1 / V, 1 / V
    hot = torch.zeros_like(p).scatter_(1, tok.long()[:, None], 1.0)
    ref = 0.5 * (hot - p)
    check(out, ref, (rel_sum(V) + 100 * U + half_step(dtype)) * ref.abs().nan_to_num(0) + 4 * U * rel_sum(V) + 1e-30, "gradient")


# Large calls (from 24 or 72 MB of logits) take the kernels that stream many rows.
MANY = [(torch.bfloat16, 250, 151936, 0, 0), (torch.bfloat16, 800, 50021, 3, 1), (torch.float32, 128, 151936, 0, 0),
        (torch.float32, 500, 37999, 1, 2), (torch.bfloat16, 38000, 1003, 0, 0), (torch.float32, 19000, 1024, 8, 0),
        (torch.bfloat16, 150, 262144, 0, 0)]


@pytest.mark.parametrize("dtype,N,V,pad,shift", MANY)
@pytest.mark.parametrize("kind", ["mixed", "peaked"])
def test_many_rows(dtype, N, V, pad, shift, kind):
    x, tok, g = rows_of(N, V, dtype, seed=N + V, pad=pad, shift=shift, kind=kind)
    tok[::2] = x[::2].argmax(1).to(torch.int32)
    tok[3::11] = -1
    x[3::22] = math.nan
    T = 0.8
    r = L().token_logprobs(x, tok, temperature=T)
    again = L().token_logprobs(x, tok, temperature=T)
    assert torch.equal(r.logprobs, again.logprobs) and torch.equal(r.stats, again.stats)
    x[3::22] = 0
    out = (tok == -1).nonzero()[:, 0]
    assert (r.logprobs[out] == 0).all() and (r.stats[out] == 0).all()
    for a in range(0, N, 512):
        b = slice(a, min(a + 512, N))
        lp, _, excess, m, tol = exact(x[b], tok[b], T)
        # a log-probability near 0 keeps its relative precision
        near = (rel_sum(V) + 4 * U) * lp.abs() + 1e-30
        check(r.logprobs[b], lp, torch.where((lp.abs() < 0.5) & (tok[b] >= 0), near, tol), "logprobs")
        on = tok[b] >= 0
        assert torch.equal(r.stats[b][on, 0].double(), m[on])
        check(r.stats[b][on, 1], excess[on], (rel_sum(V) + U) * excess[on] + 1e-30, "excess")


def test_many_rows_with_special_logits():
    N, V = 300, 131075
    x, tok, _ = rows_of(N, V, torch.bfloat16, seed=15)
    low = torch.finfo(torch.bfloat16).min
    x[0, 1::2] = -math.inf
    x[1, :] = -math.inf
    x[1, 17] = 2.5
    x[2, :] = -math.inf
    x[3, :] = low
    x[4, 500:] = low
    x[5, 9] = math.nan
    x[6, V - 1] = math.inf
    x[7, : V - 13] = -math.inf
    x[8, :] = torch.finfo(torch.bfloat16).max
    x[9, 3] = torch.finfo(torch.bfloat16).max
    x[10, :] = math.nan
    x[11, :100000] = math.nan
    x[11, 100000:] = -math.inf
    x[12, :] = 0.0
    tok[0], tok[1], tok[4], tok[7], tok[9] = 2, 17, 3, V - 2, 3
    r = L().token_logprobs(x, tok)
    lp = torch.log_softmax(x.double(), 1).gather(1, tok.long()[:, None])[:, 0]
    lp[3] = lp[8] = lp[12] = -math.log(V)
    check(r.logprobs, lp, rel_sum(V) + U * lp.abs().nan_to_num(0, 0, 0) + 1e-12, "logprobs")
    assert torch.isnan(r.logprobs).nonzero()[:, 0].tolist() == [2, 5, 6, 10, 11]


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 151936), (torch.float32, 50021)])
def test_preference_many_rows(dtype, V):
    x, tok, off, ref, w = pairs_case(4, V, dtype, seed=V + 2, lengths=[60, 1, 82, 44, 34, 72, 0, 98], tail=2)
    r = L().preference_loss(x, tok, off, ref, weights=w, beta=0.2, label_smoothing=0.1)
    check_preference(r, x, tok, off, ref, w, 0.2, 0.1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_score_nothing(dtype):
    """Tokens outside the vocabulary: log-probability 0, zero gradient, logits not used."""
    N, V = 9, 3001
    x, tok, g = rows_of(N, V, dtype, seed=6)
    tok[1], tok[3], tok[5], tok[7] = -1, V, -2147483648, 2147483647
    out_rows = [1, 3, 5, 7]
    x[out_rows] = math.nan
    r = L().token_logprobs(x, tok)
    assert (r.logprobs[out_rows] == 0).all() and (r.stats[out_rows] == 0).all()
    gl = torch.randn((N,), generator=g, device="cuda")
    gl[2] = 0.0
    x[2] = math.nan
    out = L().token_logprobs_backward(x, tok, r.stats, gl)
    assert (out[out_rows + [2]] == 0).all()
    keep = [0, 4, 6, 8]
    check_grad(out[keep], *grad_of(x[keep], tok[keep], gl[keep]))


def policy_case(N, V, dtype, seed, T=1.0, kl=0.1, **kw):
    x, tok, g = rows_of(N, V, dtype, seed, **kw)
    lp = exact(x, tok, T)[0]
    step = 0.3 * torch.randn((N,), generator=g, device="cuda", dtype=torch.float64)
    ratio = step.exp()
    near = ((ratio - 0.8).abs() < 1e-3) | ((ratio - 1.25).abs() < 1e-3)  # a rounding there would choose the branch
    old = (lp - torch.where(near, step + 0.01, step)).float()
    ref = (lp + 0.3 * torch.randn((N,), generator=g, device="cuda")).float()
    adv = torch.randn((N,), generator=g, device="cuda")
    w = torch.rand((N,), generator=g, device="cuda") / N
    return x, tok, old, ref, adv, w


def policy_exact(x, tok, old, ref, adv, w, lo, hi, kl, T):
    """(loss, its tolerance, logprobs, their tolerance, coefficients, their tolerance) in 64 bits."""
    lp, _, _, _, tol = exact(x, tok, T)
    fine = (tok >= 0) & (tok < x.shape[1]) & (w != 0)
    a, w = adv.double(), w.double()
    r = (lp - old.double()).exp()
    surr = -torch.minimum(r * a, r.clamp(1 - lo, 1 + hi) * a)
    cut = ((a > 0) & (r > 1 + hi)) | ((a < 0) & (r < 1 - lo))
    slope = torch.where(cut, torch.zeros_like(a), -a * r)
    bend = (r * a).abs()  # how far l and the slope move with the log-probability
    if kl:
        d = ref.double() - lp
        surr = surr + kl * (d.exp() - d - 1)
        slope = slope + kl * (1 - d.exp())
        bend = bend + kl * (d.exp() + 1)
    z = torch.zeros_like(lp)
    each = torch.where(fine, w * surr, z)
    c = torch.where(fine, w * slope, z)
    ctol = torch.where(fine, w.abs() * bend * (tol * 1.01 + 1e-12) + U * c.abs(), z)
    ltol = (torch.where(fine, w.abs() * bend * tol * 1.01, z)).sum() + U * each.sum().abs() + 1e-12
    return each.sum(), ltol, torch.where(fine, lp, z), torch.where(fine, tol, z), c, ctol


def check_policy(r, case, lo, hi, kl, T):
    x, tok = case[0], case[1]
    loss, ltol, lp, tol, c, ctol = policy_exact(*case, lo, hi, kl, T)
    check(r.loss, loss, ltol, "loss")
    check(r.logprobs, lp, tol, "logprobs")
    if r.grad is not None:
        ref, gtol = grad_of(x, tok, c, T)
        unit = torch.where(c[:, None] != 0, ref / torch.where(c == 0, torch.ones_like(c), c)[:, None], torch.zeros_like(ref))
        check_grad(r.grad, ref, gtol + unit.abs() * ctol[:, None])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V", [(1, 1), (1, 5), (3, 33), (7, 1003), (5, 8192), (33, 4099), (3, 151936), (2, 262144), (300, 257)])
@pytest.mark.parametrize("kl,T", [(0.0, 1.0), (0.1, 0.7)])
def test_policy_loss(dtype, N, V, kl, T):
    x, tok, old, ref, adv, w = case = policy_case(N, V, dtype, seed=N + V, T=T)
    r = L().policy_loss(x, tok, old, adv, ref_logprobs=ref if kl else None, weights=w, clip_low=0.2, clip_high=0.25,
                        kl_coef=kl, temperature=T)
    check_policy(r, case, 0.2, 0.25, kl, T)
    alone = L().policy_loss(x, tok, old, adv, ref_logprobs=ref, weights=w, clip_low=0.2, clip_high=0.25, kl_coef=kl,
                            temperature=T, grad=False)
    assert alone.grad is None and torch.equal(alone.loss, r.loss) and torch.equal(alone.logprobs, r.logprobs)


def test_policy_loss_default_weights_and_masks():
    N, V = 12, 2003
    x, tok, old, ref, adv, w = policy_case(N, V, torch.bfloat16, seed=3)
    r = L().policy_loss(x, tok, old, adv, ref_logprobs=ref, kl_coef=0.05)
    check_policy(r, (x, tok, old, ref, adv, torch.full_like(w, 1.0) / N), 0.2, 0.2, 0.05, 1.0)
    # rows left out by weight or by token are not read
    w[2], w[5], tok[7] = 0.0, -0.0, -1
    x[[2, 5, 7]] = math.nan
    old[2] = math.nan
    r = L().policy_loss(x, tok, old, adv, ref_logprobs=ref, weights=w, kl_coef=0.05)
    assert (r.grad[[2, 5, 7]] == 0).all() and (r.logprobs[[2, 5, 7]] == 0).all()
    keep = [0, 1, 3, 4, 6, 8, 9, 10, 11]
    sub = tuple(t[keep] for t in (x, tok, old, ref, adv, w))
    check_policy(type(r)(r.loss, r.logprobs[keep], r.grad[keep]), sub, 0.2, 0.2, 0.05, 1.0)
    # nothing left
    none = L().policy_loss(x, tok, old, adv, weights=torch.zeros_like(w))
    assert float(none.loss) == 0 and (none.grad == 0).all() and (none.logprobs == 0).all()
    empty = L().policy_loss(x[:0], tok[:0], old[:0], adv[:0])
    assert float(empty.loss) == 0 and empty.grad.shape == (0, V)


def test_policy_branches():
    """Each side of the clip range with each sign of the advantage, and an advantage of 0."""
    V = 1000
    x, tok, old, ref, adv, w = policy_case(10, V, torch.float32, seed=8)
    lp = exact(x, tok)[0]
    shift = torch.tensor([0.5, 0.5, -0.5, -0.5, 0.0, 0.0, 0.5, -0.5, 0.1, -0.1], device="cuda", dtype=torch.float64)
    old = (lp - shift).float()
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 2.0, -2.0, 0.0, 0.0, 1.0, 1.0], device="cuda")
    r = L().policy_loss(x, tok, old, adv, weights=w)
    check_policy(r, (x, tok, old, ref, adv, w), 0.2, 0.2, 0.0, 1.0)
    zero = (r.grad == 0).all(1).tolist()
    assert zero == [True, False, False, True, False, False, True, True, False, False]


def pairs_case(P, V, dtype, seed, longest=9, tail=3, lengths=None):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    if lengths is None:
        lengths = torch.randint(0, longest + 1, (2 * P,), generator=g)
    off = torch.cat([torch.zeros(1, dtype=torch.long), torch.as_tensor(lengths).cumsum(0)])
    x, tok, gc = rows_of(int(off[-1]) + tail, V, dtype, seed)
    tok[torch.rand(tok.shape, generator=gc, device="cuda") < 0.25] = -1
    lp = exact(x, tok)[0]
    o = off.tolist()
    seq = torch.stack([lp[a:b].sum() for a, b in zip(o, o[1:])])
    ref = (seq + 4 * torch.randn((2 * P,), generator=gc, device="cuda")).float()
    return x, tok, off.to(torch.int32).cuda(), ref, torch.rand((P,), generator=gc, device="cuda")


def check_preference(r, x, tok, off, ref, w, beta, eps):
    lp, _, _, _, tol = exact(x, tok)
    o = off.tolist()
    P = len(o) // 2
    seq = torch.stack([lp[a:b].sum() for a, b in zip(o, o[1:])])
    stol = torch.stack([tol[a:b].sum() for a, b in zip(o, o[1:])]) + 1e-12
    check(r.seq_logprobs, seq, stol + U * seq.abs(), "seq_logprobs")
    w = torch.full((P,), 1.0 / P, dtype=torch.float64, device=x.device) if w is None else w.double()
    d = seq - ref.double()
    z = beta * (d[:P] - d[P:])
    ztol = beta * (stol[:P] + stol[P:]) + 1e-13
    ls = torch.nn.functional.logsigmoid
    each = w * (-(1 - eps) * ls(z) - eps * ls(-z))
    check(r.loss, each.sum(), (w * ztol).sum() + U * each.sum().abs() + 1e-12, "loss")
    slope = -beta * w * ((1 - eps) * torch.sigmoid(-z) - eps * torch.sigmoid(z))
    coef = torch.zeros_like(lp)
    ctol = torch.zeros_like(lp)
    for q, (a, b) in enumerate(zip(o, o[1:])):
        coef[a:b] = slope[q % P] * (1 if q < P else -1)
        ctol[a:b] = beta * w[q % P] * ztol[q % P] + U * slope[q % P].abs()
    grad, gtol = grad_of(x, tok, coef)
    unit = torch.where(coef[:, None] != 0, grad / torch.where(coef == 0, torch.ones_like(coef), coef)[:, None], torch.zeros_like(grad))
    check_grad(r.grad, grad, gtol + unit.abs() * ctol[:, None])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("P,V", [(1, 7), (1, 1003), (3, 8192), (2, 151936), (40, 257), (5, 50021)])
@pytest.mark.parametrize("eps,weighted", [(0.0, False), (0.1, True)])
def test_preference_loss(dtype, P, V, eps, weighted):
    x, tok, off, ref, w = pairs_case(P, V, dtype, seed=P * 7 + V, longest=4 if V > 100000 else 9)
    w = w if weighted else None
    r = L().preference_loss(x, tok, off, ref, weights=w, beta=0.2, label_smoothing=eps)
    check_preference(r, x, tok, off, ref, w, 0.2, eps)
    assert (r.grad[int(off[-1]):] == 0).all()  # rows behind the last sequence
    alone = L().preference_loss(x, tok, off, ref, weights=w, beta=0.2, label_smoothing=eps, grad=False)
    assert alone.grad is None and torch.equal(alone.loss, r.loss) and torch.equal(alone.seq_logprobs, r.seq_logprobs)


def test_preference_lengths_of_zero_and_one():
    x, tok, off, ref, w = pairs_case(4, 1003, torch.float32, seed=9, lengths=[0, 1, 0, 3, 0, 0, 1, 1])
    r = L().preference_loss(x, tok, off, ref, beta=0.3)
    check_preference(r, x, tok, off, ref, None, 0.3, 0.0)
    none = L().preference_loss(x, tok, off[:1], ref[:0], beta=0.3)  # no pairs
    assert float(none.loss) == 0 and (none.grad == 0).all() and none.seq_logprobs.numel() == 0
    empty = L().preference_loss(x[:0], tok[:0], torch.zeros_like(off), ref, beta=0.3)
    assert empty.grad.shape == (0, 1003) and math.isfinite(float(empty.loss))


def test_preference_far_ratios_and_left_out_pairs():
    x, tok, off, ref, w = pairs_case(3, 501, torch.float32, seed=12, lengths=[3, 4, 2, 3, 1, 5])
    ref[0] += 1e5    # the loss is linear there
    ref[4] += 1e5    # and nothing here
    r = L().preference_loss(x, tok, off, ref, beta=0.5, weights=w)
    check_preference(r, x, tok, off, ref, w, 0.5, 0.0)
    w[2] = 0.0       # a pair left out, whose reference is not a number
    ref[2] = math.nan
    r = L().preference_loss(x, tok, off, ref, beta=0.5, weights=w)
    o = off.tolist()
    assert math.isfinite(float(r.loss)) and (r.grad[o[2]:o[3]] == 0).all() and (r.grad[o[5]:o[6]] == 0).all()


@pytest.mark.parametrize("spoil", [[0, 5, 3, 8, 9], [-4, 2, 4, 6, 8], [0, 2, 4, 6, 1000000], [0, 2, 4, 6, 2147483647]])
def test_preference_offsets_out_of_order(spoil):
    """A pair whose offsets fall or leave the rows: NaN, and none of its rows touched."""
    x, tok, _, _, _ = pairs_case(2, 301, torch.float32, seed=13, lengths=[3, 3, 3, 3])
    off = torch.tensor(spoil, dtype=torch.int32, device="cuda")
    ref = torch.zeros(4, device="cuda")
    r = L().preference_loss(x, tok, off, ref)
    assert math.isnan(float(r.loss))
    assert not torch.isnan(r.grad).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_in_place_of_the_logits(dtype):
    for V, pad in ((4099, 0), (151936, 0), (1003, 5)):
        case = policy_case(6, V, dtype, seed=V, pad=pad)
        x, tok, old, ref, adv, w = case
        keep = x.clone()
        r = L().policy_loss(x, tok, old, adv, weights=w)
        y = torch.empty_strided(x.shape, x.stride(), dtype=dtype, device="cuda").copy_(keep)
        s = L().policy_loss(y, tok, old, adv, weights=w, out=y)
        assert s.grad is y and torch.equal(s.grad, r.grad) and torch.equal(s.loss, r.loss)
        y = keep.clone()
        t = L().token_logprobs(y, tok)
        a = L().token_logprobs_backward(y, tok, t.stats, adv)
        b = L().token_logprobs_backward(y, tok, t.stats, adv, out=y)
        assert b is y and torch.equal(a, b)
        x, tok, off, ref, _ = pairs_case(2, V, dtype, seed=V + 1)
        a = L().preference_loss(x, tok, off, ref)
        b = L().preference_loss(x, tok, off, ref, out=x)
        assert b.grad is x and torch.equal(a.grad, b.grad) and torch.equal(a.loss, b.loss)


def test_gradients_against_differences():
    """Central differences of the kernels' own losses along random directions, fp32, vocabulary of 40.  With step h the
    third derivative's h^2 / 6 |loss'''| (below 8 |direction|^3 here: each factor of p, r and sigmoid is at most 1.5) and the
    loss's fp32 rounding 2^-24 |loss| / h are the error."""
    V, h = 40, 2.0 ** -6
    x, tok, old, ref, adv, w = policy_case(6, V, torch.float32, seed=21)
    lp = exact(x, tok)[0]
    old = (lp - torch.tensor([0.05, -0.1, 0.4, -0.4, 0.0, 0.1], device="cuda")).float()  # no border within a step
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 0.5, -0.5], device="cuda")

    def policy(y, grad):
        return L().policy_loss(y, tok, old, adv, ref_logprobs=ref, weights=w, kl_coef=0.1, grad=grad)

    p, ptok, off, pref, _ = pairs_case(2, V, torch.float32, seed=22, lengths=[2, 3, 1, 2])

    def preference(y, grad):
        return L().preference_loss(y, ptok, off, pref, beta=0.3, grad=grad)

    for fn, z in ((policy, x), (preference, p)):
        g = fn(z, True).grad.double()
        for seed in range(8):
            gen = torch.Generator(device="cuda")
            gen.manual_seed(seed)
            d = torch.randn(z.shape, generator=gen, device="cuda")
            d /= d.norm(dim=1).amax()
            up, down = (float(fn((z + s * h * d).contiguous(), False).loss) for s in (1, -1))
            far = (z + h * d).double() - (z - h * d).double()  # the step as it was rounded
            want = float((g * far).sum()) / (2 * h)
            tol = 8 * h * h / 6 * float(d.norm() ** 3) + 2 ** -24 * (abs(up) + abs(down)) / h + 1e-7
            assert abs((up - down) / (2 * h) - want) <= tol, (fn.__name__, seed)


def test_autograd_takes_the_gradient():
    x, tok, old, ref, adv, w = policy_case(5, 700, torch.float32, seed=31)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    h = torch.randn((5, 16), generator=g, device="cuda")
    weight = torch.randn((700, 16), generator=g, device="cuda", requires_grad=True)
    logits = h @ weight.t()
    r = L().policy_loss(logits, tok, old, adv, weights=w)
    logits.backward(r.grad)
    check(weight.grad, r.grad.double().t() @ h.double(), 16 * U * (r.grad.double().abs().t() @ h.double().abs()) + 1e-12, "weight")


def test_same_inputs_same_bits():
    case = policy_case(64, 151936, torch.bfloat16, seed=41)
    x, tok, old, ref, adv, w = case
    a = L().policy_loss(x, tok, old, adv, ref_logprobs=ref, weights=w, kl_coef=0.1)
    for _ in range(3):
        b = L().policy_loss(x, tok, old, adv, ref_logprobs=ref, weights=w, kl_coef=0.1)
        assert torch.equal(a.loss, b.loss) and torch.equal(a.logprobs, b.logprobs) and torch.equal(a.grad, b.grad)


def test_offsets_beyond_32_bits():
    """Rows more than 2^31 elements apart in all."""
    N, V, ld = 4, 1003, (1 << 30) + 8
    buf = torch.empty(((N - 1) * ld + V,), dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((N, V), (ld, 1))
    y, tok, g = rows_of(N, V, torch.bfloat16, seed=51)
    x.copy_(y)
    a = L().token_logprobs(x, tok)
    lp, _, excess, m, tol = exact(y, tok)  # rows at other alignments add their terms in another order
    check(a.logprobs, lp, tol, "logprobs")
    check(a.stats[:, 1], excess, (rel_sum(V) + U) * excess, "excess")
    gl = torch.randn((N,), generator=g, device="cuda")
    ref = grad_of(y, tok, gl)
    L().token_logprobs_backward(x, tok, a.stats, gl, out=x)
    check_grad(x, *ref)
    del buf, x
    torch.cuda.empty_cache()


def test_streams():
    """A call on a side stream that waits for its inputs; two calls at once on two streams."""
    cases = [policy_case(48, 50021, torch.bfloat16, seed=s) for s in (61, 62)]
    want = [L().policy_loss(c[0], c[1], c[2], c[4], weights=c[5]) for c in cases]
    pair = pairs_case(3, 50021, torch.bfloat16, seed=63)
    pw = L().preference_loss(*pair[:4])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        got = [L().policy_loss(c[0], c[1], c[2], c[4], weights=c[5], stream=s) for c, s in zip(cases, streams)]
        pg = L().preference_loss(*pair[:4], stream=streams[0])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.loss, b.loss) and torch.equal(a.grad, b.grad)
        assert torch.equal(pg.loss, pw.loss) and torch.equal(pg.grad, pw.grad)


def test_captured_graphs():
    """Two captured graphs whose replays overlap, on inputs that change between replays."""
    cases = [policy_case(16, 8192, torch.bfloat16, seed=s) for s in (71, 72)]
    pair = pairs_case(2, 8192, torch.bfloat16, seed=73)
    graphs, outs = [], []
    for c in cases:
        L().policy_loss(c[0], c[1], c[2], c[4], weights=c[5])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = L().policy_loss(c[0], c[1], c[2], c[4], weights=c[5])
            q = L().preference_loss(*pair[:4])
            t = L().token_logprobs(c[0], c[1])
        graphs.append(g)
        outs.append((r, q, t))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in (74, 75):
        for c in cases:
            c[0].copy_(rows_of(16, 8192, torch.bfloat16, seed=seed)[0])
        want = [L().policy_loss(c[0], c[1], c[2], c[4], weights=c[5]) for c in cases]
        pw = L().preference_loss(*pair[:4])
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for (r, q, t), w in zip(outs, want):
            assert torch.equal(r.loss, w.loss) and torch.equal(r.grad, w.grad)
            assert torch.equal(q.loss, pw.loss) and torch.equal(q.grad, pw.grad)
            assert torch.equal(t.logprobs, w.logprobs)
    for g in graphs:
        g.reset()


def test_large_calls_captured_and_on_streams():
    """The streaming kernels in a graph, replayed on changed logits while another stream runs the same calls."""
    c = policy_case(300, 151936, torch.bfloat16, seed=91)
    pair = pairs_case(3, 151936, torch.bfloat16, seed=92, lengths=[60, 50, 30, 70, 20, 50], tail=1)
    gl = torch.ones((300,), device="cuda")

    def calls():
        t = L().token_logprobs(c[0], c[1])
        return (t.logprobs, t.stats, L().token_logprobs_backward(c[0], c[1], t.stats, gl),
                *L().policy_loss(c[0], c[1], c[2], c[4], weights=c[5]), *L().preference_loss(*pair[:4]))

    calls()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = calls()
    c[0].copy_(rows_of(300, 151936, torch.bfloat16, seed=93)[0])
    pair[0].mul_(0.5)
    want = calls()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        g.replay()
        with torch.cuda.stream(side):
            other = calls()
        torch.cuda.synchronize()
        for a, b, d in zip(outs, want, other):
            assert torch.equal(a, b) and torch.equal(d, b)
    g.reset()


def test_refused_on_the_gpu():
    from qwen600_engine_b200._lib import SamplerError
    x, tok, old, ref, adv, w = policy_case(4, 100, torch.float32, seed=81)
    with pytest.raises(SamplerError, match="overlaps"):
        L().policy_loss(x[:2], tok[:2], old[:2], adv[:2], out=x[1:3])
    with pytest.raises(SamplerError, match="clip"):
        L().policy_loss(x, tok, old, adv, clip_low=2.0)
    with pytest.raises(SamplerError, match="needs ref"):
        L().policy_loss(x, tok, old, adv, kl_coef=0.1)
    with pytest.raises(SamplerError, match="temperature"):
        L().token_logprobs(x, tok, temperature=0.0)
    with pytest.raises(SamplerError, match="on cuda"):
        L().token_logprobs(x, tok.cpu())
    with pytest.raises(SamplerError, match="vocab"):
        L().token_logprobs(torch.zeros((1, 300000), device="cuda"), tok[:1])


# Finite masks: numbers so low that a logit next to them has no weight, and rows that hold nothing else.  The tolerances
# are those above: a row's terms are taken against its maximum, however far from zero that lies.
MASKS = [-1e7, -2e7, -1e9, -1e10, -1e20, -1e30, None]  # None: the type's lowest value


def masked_rows(N, V, dtype, seed):
    """Ordinary rows with masked stretches, with few tokens left, with nothing but the mask, with the mask beside -inf or
    beside the type's lowest value, with the mask added to the logits, and far above zero; and a token that is not below
    the row's other values by more than ordinary logits are."""
    x, tok, g = rows_of(N, V, dtype, seed)
    low = torch.finfo(dtype).min
    col = torch.arange(V, device="cuda")
    for i in range(N):
        mask = MASKS[i // 7 % len(MASKS)]
        mask = low if mask is None else mask
        t = int(tok[i])
        ends = torch.full_like(x[i], mask)
        if i % 7 == 0:    # the middle half
            ends[: V // 4], ends[V - V // 4:] = x[i, : V // 4], x[i, V - V // 4:]
        elif i % 7 == 1:  # a dozen tokens left
            ends[torch.randint(0, V, (12,), generator=g, device="cuda")] = 1.5
        elif i % 7 == 3:  # mask and -inf in turn, in stretches
            ends[col // 300 % 2 == 1] = -math.inf
        elif i % 7 == 4:  # mask and the type's lowest value, token by token
            ends[1::2] = low
        elif i % 7 == 5:  # added to the logits, as far as the type holds the sum
            ends = (x[i].float() + max(mask, low / 2)).to(dtype)
        elif i % 7 == 6:
            ends = (x[i].float() - max(mask, low / 2)).to(dtype)
        x[i] = ends
        if i % 7 < 2:
            x[i, t] = 2.0
        else:
            tok[i] = x[i].argmax()
    return x, tok, g


MASKED_T = [0.6, 0.7, 1.0, 1.5, 2.0]


def check_logprobs(r, x, tok, T):
    V = x.shape[1]
    for a in range(0, x.shape[0], 256):
        b = slice(a, a + 256)
        lp, _, excess, m, tol = exact(x[b], tok[b], T)
        check(r.logprobs[b], lp, tol, "logprobs")
        assert torch.equal(r.stats[b, 0].double(), m)
        check(r.stats[b, 1], excess, (rel_sum(V) + U) * excess + 1e-30, "excess")


@pytest.mark.parametrize("T", MASKED_T)
@pytest.mark.parametrize("dtype,N,V", [(torch.bfloat16, 250, 151936), (torch.float32, 130, 50021), (torch.bfloat16, 3200, 4099)])
def test_finite_masks_in_many_rows(dtype, N, V, T):
    x, tok, _ = masked_rows(N, V, dtype, seed=V)
    check_logprobs(L().token_logprobs(x, tok, temperature=T), x, tok, T)


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 151936), (torch.float32, 50021)])
def test_finite_masks_in_many_rows_of_pairs(dtype, V):
    lengths = [60, 1, 82, 44, 34, 72, 0, 98]
    x, tok, g = masked_rows(sum(lengths) + 2, V, dtype, seed=V + 1)
    off = torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)
    lp = exact(x, tok)[0]
    seq = torch.stack([lp[a:b].sum() for a, b in zip(off.tolist(), off.tolist()[1:])])
    ref = (seq + 4 * torch.randn((8,), generator=g, device="cuda")).float()
    r = L().preference_loss(x, tok, off, ref, beta=0.2)
    check_preference(r, x, tok, off, ref, None, 0.2, 0.0)


def policy_around(x, tok, g, T):
    """Inputs of the policy loss for given logits: ratios on both sides of the clip range, none at a border."""
    N = x.shape[0]
    lp = exact(x, tok, T)[0]
    step = 0.3 * torch.randn((N,), generator=g, device="cuda", dtype=torch.float64)
    near = ((step.exp() - 0.8).abs() < 1e-3) | ((step.exp() - 1.25).abs() < 1e-3)
    old = (lp - torch.where(near, step + 0.01, step)).float()
    ref = (lp + 0.3 * torch.randn((N,), generator=g, device="cuda")).float()
    return x, tok, old, ref, torch.randn((N,), generator=g, device="cuda"), torch.rand((N,), generator=g, device="cuda") / N


@pytest.mark.parametrize("T", MASKED_T)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V", [(49, 257), (49, 5003), (49, 50021), (21, 151936)])
def test_finite_masks_in_few_rows(dtype, N, V, T):
    x, tok, g = masked_rows(N, V, dtype, seed=N + V)
    r = L().token_logprobs(x, tok, temperature=T)
    check_logprobs(r, x, tok, T)
    gl = torch.randn((N,), generator=g, device="cuda")
    check_grad(L().token_logprobs_backward(x, tok, r.stats, gl, temperature=T), *grad_of(x, tok, gl, T))
    case = policy_around(x, tok, g, T)
    alone = L().policy_loss(x, tok, case[2], case[4], ref_logprobs=case[3], weights=case[5], clip_low=0.2, clip_high=0.25,
                            kl_coef=0.1, temperature=T, grad=False)
    check_policy(alone, case, 0.2, 0.25, 0.1, T)


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 5003), (torch.float32, 257)])
def test_finite_masks_in_few_rows_of_pairs(dtype, V):
    lengths = [9, 1, 8, 7, 12, 7, 0, 4]
    x, tok, g = masked_rows(sum(lengths) + 2, V, dtype, seed=V + 1)
    off = torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)
    lp = exact(x, tok)[0]
    seq = torch.stack([lp[a:b].sum() for a, b in zip(off.tolist(), off.tolist()[1:])])
    ref = (seq + 4 * torch.randn((8,), generator=g, device="cuda")).float()
    check_preference(L().preference_loss(x, tok, off, ref, beta=0.2), x, tok, off, ref, None, 0.2, 0.0)


@pytest.mark.parametrize("T", MASKED_T)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V", [(49, 257), (49, 5003), (49, 50021), (21, 151936)])
def test_finite_masks_in_the_policy_gradient(dtype, N, V, T):
    x, tok, g = masked_rows(N, V, dtype, seed=N + V + 1)
    case = policy_around(x, tok, g, T)
    r = L().policy_loss(x, tok, case[2], case[4], ref_logprobs=case[3], weights=case[5], clip_low=0.2, clip_high=0.25,
                        kl_coef=0.1, temperature=T)
    check_policy(r, case, 0.2, 0.25, 0.1, T)


@pytest.mark.parametrize("P,spoil", [(2, {1: 6, 2: 3}), (2, {4: 2}), (40, {80: 100}), (40, {41: 70})])
def test_preference_offsets_that_fall_anywhere(P, spoil):
    """Sequences could share rows then: every pair's sums are NaN and no row has a gradient, also where the pair beside the
    fall has no weight."""
    x, tok, off, ref, w = pairs_case(P, 301, torch.float32, seed=14, lengths=[3] * (2 * P))
    r = L().preference_loss(x, tok, off, ref, weights=w)
    assert math.isfinite(float(r.loss)) and (r.grad != 0).any()
    for i, v in spoil.items():
        off[i] = v
    for q in range(2 * P):
        if off[q] > off[q + 1]:
            w[q % P] = 0.0
    r = L().preference_loss(x, tok, off, ref, weights=w)
    assert math.isnan(float(r.loss)) and torch.isnan(r.seq_logprobs).all()
    assert (r.grad == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_gradient_in_place_is_seen_by_autograd(dtype):
    """Logits that autograd keeps for its backward and that a gradient replaced are reported, not used."""
    x, tok, old, _, adv, w = policy_case(5, 700, dtype, seed=95)
    off = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda")
    stats = L().token_logprobs(x, tok).stats
    calls = [lambda y: L().policy_loss(y, tok, old, adv, weights=w, out=y),
             lambda y: L().token_logprobs_backward(y, tok, stats, adv, out=y),
             lambda y: L().preference_loss(y, tok, off, adv[:2], out=y)]
    for call in calls:
        leaf = x.clone().requires_grad_(True)
        y = leaf * 1.0
        kept = (y * y).sum()
        call(y)
        with pytest.raises(RuntimeError, match="inplace"):
            kept.backward()
        with torch.inference_mode():
            z = x.clone()
        call(z)  # tensors without a version
        y = x.clone()
        before = y._version
        L().policy_loss(y, tok, old, adv, weights=w)
        assert y._version == before  # only read


def test_gradient_beside_another_loss():
    """The documented way to take a loss of these together with one of autograd's; without a history of its own it
    cannot be taken for one of them."""
    x, tok, old, _, adv, w = policy_case(5, 300, torch.float32, seed=97)
    leaf = x.clone().requires_grad_(True)
    logits = leaf * 1.0
    other = (logits * logits).sum()
    r = L().policy_loss(logits, tok, old, adv, weights=w)
    assert not r.loss.requires_grad and not r.logprobs.requires_grad and not r.grad.requires_grad
    with pytest.raises(RuntimeError):
        r.loss.backward()
    torch.autograd.backward([logits, other], [r.grad, None])
    want = r.grad.double() + 2 * x.double()
    assert ((leaf.grad.double() - want).abs() <= 2 * U * (r.grad.double().abs() + 2 * x.double().abs())).all()
