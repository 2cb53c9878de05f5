"""Distillation from a teacher's lists against the formula in 64 bits.

Tolerances.  u = 2^-24.  S_r, the sum of the unlisted terms against their own
maximum, is good to REL = (4 + 6 log V + V / 256 + 21) u relative (terms: three
rounded steps of the exponent and an exponential of 4 u; at most V / 256 + 21
additions in fp32); the listed sum and everything else are 64-bit.  So
log S = log(S_l + S_r) is off by REL p_r and log p_r by REL (1 + p_r):
  row loss   (Q p_r + r (1 + p_r)) REL, and its rounding u |l|
  unlisted   w / T p_j (Q REL (1 + p_r) + r / p_r REL) for the coefficient, and
             (3 |x - m_r| / T + 5) u of the value for the term and the product
  listed     w / T Q p_e p_r REL
and the output's rounding, eps / 2 of the value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = 2.0 ** -126
INF = float("inf")


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def distill(*a, **kw):
    from qwen600_engine_b200 import losses
    return losses.distill_loss(*a, **kw)


def rel_sum(V):
    return (4 + 6 * math.log(max(V, 2)) + V / 256 + 21) * U


def case_of(N, V, k, dtype, seed, T=1.0, pad=0, shift=0, spread=1.0):
    """Logits, and lists of a teacher whose logits are near them."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn((N, V), generator=g, device="cuda") * (0.5 + 4 * torch.rand((N, 1), generator=g, device="cuda"))
    x += 20 * torch.rand((N, 1), generator=g, device="cuda") - 10
    buf = torch.full((N * (V + pad) + shift,), 99.0, dtype=dtype, device="cuda")
    view = buf[shift:].view(N, V + pad)[:, :V]
    view.copy_(x)
    teacher = torch.log_softmax((x + spread * torch.randn((N, V), generator=g, device="cuda")).double() / T, 1)
    lps, tok = teacher.topk(min(k, V), 1)
    if k > V:
        lps = torch.nn.functional.pad(lps, (0, k - V), value=-INF)
        tok = torch.nn.functional.pad(tok, (0, k - V), value=-1)
    return view, tok.int().contiguous(), lps.float().contiguous(), g


def exact(x, tok, lps, w=None, T=1.0, rest=True):
    """(row losses, gradient, tolerances of both) in 64 bits, the gradient by the formula."""
    N, V = x.shape
    l, tol_l = torch.zeros(N, dtype=torch.float64, device=x.device), torch.zeros(N, dtype=torch.float64, device=x.device)
    grad, tol = torch.zeros((N, V), dtype=torch.float64, device=x.device), torch.zeros((N, V), dtype=torch.float64, device=x.device)
    w = torch.full((N,), 1.0 / N, dtype=torch.float64, device=x.device) if w is None else w.double()
    for i in range(N):
        seen, at, given = set(), [], []
        for t, v in zip(tok[i].tolist(), lps[i].tolist()):
            if 0 <= t < V and t not in seen:
                seen.add(t)
                at.append(t)
                given.append(v)
        if float(w[i]) == 0.0 or not at or (not rest and all(v == -INF for v in given)):
            continue
        at, given = torch.tensor(at, device=x.device), torch.tensor(given, dtype=torch.float64, device=x.device)
        y = x[i].double() / T
        lp = torch.log_softmax(y, 0)
        p = lp.exp()
        out = y.clone()
        out[at] = -INF
        unlisted = torch.logsumexp(out, 0) - torch.logsumexp(y, 0)  # log p_r
        p_r = float(unlisted.exp())
        if not rest:
            given = given - torch.logsumexp(given, 0)
        q = given.exp()
        r = max(0.0, 1.0 - float(q.sum())) if rest and float(unlisted) > -INF else 0.0
        mass = float(q.sum()) + r if rest else 1.0
        l[i] = torch.where(q > 0, q * (given - lp[at]), torch.zeros_like(q)).sum()
        if r > 0:
            l[i] += r * (math.log(r) - unlisted)
        c = w[i] / T
        inside = (out - out.amax()).exp() / (out - out.amax()).exp().sum() if p_r > 0 or float(unlisted) > -INF else torch.zeros_like(p)
        row = c * (mass * p - r * inside)
        row[at] = c * (mass * p[at] - q)
        R = rel_sum(V)
        t = c.abs() * (mass * p * R * (1 + p_r) + r * inside * R) + row.abs() * (3 * (out.amax() - out).nan_to_num(nan=100).clamp(max=100) + 5) * U + c.abs() * TINY
        t[at] = c.abs() * mass * p[at] * p_r * R + row[at].abs() * U
        grad[i], tol[i] = row, t + 1e-300
        tol_l[i] = (mass * p_r + r * (1 + p_r)) * R + U * l[i].abs() + 1e-12
    return l, grad, tol_l, tol, (w * l).sum(), (w.abs() * tol_l).sum() + U * (w * l).sum().abs()


def check(x, tok, lps, w=None, T=1.0, rest=True, **kw):
    r = distill(x, tok, lps, weights=w, temperature=T, rest=rest, **kw)
    l, grad, tol_l, tol, loss, tol_loss = exact(x, tok, lps, w, T, rest)
    assert r.loss.dtype == r.row_losses.dtype == torch.float32 and r.grad.dtype == x.dtype and r.grad.shape == x.shape
    finite = l.isfinite()
    assert torch.equal(r.row_losses[~finite].double(), l[~finite])
    off = (r.row_losses.double() - l).abs()[finite]
    assert (off <= tol_l[finite]).all(), float((off / tol_l[finite].clamp(min=1e-300)).max())
    if finite.all():
        assert abs(float(r.loss) - float(loss)) <= float(tol_loss)
    h = torch.finfo(x.dtype).eps / 2
    lim = tol * (1 + h) + h * grad.abs() + torch.finfo(x.dtype).smallest_normal * 2 * h
    off = (r.grad.double() - grad).abs()
    assert (off <= lim).all(), float((off / lim).max())
    return r


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (1, 2, 1), (2, 3, 5), (3, 7, 4), (4, 33, 20), (2, 1000, 1), (4, 1003, 256), (3, 8192, 64),
                                   (3, 50021, 129), (2, 151936, 64), (1, 262144, 20), (40, 2049, 20), (200, 700, 8)])
def test_loss_and_gradient(dtype, rest, N, V, k):
    x, tok, lps, g = case_of(N, V, k, dtype, seed=N + V + k)
    check(x, tok, lps, rest=rest)


@pytest.mark.parametrize("T", [0.5, 2.0, 8.0])
@pytest.mark.parametrize("rest", [True, False])
def test_temperature_and_weights(T, rest):
    x, tok, lps, g = case_of(12, 4099, 30, torch.bfloat16, seed=7, T=T)
    w = torch.randn((12,), generator=g, device="cuda")
    w[3] = w[8] = 0
    x[3], lps[8] = float("nan"), float("nan")  # rows that are left out are not read
    x2, lps2 = x.clone(), lps.clone()
    x2[3], lps2[8] = 0, 0
    r = distill(x, tok, lps, weights=w, temperature=T, rest=rest)
    s = check(x2, tok, lps2, w, T, rest)
    assert all(torch.equal(p, q) for p, q in zip(r, s))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,shift", [(1, 0), (0, 3), (8, 8), (11, 5)])
def test_strided_rows(dtype, pad, shift):
    x, tok, lps, g = case_of(5, 6001, 17, dtype, seed=pad, pad=pad, shift=shift)
    tok[:, 0], tok[:, 1], tok[:, 2], tok[:, 3] = 0, 6000, 1, 5999  # tokens outside the vectors
    check(x, tok, lps)
    out = torch.full((5, 6001 + pad), 55.0, dtype=dtype, device="cuda")[:, :6001]
    r = distill(x, tok, lps, out=out)
    assert r.grad.data_ptr() == out.data_ptr() and torch.equal(out, distill(x, tok, lps).grad)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_in_place_of_the_logits(dtype):
    x, tok, lps, g = case_of(9, 30011, 40, dtype, seed=1)
    want = distill(x, tok, lps)
    got = distill(x, tok, lps, out=x)
    assert got.grad.data_ptr() == x.data_ptr() and torch.equal(x, want.grad) and torch.equal(got.loss, want.loss)


def test_lists_with_gaps_and_repeats():
    x, tok, lps, g = case_of(6, 3001, 16, torch.float32, seed=2)
    tok[0, 3:] = -1
    tok[1] = -1                       # no entry: nothing
    tok[2, 5] = tok[2, 0]             # again, with another probability: counts where it stands first
    tok[2, 9:] = tok[2, 1]
    tok[3, 4] = 3001
    tok[4, 0], lps[4, 0] = 2 ** 31 - 1, float("nan")
    lps[5, 3:] = -INF
    for rest in (True, False):
        r = check(x, tok, lps, rest=rest)
        assert float(r.row_losses[1]) == 0 and not r.grad[1].any()
    lps[5] = -INF                     # the teacher gives the list nothing
    assert float(check(x, tok, lps, rest=False).row_losses[5]) == 0
    assert float(check(x, tok, lps, rest=True).row_losses[5]) > 0


def test_same_token_all_over():
    x, tok, lps, g = case_of(3, 5000, 256, torch.bfloat16, seed=3)
    tok[:] = tok[:, :1].clone()
    check(x, tok, lps)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_logits(dtype):
    x, tok, lps, g = case_of(6, 4001, 12, dtype, seed=4)
    lowest = torch.finfo(dtype).min
    keep = x.clone()
    x[0], x[1] = -INF, lowest
    for i in (0, 1):                  # everything but the list masked
        x[i].scatter_(0, tok[i].long(), keep[i].gather(0, tok[i].long()))
    x[2, tok[2, 3]] = -INF            # a listed one masked: +inf, with a gradient that is not
    x[3].scatter_(0, tok[3].long(), -INF)
    x[4, 200:] = -1e30
    lps[5, 2] = -INF
    x[5, tok[5, 2]] = -INF            # masked, and nothing to the teacher
    r = check(x, tok, lps)
    assert r.row_losses[2] == INF and r.row_losses[3] == INF and r.loss == INF and r.row_losses[0].isfinite()
    assert r.grad.isfinite().all()
    check(x, tok, lps, rest=False)


@pytest.mark.parametrize("bad", ["nan", "inf", "all -inf"])
@pytest.mark.parametrize("place", ["listed", "unlisted", "first", "last"])
def test_rows_without_a_distribution(bad, place):
    x, tok, lps, g = case_of(4, 5003, 10, torch.bfloat16, seed=5)
    tok[1, 9], tok[1, 8] = 2500, 2501
    at = {"listed": 2500, "unlisted": 2502, "first": 0, "last": 5002}[place]
    clean = distill(x, tok, lps)
    if bad == "all -inf":
        x[1] = -INF
    else:
        x[1, at] = float(bad)
    r = distill(x, tok, lps)
    assert r.loss.isnan() and r.row_losses[1].isnan() and r.grad[1].isnan().all()
    for i in (0, 2, 3):
        assert torch.equal(r.grad[i], clean.grad[i]) and torch.equal(r.row_losses[i], clean.row_losses[i])


def test_teacher_with_nan():
    x, tok, lps, g = case_of(3, 5003, 10, torch.float32, seed=6)
    lps[1, 4] = float("nan")
    for rest in (True, False):
        r = distill(x, tok, lps, rest=rest)
        assert r.loss.isnan() and r.grad[1].isnan().all() and r.grad[::2].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_peaked_rows_keep_the_rest(dtype):
    """What the list leaves is 1e-30 of the row: its logarithm still counts."""
    x, tok, lps, g = case_of(4, 20011, 8, dtype, seed=8)
    x.scatter_(1, tok.long(), 70.0)
    r = check(x, tok, lps)
    assert r.row_losses.isfinite().all()


def test_rest_nearer_than_32_bits_to_nothing():
    """Listed probabilities that add up to a little more than 1, and a whole vocabulary listed."""
    x, tok, lps, g = case_of(3, 40, 40, torch.float32, seed=9)
    check(x, tok, lps)
    x, tok, lps, g = case_of(3, 500, 40, torch.float32, seed=9)
    check(x, tok, lps + 1e-3)


def test_shifted_lists_without_rest():
    x, tok, lps, g = case_of(5, 3001, 20, torch.float32, seed=10)
    a, b = distill(x, tok, lps, rest=False), distill(x, tok, lps + 64.0, rest=False)
    assert torch.allclose(a.grad, b.grad, rtol=0, atol=1e-5) and abs(float(a.loss) - float(b.loss)) < 5e-5
    check(x, tok, lps + 64.0, rest=False)


@pytest.mark.parametrize("rest", [True, False])
def test_gradient_against_differences(rest):
    """(l(x + h e) - l(x - h e)) / 2 h in 64 bits: error h^2 / 6 times a third derivative below 1."""
    x, tok, lps, g = case_of(2, 60, 12, torch.float32, seed=11, T=1.3)
    r = distill(x, tok, lps, temperature=1.3, rest=rest)
    h = 1e-4
    for i in range(2):
        for j in range(60):
            d = x.double()
            d[i, j] += h
            up = exact(d, tok, lps, T=1.3, rest=rest)[4]
            d[i, j] -= 2 * h
            assert abs(float((up - exact(d, tok, lps, T=1.3, rest=rest)[4]) / (2 * h)) - float(r.grad[i, j])) <= h * h + 4e-6


def test_loss_alone_and_no_row():
    x, tok, lps, g = case_of(7, 9001, 11, torch.bfloat16, seed=12)
    a, b = distill(x, tok, lps), distill(x, tok, lps, grad=False)
    assert b.grad is None and torch.equal(a.loss, b.loss) and torch.equal(a.row_losses, b.row_losses)
    r = distill(x[:0], tok[:0], lps[:0])
    assert float(r.loss) == 0 and r.grad.shape == (0, 9001)


def test_gradient_reaches_the_weights():
    """logits.backward(grad) beside another loss: the sum of both gradients."""
    h = torch.randn((6, 32), device="cuda")
    weight = torch.randn((900, 32), device="cuda", requires_grad=True)
    x, tok, lps, g = case_of(6, 900, 10, torch.float32, seed=13)
    logits = h @ weight.t()
    r = distill(logits.detach(), tok, lps)
    other = weight.square().sum()
    torch.autograd.backward([logits, other], [r.grad, None])
    want = r.grad.double().t() @ h.double() + 2 * weight.detach().double()
    assert torch.allclose(weight.grad.double(), want, rtol=1e-5, atol=1e-5)


def test_large_batches_and_graphs():
    x, tok, lps, g = case_of(600, 20011, 64, torch.bfloat16, seed=14)
    w = (torch.rand((600,), generator=g, device="cuda") < 0.8).float()
    check(x, tok, lps, w)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(x)
    with torch.cuda.graph(graph):
        r = distill(x, tok, lps, weights=w, out=out)
    graph.replay()
    again = distill(x, tok, lps, weights=w)
    assert torch.equal(r.grad, again.grad) and torch.equal(r.loss, again.loss)
    x.copy_(x.flip(0))
    graph.replay()
    again = distill(x, tok, lps, weights=w)
    assert torch.equal(r.grad, again.grad) and torch.equal(r.loss, again.loss)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    s = distill(x, tok, lps, weights=w, stream=side)
    side.synchronize()
    assert torch.equal(s.grad, again.grad)


def test_a_teacher_that_lists_everything_is_the_whole_divergence():
    """Teacher and student from two heads; k = vocabulary: the full divergence and its gradient."""
    from qwen600_engine_b200 import losses
    g = torch.Generator(device="cuda")
    g.manual_seed(15)
    teacher, student = torch.randn((30, 250), generator=g, device="cuda"), torch.randn((30, 250), generator=g, device="cuda")
    t = losses.top_logprobs(teacher, 250, temperature=2.0)
    r = distill(student, t.tokens, t.logprobs, temperature=2.0)
    s = student.double().requires_grad_(True)
    kl = torch.nn.functional.kl_div(torch.log_softmax(s / 2, 1), torch.log_softmax(teacher.double() / 2, 1), log_target=True, reduction="batchmean")
    kl.backward()
    assert abs(float(r.loss) - float(kl)) <= rel_sum(250) + 250 * U
    assert (r.grad.double() - s.grad).abs().max() <= (rel_sum(250) + 250 * U) / 60
