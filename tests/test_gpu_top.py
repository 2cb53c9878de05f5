"""The best tokens of a row and the steps of beam search over them, against the
definitions in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32 relative to the value.  A
log-probability is (x - m) / T - log S: its first part is exact up to 64-bit
rounding, and S, a sum of terms exp((x - m) / T), is good to
  REL = (4 + 6 log V + V / 256 + 21) u
relative: a term's exponent is rounded three times (3 u |x - m| / T on the term,
weighted with the terms below 2 log V), its exponential is good to 4 u, and at
most V / 256 + 16 terms and 5 more levels are added in fp32.  The result is
rounded to fp32: u |lp|.  Tokens and parents have to be equal wherever no two
different beams' candidates lie within twice that of one another."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float("inf")


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def top(x, k, T=1.0, **kw):
    from qwen600_engine_b200 import losses
    return losses.top_logprobs(x, k, temperature=T, **kw)


def select(*a, **kw):
    from qwen600_engine_b200 import beams
    return beams.beam_select(*a, **kw)


def rel_sum(V):
    return (4 + 6 * math.log(max(V, 2)) + V / 256 + 21) * U


def rows_of(N, V, dtype, seed, kind="mixed", pad=0, shift=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn((N, V), generator=g, device="cuda") * (0.5 + 4 * torch.rand((N, 1), generator=g, device="cuda"))
    x += 20 * torch.rand((N, 1), generator=g, device="cuda") - 10
    if kind == "equal":
        x[:] = 3.0
    if kind == "few values":
        x = (x / 4).round()
    if kind == "rising":
        x = torch.arange(V, device="cuda").float().expand(N, V) / 64
    if kind == "falling":
        x = -torch.arange(V, device="cuda").float().expand(N, V) / 64
    if kind == "block":  # everything that counts lies in one stretch
        x[:, V // 3:V // 3 + 600] += 200
    if kind == "masked":
        x[torch.rand((N, V), generator=g, device="cuda") < 0.97] = -INF
    if kind == "lowest":
        x[torch.rand((N, V), generator=g, device="cuda") < 0.97] = torch.finfo(dtype).min
    buf = torch.full((N * (V + pad) + shift,), 99.0, dtype=dtype, device="cuda")
    view = buf[shift:].view(N, V + pad)[:, :V]
    view.copy_(x)
    return view


def exact_logprobs(x, T=1.0):
    d = x.double()
    return (d - d.amax(1, keepdim=True)) / T - ((d - d.amax(1, keepdim=True)) / T).exp().sum(1, keepdim=True).log()


def exact_top(x, k, T=1.0):
    value, at = x.double().sort(dim=1, descending=True, stable=True)
    value, at = value[:, :k], at[:, :k]
    if k > x.shape[1]:
        more = k - x.shape[1]
        value = torch.nn.functional.pad(value, (0, more), value=-INF)
        at = torch.nn.functional.pad(at, (0, more), value=0)
    lp = exact_logprobs(x, T).gather(1, at)
    none = value == -INF
    return torch.where(none, torch.full_like(lp, -INF), lp), torch.where(none, torch.full_like(at, -1), at).int()


def check_top(x, k, T=1.0):
    r = top(x, k, T)
    lp, tok = exact_top(x, k, T)
    assert r.logprobs.shape == r.tokens.shape == (x.shape[0], k)
    assert r.logprobs.dtype == torch.float32 and r.tokens.dtype == torch.int32
    assert torch.equal(r.tokens, tok)
    none = tok < 0
    assert (r.logprobs[none] == -INF).all()
    off = (r.logprobs.double() - lp).abs()[~none]
    assert (off <= rel_sum(x.shape[1]) + U * lp.abs()[~none] + 1e-12).all(), float(off.max())
    return r


SHAPES = [(1, 1, 1), (1, 2, 2), (3, 7, 4), (5, 33, 33), (2, 1000, 20), (4, 1003, 256), (2, 8192, 1), (3, 50021, 250), (3, 151936, 64),
          (1, 262144, 17), (37, 4099, 5), (300, 2049, 20)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V,k", SHAPES)
def test_top(dtype, N, V, k):
    check_top(rows_of(N, V, dtype, seed=N + V + k), k, T=0.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["equal", "few values", "rising", "falling", "block", "masked", "lowest"])
@pytest.mark.parametrize("V,k", [(3001, 1), (3001, 40), (70007, 200), (70007, 256)])
def test_top_where_order_is_hard(dtype, kind, V, k):
    check_top(rows_of(3, V, dtype, seed=V + k, kind=kind), k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,shift", [(1, 0), (0, 1), (3, 5), (8, 8), (13, 7)])
def test_top_of_strided_rows(dtype, pad, shift):
    check_top(rows_of(5, 6001, dtype, seed=pad, pad=pad, shift=shift), 33)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_lists_no_masked_token(dtype):
    x = rows_of(6, 5003, dtype, seed=3)
    x[0] = -INF
    x[1, 4:] = -INF
    x[2, :-2] = -INF
    x[3] = -INF
    x[3, 2500] = torch.finfo(dtype).min
    x[4] = torch.finfo(dtype).min
    r = top(x, 9)
    assert (r.tokens[0] == -1).all() and (r.logprobs[0] == -INF).all()
    assert r.tokens[1].sort().values.tolist() == [-1] * 5 + [0, 1, 2, 3]
    assert sorted(r.tokens[2].tolist()) == [-1] * 7 + [5001, 5002]
    assert r.tokens[3].tolist() == [2500] + [-1] * 8 and float(r.logprobs[3, 0]) == 0.0
    assert r.tokens[4].tolist() == list(range(9))
    check_top(x[1:], 9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), INF])
@pytest.mark.parametrize("at", [0, 1, 2517, 5002])
def test_top_of_rows_with_nan_or_inf(dtype, bad, at):
    x = rows_of(3, 5003, dtype, seed=5)
    x[1, at] = bad
    r = top(x, 6)
    assert (r.tokens[1] == -1).all() and r.logprobs[1].isnan().all()
    x[1] = -INF
    x[1, at] = bad
    r = top(x, 6)
    assert (r.tokens[1] == -1).all() and r.logprobs[1].isnan().all()
    check_top(x[::2], 6)


def test_top_equal_zeros_of_either_sign_by_token():
    x = torch.zeros((1, 4000), device="cuda")
    x[0, ::2] = -0.0
    assert top(x, 5).tokens.tolist() == [[0, 1, 2, 3, 4]]


@pytest.mark.parametrize("T", [1e-6, 0.01, 50.0, 1e6])
def test_top_at_any_temperature(T):
    x = rows_of(3, 9001, torch.float32, seed=8)
    r = top(x, 12, T)
    lp, tok = exact_top(x, 12, T)
    assert torch.equal(r.tokens, tok)
    total = exact_logprobs(x, T).amax(1, keepdim=True).neg().exp()  # the sum of the terms
    assert ((r.logprobs.double() - lp).abs() <= rel_sum(9001) * total.log().clamp(min=1) + U * lp.abs() + 1e-12).all()


def test_top_of_many_rows_and_no_row():
    check_top(rows_of(1500, 20011, torch.bfloat16, seed=1), 20)
    r = top(torch.empty((0, 100), device="cuda"), 3)
    assert r.logprobs.shape == (0, 3) and r.tokens.shape == (0, 3)


def test_top_agrees_with_the_score_of_the_token():
    """The log-probability of the best token is that of token_logprobs."""
    from qwen600_engine_b200 import losses
    x = rows_of(64, 151936, torch.bfloat16, seed=2)
    r = top(x, 3)
    for i in range(3):
        lp = losses.token_logprobs(x, r.tokens[:, i].contiguous()).logprobs
        assert ((lp.double() - r.logprobs[:, i].double()).abs() <= 2 * rel_sum(151936) + 2 * U * lp.abs()).all()


# ------------------------------------------------------------------ beam search
def exact_beams(x, scores, n, finished, eos, pad, T, keep):
    """Per entry [(score, beam, token)] in order, and the outputs' places."""
    batch, beams = scores.shape
    lp = exact_logprobs(x, T)
    out = []
    for b in range(batch):
        c = []
        for i in range(beams):
            s = float(scores[b, i])
            if s == -INF:
                continue
            if finished is not None and bool(finished[b, i]):
                c.append((s, i, pad, 0))
                continue
            row = lp[b * beams + i] + scores[b, i].double()
            value, at = row.sort(descending=True, stable=True)
            c += [(v, i, t, t) for v, t in zip(value[:n + 1].tolist(), at[:n + 1].tolist()) if v > -INF]
        c.sort(key=lambda e: (-e[0], e[1], e[3]))
        out.append([e[:3] for e in c])
    return out


def check_beams(x, scores, n=None, finished=None, eos=-1, pad=None, T=1.0, keep=False):
    batch, beams = scores.shape
    r = select(x, scores, n=n, finished=finished, eos_token=eos, pad_token=pad, temperature=T, keep_slots=keep)
    n, pad = n or beams, eos if pad is None else pad
    assert r.scores.shape == r.parents.shape == r.tokens.shape == r.finished.shape == (batch, n)
    assert r.finished.dtype == torch.bool and r.parents.dtype == r.tokens.dtype == torch.int32
    tol = 2 * rel_sum(x.shape[1])
    for b, ref in enumerate(exact_beams(x, scores, n, finished, eos, pad, T, keep)):
        got = list(zip(r.scores[b].tolist(), r.parents[b].tolist(), r.tokens[b].tolist(), r.finished[b].tolist()))
        if keep:
            by_parent = {}
            for g in got:
                by_parent.setdefault(g[1], []).append(g)
            for p, children in by_parent.items():
                if p >= 0:
                    assert got[p][1] == p and got[p][0] == max(c[0] for c in children), "the best child stays in its parent's place"
            others = [g for i, g in enumerate(got) if g[1] != i]
            assert [g[0] for g in others] == sorted((g[0] for g in others), reverse=True)
            got.sort(key=lambda g: (-g[0], g[1] if g[1] >= 0 else beams))
        assert [g[0] for g in got] == sorted((g[0] for g in got), reverse=True)
        live = [g for g in got if g[1] >= 0]
        assert len(live) == min(n, len(ref)) and all(g == (-INF, -1, -1, True) for g in got[len(live):])
        assert len({g[1:3] for g in live}) == len(live), "a continuation twice"
        near = any(ref[i][0] - ref[i + 1][0] <= 2 * (tol + U * abs(ref[i][0])) and ref[i][1] != ref[i + 1][1]
                   for i in range(min(n, len(ref) - 1)))
        score_of = {e[1:]: e[0] for e in ref}
        for g, e in zip(live, ref):
            assert abs(g[0] - e[0]) <= tol + U * abs(e[0]) + 1e-12
            if near:
                assert abs(score_of[g[1:3]] - g[0]) <= tol + U * abs(g[0]) + 1e-12
            elif not keep:
                assert g[1:3] == e[1:]
            assert g[3] == ((eos >= 0 and g[2] == eos) or (finished is not None and bool(finished[b, g[1]])))
        if keep and not near:
            assert {g[1:3] for g in live} == {e[1:] for e in ref[:n]}
    return r


def scores_of(batch, beams, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return -3 * torch.rand((batch, beams), generator=g, device="cuda") - 20 * torch.rand((batch, 1), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,beams,V,n", [(1, 1, 1, 1), (1, 1, 1000, 3), (1, 4, 151936, 8), (3, 2, 7, 14), (2, 3, 5, 20), (5, 5, 1003, 10),
                                             (2, 64, 3001, 128), (1, 64, 50021, 256), (33, 3, 2049, 3), (4, 8, 262144, 8)])
def test_beams(dtype, batch, beams, V, n):
    check_beams(rows_of(batch * beams, V, dtype, seed=batch + V), scores_of(batch, beams, n), n, T=0.9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["mixed", "few values", "masked", "block"])
@pytest.mark.parametrize("beams,V,n", [(2, 1000, 200), (3, 3001, 256), (1, 6000, 129), (5, 600, 256)])
def test_long_lists_of_few_parts(dtype, kind, beams, V, n):
    x = rows_of(2 * beams, V, dtype, seed=V + n, kind=kind, pad=3)
    check_beams(x, scores_of(2, beams, n), n)
    check_top(x, n)


@pytest.mark.parametrize("T", [1e-3, 0.05, 40.0])
@pytest.mark.parametrize("keep", [False, True])
def test_beams_at_any_temperature(T, keep):
    """Sums of up to 2^24 and more: the 64-bit sums' spacing is far below an fp32 logit's."""
    x = rows_of(15, 5003, torch.float32, seed=16)
    r = select(x, scores_of(3, 5, 8), n=5, temperature=T, keep_slots=keep)
    for b, ref in enumerate(exact_beams(x, scores_of(3, 5, 8), 5, None, -1, -1, T, keep)):
        got = sorted(zip(r.scores[b].tolist(), r.parents[b].tolist(), r.tokens[b].tolist()), key=lambda g: (-g[0], g[1], g[2]))
        for g, e in zip(got, ref):
            total = max(1.0, 5003 ** 0.5 / T)
            assert abs(g[0] - e[0]) <= rel_sum(5003) * total + 2 * U * abs(e[0])
        assert {g[1:] for g in got} == {e[1:] for e in ref[:5]}


@pytest.mark.parametrize("kind", ["few values", "equal", "masked", "lowest", "block", "rising"])
@pytest.mark.parametrize("beams,n", [(1, 200), (6, 12), (16, 256)])
def test_beams_where_order_is_hard(kind, beams, n):
    """Rows alike but for their scores, so that equal sums are equal bits."""
    x = rows_of(1, 8192, torch.bfloat16, seed=17, kind=kind).repeat(3 * beams, 1)
    scores = -torch.arange(3 * beams, device="cuda").view(3, beams).float() % 7
    check_beams(x, scores, n)
    check_beams(x, torch.zeros_like(scores), n)
    check_beams(x, scores - 2.0 ** 22, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("share", [0.0, 0.4, 1.0])
def test_finished_beams(dtype, keep, share):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(share * 10))
    x = rows_of(30, 4001, dtype, seed=4)
    finished = torch.rand((5, 6), generator=g, device="cuda") < share
    x[finished.view(-1)] = float("nan")  # not read
    eos = int(x.nan_to_num(-1e4)[0].argmax())
    check_beams(x, scores_of(5, 6, 6), None if keep else 9, finished, eos=eos, keep=keep)
    check_beams(x, scores_of(5, 6, 7), 6, finished, eos=eos, pad=-7, keep=keep)


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("beams", [2, 5, 16, 64])
def test_search_begins_with_one_beam(keep, beams):
    """The others' score is -inf: their rows, all alike, offer nothing."""
    x = rows_of(3, 20011, torch.bfloat16, seed=beams).repeat_interleave(beams, 0)
    scores = torch.full((3, beams), -INF, device="cuda")
    scores[:, 0] = 0
    r = check_beams(x, scores, beams, keep=keep)
    assert (r.parents == 0).all()


def test_equal_scores_go_by_beam_then_token():
    x = torch.zeros((4, 4096), device="cuda")
    x[:, 100:103] = 5.0
    r = select(x, torch.zeros((1, 4), device="cuda"), n=10)
    assert r.parents.tolist() == [[0, 0, 0, 1, 1, 1, 2, 2, 2, 3]]
    assert r.tokens.tolist() == [[100, 101, 102] * 3 + [100]]
    r = select(torch.zeros((8, 2048), device="cuda", dtype=torch.bfloat16), torch.zeros((2, 4), device="cuda"), n=200)
    assert (r.parents == 0).all() and torch.equal(r.tokens.cpu(), torch.arange(200, dtype=torch.int32).expand(2, 200))


@pytest.mark.parametrize("keep", [False, True])
def test_masked_beams(keep):
    x = rows_of(12, 3001, torch.float32, seed=9)
    x[0] = -INF        # a beam without continuations
    x[3:6] = -INF      # an entry without any
    x[6:9, 5:] = -INF
    x[9:, 1:] = -INF   # one token a beam
    check_beams(x, scores_of(4, 3, 1), 3, keep=keep)
    if not keep:
        check_beams(x, scores_of(4, 3, 1), 20)


@pytest.mark.parametrize("bad", [float("nan"), INF])
def test_entries_with_nan(bad):
    x = rows_of(12, 3001, torch.bfloat16, seed=10)
    scores = scores_of(4, 3, 2)
    clean = select(x, scores, n=5)
    x[4, 2999] = bad
    scores[2, 1] = bad
    finished = torch.zeros((4, 3), dtype=torch.bool, device="cuda")
    finished[2, 1] = True
    for f in (None, finished):
        r = select(x, scores, n=5, finished=f)
        for b in (1, 2):
            assert r.scores[b].isnan().all() and (r.parents[b] == -1).all() and (r.tokens[b] == -1).all()
        for b in (0, 3):
            assert all(torch.equal(p[b], q[b]) for p, q in zip(r, clean))
    finished[1, 1] = True  # a finished beam's logits are not read
    assert not select(x, scores, n=5, finished=finished).scores[1].isnan().any()


@pytest.mark.parametrize("keep", [False, True])
def test_beams_far_from_zero(keep):
    """Scores so low that fp32 cannot tell candidates apart; the lowest of all."""
    x = rows_of(12, 3001, torch.float32, seed=18)
    scores = torch.full((3, 4), -3e6, device="cuda")
    scores[1] = torch.finfo(torch.float32).min
    scores[2] = torch.tensor([0.0, -1e30, 0.5, 1e30])
    r = select(x, scores, n=4, keep_slots=keep)
    ref = exact_beams(x, scores, 4, None, -1, -1, 1.0, keep)
    assert {(p, t) for p, t in zip(r.parents[0].tolist(), r.tokens[0].tolist())} == {e[1:] for e in ref[0][:4]}
    assert (r.scores[1] == torch.finfo(torch.float32).min).all() and (r.tokens[1] >= 0).all()
    assert (r.parents[2] == 3).sum() == 4 and (r.scores[2] == 1e30).all()


@pytest.mark.parametrize("keep", [False, True])
def test_beams_of_strided_rows(keep):
    check_beams(rows_of(15, 6001, torch.bfloat16, seed=12, pad=7, shift=3), scores_of(3, 5, 3), 5, keep=keep)


def test_no_entry():
    r = select(torch.empty((0, 50), device="cuda"), torch.empty((0, 4), device="cuda"), n=6)
    assert r.scores.shape == r.finished.shape == (0, 6)


def test_same_bits_on_any_stream_and_in_a_graph():
    x, scores = rows_of(64, 30011, torch.bfloat16, seed=14), scores_of(8, 8, 4)
    one, two = select(x, scores, n=16), top(x, 40)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a, b = select(x, scores, n=16, stream=side), top(x, 40, stream=side)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(one + two, a + b))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c, d = select(x, scores, n=16), top(x, 40)
    held = x.clone()
    x.copy_(rows_of(64, 30011, torch.bfloat16, seed=15))
    g.replay()
    fresh = select(x, scores, n=16) + top(x, 40)
    assert all(torch.equal(p, q) for p, q in zip(c + d, fresh))
    x.copy_(held)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(c + d, one + two))
