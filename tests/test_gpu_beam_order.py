"""Equal scores of a search go by beam, then by token, also at the border of what
is chosen.

An entry's rows are alike, bit for bit and in their alignment, so that their sums
of exponentials are the same bits, and beams with the same score so far give equal
tokens equal bits.  Among such beams the order is that of the logits, then of the
beams, then of the tokens: different logits differ by far more than a 64-bit sum's
spacing.  Beams whose scores so far differ keep that order among those of the same
score (between them rounding decides)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def row_of(V, dtype, kind, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(V, generator=g, device="cuda") * 3
    rand = torch.rand(V, generator=g, device="cuda")
    if kind == "equal":
        x[:] = 3.0
    if kind == "few values":
        x = x.round()
    if kind == "two values":
        x = (rand < 0.02).float()
    if kind == "masked":
        x = torch.where(rand < 0.97, -INF, x.round())
    if kind == "lowest":
        x[rand < 0.97] = torch.finfo(dtype).min
    if kind == "all lowest":
        x[:] = torch.finfo(dtype).min
    if kind == "zeros":
        x = torch.where(rand < 0.5, -0.0, 0.0)
    if kind == "block":  # equal ones behind one another, across a unit's border
        x = x.clamp(max=4)
        x[V // 3:V // 3 + 700] = 9.0
    if kind == "last":
        x = x.clamp(max=4)
        x[-7:] = 9.0
    return x.to(dtype)


KINDS = ["few values", "equal", "two values", "masked", "lowest", "all lowest", "zeros", "block", "last"]


def expected(row, beams, count):
    """The first `count` (beam, token) of beams alike."""
    value, at = (row.double() + 0.0).sort(descending=True, stable=True)
    value, at = value.tolist(), at.tolist()
    out, i = [], 0
    while i < len(at) and len(out) < count and value[i] > -INF:
        j = i
        while j < len(at) and value[j] == value[i] and j - i < count:
            j += 1
        for b in beams:
            out += [(b, t) for t in at[i:j]]
            if len(out) >= count:
                break
        while j < len(at) and value[j] == value[i]:
            j += 1
        i = j
    return out[:count]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("beams,V,n", [(1, 1000, 1), (2, 4096, 5), (4, 50000, 8), (6, 8192, 12), (16, 8192, 256), (3, 152, 256), (64, 3000, 100)])
@pytest.mark.parametrize("base", [0.0, -17.25, -2.0 ** 22])
def test_equal_beams(dtype, kind, beams, V, n, base):
    from qwen600_engine_b200.beams import beam_select
    row = row_of(V, dtype, kind, seed=V + n)
    x = row.repeat(2 * beams, 1)
    r = beam_select(x, torch.full((2, beams), base, device="cuda"), n=n)
    want = expected(row, range(beams), n)
    want += [(-1, -1)] * (n - len(want))
    for b in range(2):
        assert list(zip(r.parents[b].tolist(), r.tokens[b].tolist())) == want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("beams,V,n", [(4, 50000, 8), (6, 8192, 12), (16, 8192, 256), (64, 3000, 100)])
@pytest.mark.parametrize("ended", [False, True])
def test_beams_of_several_scores(dtype, kind, beams, V, n, ended):
    """Whole steps apart, like many logits; with an ended beam between the others."""
    from qwen600_engine_b200.beams import beam_select
    row = row_of(V, dtype, kind, seed=V + n)
    scores = -(torch.arange(beams, device="cuda") % 3).float().expand(2, beams).contiguous()
    finished = torch.zeros((2, beams), dtype=torch.bool, device="cuda")
    finished[:, 1] = ended
    r = beam_select(row.repeat(2 * beams, 1), scores, n=n, finished=finished, eos_token=0, pad_token=-9)
    for b in range(2):
        got = list(zip(r.parents[b].tolist(), r.tokens[b].tolist()))
        live = [g for g in got if g[0] >= 0]
        assert len(set(live)) == len(live) and (len(live) == n or kind == "masked")
        assert (1, -9) in live if ended else all(t >= 0 for _, t in live)
        for k in range(3):
            alike = [i for i in range(k, beams, 3) if not (ended and i == 1)]
            mine = [g for g in live if g[0] in alike]
            assert mine == expected(row, alike, len(mine))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("beams,V", [(4, 50000), (16, 8192), (64, 3000)])
def test_places_kept(kind, beams, V):
    """The chosen ones are the same; a beam's best one in its place, the others by rank in the places left."""
    from qwen600_engine_b200.beams import beam_select
    row = row_of(V, torch.bfloat16, kind, seed=V)
    r = beam_select(row.repeat(beams, 1), torch.zeros((1, beams), device="cuda"), keep_slots=True)
    want = expected(row, range(beams), beams)
    places, later = [(-1, -1)] * beams, []
    for w in want:
        if places[w[0]] == (-1, -1):
            places[w[0]] = w
        else:
            later.append(w)
    for i in range(beams):
        if places[i] == (-1, -1) and later:
            places[i] = later.pop(0)
    assert list(zip(r.parents[0].tolist(), r.tokens[0].tolist())) == places
