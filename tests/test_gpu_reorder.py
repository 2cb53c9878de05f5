"""States moved to the beams that go on: every byte against indexing, and a whole
search against one on the host."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def reorder(states, parents, **kw):
    from qwen600_engine_b200 import beams
    return beams.beam_reorder(states, parents, **kw)


def sources(parents):
    batch, beams = parents.shape
    own = torch.arange(beams, device=parents.device).expand(batch, beams)
    p = torch.where((parents >= 0) & (parents < beams), parents.long(), own)
    return (p + beams * torch.arange(batch, device=parents.device)[:, None]).view(-1)


def moved(t, parents, dim=0, lengths=None, length_dim=-2):
    """What `t` has to be, by indexing."""
    want = t.index_select(dim, sources(parents))
    if lengths is None:
        return want
    shape = [1] * t.dim()
    shape[length_dim] = t.shape[length_dim]
    at = torch.arange(t.shape[length_dim], device=t.device).view(shape)
    shape = [1] * t.dim()
    shape[dim] = t.shape[dim]
    held = at < lengths.repeat_interleave(parents.shape[1]).view(shape)
    return torch.where(held, want, t)


def numbers(shape, dtype, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randint(-100, 100, shape, generator=g, device="cuda")
    return x.to(dtype) if dtype != torch.bool else x > 0


def parents_of(maps):
    return torch.tensor(maps, dtype=torch.int32, device="cuda")


MAPS = [[0, 1, 2, 3, 4, 5], [1, 2, 3, 4, 5, 0], [5, 4, 3, 2, 1, 0], [0, 0, 0, 0, 0, 0], [5, 5, 5, 5, 5, 5], [1, 0, 3, 2, 5, 4],
        [1, 2, 0, 0, 4, 1], [1, 2, 3, 4, 5, 5], [0, 0, 1, 2, 3, 4], [2, 2, 0, 0, 5, 4], [-1, 0, 99, 3, -2 ** 31, 2], [0, 0, 2, 2, 4, 4],
        [3, 4, 5, 0, 1, 2], [1, 2, 0, 4, 5, 3], [1, 1, 3, 3, 5, 0]]


@pytest.mark.parametrize("dtype", [torch.uint8, torch.bool, torch.bfloat16, torch.float32, torch.int64, torch.complex128])
@pytest.mark.parametrize("width", [1, 3, 8, 64, 1000])
def test_maps(dtype, width):
    p = parents_of(MAPS)
    t = numbers((len(MAPS) * 6, width), dtype, seed=width)
    want = moved(t, p)
    assert reorder(t, p) is None
    assert torch.equal(t, want)


@pytest.mark.parametrize("beams", [1, 2, 7, 16, 33, 64, 257, 1024])
def test_any_map(beams):
    rng = random.Random(beams)
    maps = []
    for i in range(12):
        kind = i % 4
        m = list(range(beams))
        if kind == 0:
            rng.shuffle(m)
        elif kind == 1:
            m = [rng.randrange(beams) for _ in m]
        elif kind == 2:  # few go on
            m = [rng.choice((0, beams - 1, beams // 2)) for _ in m]
        else:
            m = [rng.randrange(-1, beams + 1) for _ in m]
        maps.append(m)
    p = parents_of(maps)
    t = numbers((12 * beams, 37), torch.float32, seed=beams)
    want = moved(t, p)
    reorder(t, p)
    assert torch.equal(t, want)


@pytest.mark.parametrize("dtype,width", [(torch.bfloat16, 1), (torch.bfloat16, 36), (torch.bfloat16, 128), (torch.float32, 5), (torch.uint8, 77)])
@pytest.mark.parametrize("layout", ["rows first", "by head", "positions, then heads", "stacked layers", "stacked layers by head"])
def test_lengths(dtype, width, layout):
    p = parents_of([MAPS[1], MAPS[6], MAPS[10], MAPS[3], MAPS[9]])
    lengths = torch.tensor([0, 1, 50, 61, 1000], dtype=torch.int32, device="cuda")  # of 61 positions
    lengths[3] = -5 if layout == "by head" else 61
    shape, kw = {"rows first": ((30, 61, width), {}), "by head": ((30, 3, 61, width), {}),
                 "positions, then heads": ((30, 61, 3, width), {"length_dim": -3}),
                 "stacked layers": ((4, 30, 61, width), {"dim": 1}), "stacked layers by head": ((2, 2, 30, 3, 61, width), {"dim": 2})}[layout]
    t = numbers(shape, dtype, seed=width)
    want = moved(t, p, lengths=lengths.clamp(min=0), **kw)
    reorder(t, p, lengths=lengths, **kw)
    assert torch.equal(t, want)
    t = numbers(shape, dtype, seed=width + 1)
    want = moved(t, p, dim=kw.get("dim", 0))
    reorder(t, p, dim=kw.get("dim", 0))
    assert torch.equal(t, want)


def test_views_leave_what_lies_between():
    p = parents_of([MAPS[6], MAPS[1]])
    lengths = torch.tensor([20, 31], dtype=torch.int32, device="cuda")
    whole = numbers((12, 2, 33, 4, 20), torch.bfloat16, seed=1)
    want = whole.clone()
    for view in (lambda w: w[:, 1, 1:32, 1:3, 2:9], lambda w: w[:, 0, :31]):
        view(want).copy_(moved(view(want), p, lengths=lengths, length_dim=1))
        reorder(view(whole), p, lengths=lengths, length_dim=1)
        assert torch.equal(whole, want)
    t = numbers((5, 12), torch.float32, seed=2)  # rows in the last dimension
    want = moved(t, p, dim=1)
    reorder(t, p, dim=1)
    assert torch.equal(t, want)
    t = numbers((12, 40, 7), torch.float32, seed=3).transpose(1, 2)  # positions innermost
    want = moved(t, p, lengths=lengths, length_dim=2)
    reorder(t, p, lengths=lengths, length_dim=2)
    assert torch.equal(t, want)


def test_keys_and_values_between_one_another():
    p = parents_of([MAPS[9], MAPS[1]])
    whole = numbers((3, 2, 12, 30, 8), torch.bfloat16, seed=4)  # layers, keys and values, rows
    want = moved(whole, p, dim=2)
    reorder([whole[:, 0], whole[:, 1]], p, dim=1)
    assert torch.equal(whole, want)
    whole = numbers((12, 2, 30, 8), torch.bfloat16, seed=5)
    want = moved(whole, p)
    reorder([whole[:, 0], whole[:, 1]], p)
    assert torch.equal(whole, want)


@pytest.mark.parametrize("count", [1, 2, 39, 40, 41, 100])
def test_lists_of_unlike_states(count):
    p = parents_of([MAPS[6], MAPS[2], MAPS[4]])
    shapes = [((18, 40, 16), torch.bfloat16), ((18, 3), torch.int64), ((18,), torch.int32), ((18, 1), torch.uint8), ((18, 5, 40, 7), torch.float32),
              ((18, 0, 4), torch.float32)]
    states = [numbers(*shapes[i % 6], seed=i) for i in range(count)]
    want = [moved(t, p) for t in states]
    reorder(states, p)
    assert all(torch.equal(t, w) for t, w in zip(states, want))
    reorder([], p)


def test_large_state():
    """A cache whose offsets pass 32 bits."""
    p = parents_of([[1, 0, 1]])
    t = torch.zeros((3, 70000, 17000), dtype=torch.uint8, device="cuda")
    t[0, 69990:] = 3
    t[1, 69990:] = numbers((10, 17000), torch.uint8, seed=6)
    t[2, 5] = 9
    first, second = t[0, 69990:].clone(), t[1, 69990:].clone()
    reorder(t, p, lengths=torch.tensor([70000], dtype=torch.int32, device="cuda"))
    assert torch.equal(t[0, 69990:], second) and torch.equal(t[1, 69990:], first) and torch.equal(t[2, 69990:], second)
    assert not t[:, :69990].any()


def test_no_entry():
    reorder(torch.empty((0, 5), device="cuda"), torch.empty((0, 4), dtype=torch.int32, device="cuda"))


def test_streams_and_graphs():
    p = parents_of([MAPS[1], MAPS[6]])
    lengths = torch.tensor([9, 30], dtype=torch.int32, device="cuda")
    start = numbers((4, 12, 31, 24), torch.bfloat16, seed=7)
    t = start.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    reorder(t, p, dim=1, lengths=lengths, stream=side)
    side.synchronize()
    want = moved(start, p, dim=1, lengths=lengths)
    assert torch.equal(t, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        reorder(t, p, dim=1, lengths=lengths)
    assert torch.equal(t, want)
    p.copy_(parents_of([MAPS[7], MAPS[2]]))  # the next step's parents and lengths
    lengths += 1
    for _ in range(2):
        want = moved(want, p, dim=1, lengths=lengths)
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(t, want)


def test_autograd_sees_the_write():
    t = torch.ones((6, 3), device="cuda", requires_grad=True)
    y = (t * 2).clone()
    z = (y * y).sum()
    reorder(y.detach(), parents_of([MAPS[1]]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


# ------------------------------------------------------------------ together
def test_sampler_history_follows_the_beams():
    """Penalties of reordered rows are those of samplers that saw the parents' tokens."""
    from qwen600_engine_b200.sampler import Sampler
    V, B = 3001, 6
    g = torch.Generator(device="cuda")
    g.manual_seed(8)

    def make():
        return Sampler(0.0, 1.0, 0.0, 0, 1.3, 0.4, 0.2, 5, 1, max_batch=B, vocab=V)

    steps = [torch.randn((B, V), generator=g, device="cuda") for _ in range(14)]
    p = parents_of([MAPS[6][:3], [1, 1, 0]])  # two entries of three beams
    row = sources(p)
    s = make()
    other = make()
    for x in steps[:7]:
        s.sample(x * 0.02)
        other.sample(x.index_select(0, row) * 0.02)
    s.reorder_history(p)
    for x in steps[7:]:
        assert torch.equal(s.sample(x * 0.02), other.sample(x * 0.02))
    Sampler(0.0, 1.0, 0.0, 0, 1.0, 0.0, 0.0, 0, 1, max_batch=B, vocab=V).reorder_history(p)  # no history: nothing to move


@pytest.mark.parametrize("keep", [False, True])
def test_a_search_from_hidden_states(keep):
    """lm_head, selection and reordering step by step, against a search on the host over the same logits."""
    from qwen600_engine_b200 import beams
    from qwen600_engine_b200.sampler import lm_head
    batch, width, V, D, steps, eos = 3, 4, 2048, 128, 9, 5
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    weight = (torch.randn((V, D), generator=g, device="cuda") * 0.3).to(torch.bfloat16)
    weight[eos] += 0.05
    embed = torch.randn((V, D), generator=g, device="cuda")
    state = torch.randn((batch, 1, D), generator=g, device="cuda").expand(batch, width, D).reshape(-1, D).contiguous()
    cache = torch.zeros((2, batch * width, steps, 8), dtype=torch.bfloat16, device="cuda")  # a position's token, as the program keeps it
    history = torch.full((batch * width, steps), -1, dtype=torch.int32, device="cuda")
    scores = torch.full((batch, width), -float("inf"), device="cuda")
    scores[:, 0] = 0
    finished = torch.zeros((batch, width), dtype=torch.bool, device="cuda")
    host = [[(0.0, (), state[b * width].double().cpu(), False)] for b in range(batch)]
    lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def advance(h, tok):
        return 0.7 * h + embed[tok.long().clamp(min=0)].to(h.dtype)

    for step in range(steps):
        _, logits = lm_head(state.to(torch.bfloat16), weight)
        r = beams.beam_select(logits, scores, finished=finished, eos_token=eos, keep_slots=keep)
        beams.beam_reorder([cache], r.parents, dim=1, lengths=lengths)
        beams.beam_reorder([history, state], r.parents)
        scores, finished = r.scores, r.finished
        history[:, step] = r.tokens.view(-1)
        cache[:, :, step] = r.tokens.view(1, -1, 1).to(torch.bfloat16)
        lengths += 1
        state = advance(state, r.tokens.view(-1))
        # the host's search, from the logits of the hidden states that its own beams hold
        for b in range(batch):
            c = []
            for s, toks, h, done in host[b]:
                if done:
                    c.append((s, toks + (eos,), h, True))
                    continue
                _, x = lm_head(h.float().to(torch.bfloat16).view(1, -1).cuda(), weight)
                lp = torch.log_softmax(x.double(), 1)[0]
                v, at = (t[:width] for t in lp.sort(descending=True, stable=True))  # equal ones by token
                c += [(s + float(y), toks + (int(t),), None if done else h, int(t) == eos) for y, t in zip(v, at)]
            c.sort(key=lambda e: -e[0])
            host[b] = [(s, toks, advance(h.float().cuda(), torch.tensor([toks[-1]], device="cuda"))[0].double().cpu(), done)
                       for s, toks, h, done in c[:width]]
    for b in range(batch):
        got = sorted(((float(scores[b, i]), tuple(history[b * width + i].tolist())) for i in range(width)), reverse=True)
        want = [(s, toks) for s, toks, _, _ in host[b]]
        for (s, toks), (t, other) in zip(got, want):
            assert toks == other and abs(s - t) < 1e-4
    assert torch.equal(cache[0, :, :, 0].float(), history.to(torch.bfloat16).float())
