"""The operators on the best few tokens of a row that are measured, in a plain form and as the framework's calls.

* ``top_logprobs``: the k best tokens of each row of logits with their log-probabilities.
* ``distill_loss``: divergence from a teacher that is known by its best tokens, with the gradient of the logits.
* ``beam_select``: one step of beam search over beams and vocabulary.
* ``beam_reorder``: per-row states moved to the beams that go on, in place.

Where ``own`` is false, ``run`` computes the plain form from elementary torch operations; where it is true, it makes the
framework's calls.
"""
import math

import torch

own = False

VOCAB = 151936  # columns of the logits in this repository's configuration
LAYERS, KV = 28, 1024  # its layers, and the width of a position's keys or values in one of them

_DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # alternatives returned beside one sampled token of one sequence
        {"name": "top one row", "op": "top", "rows": 1, "vocab": VOCAB, "k": 20, "dtype": "bf16", "temperature": 0.6},
        # a teacher's pass over a micro-batch of 1024 positions
        {"name": "top teacher batch", "op": "top", "rows": 1024, "vocab": VOCAB, "k": 64, "dtype": "bf16", "temperature": 1.0},
        # fp32 logits over an odd vocabulary, a long list
        {"name": "top f32 long list", "op": "top", "rows": 61, "vocab": 50021, "k": 250, "dtype": "f32", "temperature": 0.8},
        # the last positions of a short answer
        {"name": "distill few rows", "op": "distill", "rows": 8, "vocab": VOCAB, "k": 20, "dtype": "bf16", "rest": True, "temperature": 1.0},
        # a micro-batch of 2048 positions, a quarter of them prompt or padding
        {"name": "distill micro-batch", "op": "distill", "rows": 2048, "vocab": VOCAB, "k": 64, "dtype": "bf16", "rest": True, "temperature": 1.0},
        # fp32 logits over a small odd vocabulary, the teacher renormalised over a long list and softened
        {"name": "distill f32 odd", "op": "distill", "rows": 300, "vocab": 37999, "k": 129, "dtype": "f32", "rest": False, "temperature": 2.0},
        # one sequence's search; twice as many candidates as beams, so that enough go on behind those that end
        {"name": "beams one sequence", "op": "beams", "batch": 1, "beams": 4, "vocab": VOCAB, "n": 8, "finished": 0, "keep": False, "masked": False, "dtype": "bf16", "temperature": 1.0},
        # a serving batch whose ended beams stay in the race, children in their parents' places
        {"name": "beams serving batch", "op": "beams", "batch": 64, "beams": 8, "vocab": VOCAB, "n": 8, "finished": 1, "keep": True, "masked": False, "dtype": "bf16", "temperature": 1.0},
        # fp32 logits over an odd vocabulary most of which a grammar masks
        {"name": "beams f32 masked", "op": "beams", "batch": 7, "beams": 5, "vocab": 50021, "n": 10, "finished": 2, "keep": False, "masked": True, "dtype": "f32", "temperature": 0.7},
        # one short sequence's keys and values after a step: all layers, the first positions of a long cache
        {"name": "reorder short", "op": "reorder", "outer": 2 * LAYERS, "batch": 1, "beams": 4, "moved": 2, "heads": 0, "capacity": 512, "length": 40, "width": KV, "dtype": "bf16"},
        # a batch of eight sequences of different lengths
        {"name": "reorder batch", "op": "reorder", "outer": 2 * LAYERS, "batch": 8, "beams": 4, "moved": 2, "heads": 0, "capacity": 1024, "length": 1000, "width": KV, "dtype": "bf16"},
        # keys and values by head, of an odd width, more beams
        {"name": "reorder heads", "op": "reorder", "outer": 12, "batch": 3, "beams": 10, "moved": 4, "heads": 5, "capacity": 301, "length": 299, "width": 36, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["top", "distill", "beams", "reorder"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "reorder":
        beams = _spread(rng, 2, 16)
        heads, width = rng.choice([(0, 8 * _spread(rng, 8, 128)), (_spread(rng, 1, 8), _spread(rng, 16, 256))])
        batch, outer = _spread(rng, 1, 8), _spread(rng, 2, 2 * LAYERS)
        most = (1 << 30) // (batch * beams * outer * max(1, heads) * width)
        capacity = _spread(rng, 8, max(9, min(2048, most)))
        return {"op": op, "outer": outer, "batch": batch, "beams": beams, "moved": rng.randint(1, beams - 1), "heads": heads,
                "capacity": capacity, "length": _spread(rng, 1, capacity), "width": width, "dtype": dtype}
    vocab = _spread(rng, 1000, VOCAB)
    most = (1024 if dtype == "bf16" else 512) * VOCAB // vocab
    temperature = rng.choice([0.7, 1.0, 2.0])
    if op == "beams":
        beams = _spread(rng, 1, 16)
        batch = _spread(rng, 1, max(1, min(64, most // beams)))
        keep = rng.random() < 0.4
        return {"op": op, "batch": batch, "beams": beams, "vocab": vocab, "n": beams if keep else rng.randint(1, 2 * beams),
                "finished": rng.randint(0, beams - 1), "keep": keep, "masked": rng.random() < 0.3, "dtype": dtype, "temperature": temperature}
    case = {"op": op, "rows": _spread(rng, 1, min(1500, most)), "vocab": vocab, "k": _spread(rng, 1, 256), "dtype": dtype, "temperature": temperature}
    if op == "distill":
        case["rest"] = rng.random() < 0.6
    return case


# ------------------------------------------------------------------ inputs
def _logits(g, rows, vocab, dtype):
    """Rows between flat and peaked: Gumbel noise of a scale and an offset of the row's own."""
    x = torch.rand((rows, vocab), generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7).log_().neg_().log_().neg_()
    x.mul_(1.0 + 2.0 * torch.rand((rows, 1), generator=g, device="cuda"))
    x.add_(16.0 * torch.rand((rows, 1), generator=g, device="cuda") - 8.0)
    return x.to(_DTYPE[dtype])


def _places(g, batch, beams, count):
    """[batch, beams] truth values, `count` of each entry's true."""
    order = torch.rand((batch, beams), generator=g, device="cuda").argsort(1).argsort(1)
    return order < count


def _lengths(case):
    """Ragged: the last sequence is about half as long as the first."""
    return [max(1, round(case["length"] * (1 - 0.5 * b / case["batch"]))) for b in range(case["batch"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "reorder":
        batch, beams = case["batch"], case["beams"]
        shape = [case["outer"], batch * beams] + ([case["heads"]] if case["heads"] else []) + [case["capacity"], case["width"]]
        s["cache"] = torch.randn(shape, generator=g, device="cuda", dtype=_DTYPE[case["dtype"]])
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        # what a step that keeps children in their parents' places leaves: `moved` beams of each sequence end, and each of
        # their places is taken by a further child of one that goes on
        gone = _places(g, batch, beams, case["moved"])
        order = gone.int().argsort(dim=1, stable=True)  # those that go on, then those that end
        stay = beams - case["moved"]
        rank = torch.arange(beams, device="cuda").expand(batch, beams)
        source = order.gather(1, torch.where(rank < stay, rank, (rank - stay) % stay))
        s["parents"] = torch.empty((batch, beams), dtype=torch.int32, device="cuda").scatter_(1, order, source.int())
        return s
    temperature = case["temperature"]
    if case["op"] == "beams":
        batch, beams, n = case["batch"], case["beams"], case["n"]
        s["logits"] = _logits(g, batch * beams, case["vocab"], case["dtype"])
        if case["masked"]:
            s["logits"].masked_fill_(torch.rand(s["logits"].shape, generator=g, device="cuda") < 0.95, float("-inf"))
        s["finished_beams"] = _places(g, batch, beams, case["finished"])
        s["eos"] = 7
        s["scores"] = (-30.0 * torch.rand((batch, 1), generator=g, device="cuda") - 4.0 * torch.rand((batch, beams), generator=g, device="cuda") - 1.0)
        # candidates of different beams that are nearer than rounding can tell apart are moved away from one another
        best, tokens = _best(s["logits"], min(n + 1, case["vocab"]))
        lp = _logprobs_of(s["logits"], best, tokens, temperature).view(batch, beams, -1)
        lp = torch.where(s["finished_beams"][:, :, None], torch.full_like(lp, float("-inf")), lp)
        lp[:, :, 0] = torch.where(s["finished_beams"], torch.zeros_like(lp[:, :, 0]), lp[:, :, 0])
        beam = torch.arange(beams, device="cuda")[None, :, None].expand_as(lp).reshape(batch, -1)
        for _ in range(4):
            every, at = (s["scores"].double()[:, :, None] + lp).view(batch, -1).sort(1, descending=True)
            of = beam.gather(1, at)
            near = ((every[:, :-1] - every[:, 1:] < 1e-3) & (of[:, :-1] != of[:, 1:]))[:, :2 * n].any(1, keepdim=True)
            s["scores"] = torch.where(near, s["scores"] - torch.rand((batch, beams), generator=g, device="cuda"), s["scores"])
        return s
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    s["logits"] = _logits(g, rows, vocab, case["dtype"])
    if case["op"] == "distill":
        # the teacher's logits: the student's, moved
        teacher = (s["logits"].float() + 1.5 * torch.randn((rows, vocab), generator=g, device="cuda")).to(_DTYPE[case["dtype"]])
        best, tokens = _best(teacher, k)
        s["teacher_tokens"], s["teacher_logprobs"] = tokens.int(), _logprobs_of(teacher, best, tokens, temperature).float()
        left = torch.rand((rows,), generator=g, device="cuda").argsort() >= _left_out(case)
        s["weights"] = left.float() / left.sum().clamp(min=1)  # mean over the answers' tokens
    return s


def _left_out(case):
    return case["rows"] // 4 if case["rows"] > 8 else 0


# ------------------------------------------------------------------ plain forms
def _best(logits, k):
    """Values and tokens of each row's k largest logits, equal ones by token: each logit's bits as a whole number of the same
    order, followed by the token's distance from the end."""
    bits = (logits.float() + 0.0).view(torch.int32)  # + 0.0: a zero without sign
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    at = ((bits << 18) - torch.arange(logits.shape[1], device=logits.device)).topk(k, dim=1).indices
    return logits.gather(1, at).float(), at


def _logprobs_of(logits, values, tokens, temperature):
    """Log-probabilities in 64 bits from 32-bit terms."""
    x = logits.float()
    top = x.amax(1, keepdim=True)
    total = ((x - top) / temperature).exp_().sum(1, keepdim=True, dtype=torch.float64)
    return (values.double() - top.double()) / temperature - total.log()


def _plain_top(s):
    best, tokens = _best(s["logits"], s["k"])
    return _logprobs_of(s["logits"], best, tokens, s["temperature"]).float(), tokens.int()


def _plain_distill(s):
    temperature, dtype = s["temperature"], s["logits"].dtype
    x, at = s["logits"].float(), s["teacher_tokens"].long()
    top = x.amax(1, keepdim=True)
    listed_x = x.gather(1, at)
    terms = ((x - top) / temperature).exp_()
    terms.scatter_(1, at, 0.0)
    rest = terms.sum(1, keepdim=True, dtype=torch.float64)  # unlisted tokens, apart from the listed ones
    d = (listed_x.double() - top.double()) / temperature
    total = rest + d.exp().sum(1, keepdim=True)
    q = s["teacher_logprobs"].double().exp()
    log_q = s["teacher_logprobs"].double()
    if s["rest"]:
        q_rest = (1 - q.sum(1, keepdim=True)).clamp(min=0)
        left = torch.xlogy(q_rest, q_rest) - q_rest * (rest / total).log()
        left = torch.where(q_rest > 0, left, torch.zeros_like(left))
    else:
        log_q = log_q - q.sum(1, keepdim=True).log()
        q = log_q.exp()
        q_rest = left = torch.zeros_like(rest)
    row = (q * (log_q - (d - total.log()))).sum(1) + left[:, 0]
    w = s["weights"].double()
    c = w[:, None] / temperature
    mass = q.sum(1, keepdim=True) + q_rest
    grad = terms.mul_((c * (mass / total - q_rest / rest)).float())
    grad.scatter_(1, at, (c * (mass * d.exp() / total - q)).float())
    zero = torch.zeros_like(row)
    row = torch.where(w != 0, row, zero)
    return (w * row).sum().float(), row.float(), grad.to(dtype)


def _plain_beams(s):
    batch, beams, n, eos = s["batch"], s["beams"], s["n"], s["eos"]
    k = min(n, s["vocab"])
    best, tokens = _best(s["logits"], k)
    score = s["scores"].double()[:, :, None] + _logprobs_of(s["logits"], best, tokens, s["temperature"]).view(batch, beams, k)
    tokens = tokens.int().view(batch, beams, k)
    done = s["finished_beams"]
    # an ended beam goes on with its own score and nothing else
    first = torch.arange(k, device=score.device) == 0
    alone = torch.where(first, s["scores"].double()[:, :, None], torch.full_like(score, float("-inf")))
    score = torch.where(done[:, :, None], alone, score).view(batch, -1)
    tokens = torch.where(done[:, :, None], torch.full_like(tokens, eos), tokens).view(batch, -1)
    score, at = score.sort(dim=1, descending=True, stable=True)  # equal ones by beam, then by token
    score, at = score[:, :n], at[:, :n]
    none = score == float("-inf")
    parents = torch.where(none, torch.full_like(at, -1), at // k)
    tokens = torch.where(none, torch.full_like(at, -1), tokens.gather(1, at).long())
    ended = none | (tokens == eos) | (done.gather(1, parents.clamp(min=0)) & ~none)
    if s["keep"]:
        rank = torch.arange(n, device=score.device)
        earlier = (parents[:, :, None] == parents[:, None, :]) & (rank[None, :] < rank[:, None])
        stays = ~none & ~earlier.any(2)
        taken = (torch.where(stays, parents, torch.full_like(parents, -1))[:, None, :] == rank[None, :, None]).any(2)
        free = taken.int().argsort(dim=1, stable=True)
        slot = torch.where(stays, parents, free.gather(1, ((~stays).cumsum(1) - 1).clamp(min=0)))
        put = lambda t: torch.empty_like(t).scatter_(1, slot, t)  # noqa: E731
        score, parents, tokens, ended = put(score), put(parents), put(tokens), put(ended)
    return score.float(), parents.int(), tokens.int(), ended


def _plain_reorder(s):
    cache, parents = s["cache"], s["parents"]
    batch, beams = parents.shape
    row = (parents + beams * torch.arange(batch, device=parents.device)[:, None]).view(-1)
    held = torch.arange(s["capacity"], device=parents.device) < s["lengths"].repeat_interleave(beams)[:, None]
    held = held[None, :, None, :, None] if s["heads"] else held[None, :, :, None]
    torch.where(held, cache[:, row.long()], cache, out=cache)
    return cache


def run(state):
    s = state
    op = s["op"]
    if not own:
        return {"top": _plain_top, "distill": _plain_distill, "beams": _plain_beams, "reorder": _plain_reorder}[op](s)
    from qwen600_engine_b200 import beams, losses
    if op == "top":
        r = losses.top_logprobs(s["logits"], s["k"], temperature=s["temperature"])
        return r.logprobs, r.tokens
    if op == "distill":
        r = losses.distill_loss(s["logits"], s["teacher_tokens"], s["teacher_logprobs"], weights=s["weights"],
                                temperature=s["temperature"], rest=s["rest"])
        return r.loss, r.row_losses, r.grad
    if op == "beams":
        r = beams.beam_select(s["logits"], s["scores"], n=s["n"], finished=s["finished_beams"], eos_token=s["eos"],
                              temperature=s["temperature"], keep_slots=s["keep"])
        return r.scores, r.parents, r.tokens, r.finished
    beams.beam_reorder(s["cache"], s["parents"], dim=1, lengths=s["lengths"], length_dim=-2)
    return s["cache"]


# ------------------------------------------------------------------ work
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "reorder":
        # each place that changes is written, each beam that is taken from is read once
        stay = case["beams"] - case["moved"]
        position = case["outer"] * max(1, case["heads"]) * case["width"] * size
        return {"bytes": sum(_lengths(case)) * position * (case["moved"] + min(case["moved"], stay)), "flops": 0}
    v = case["vocab"]
    if case["op"] == "top":
        return {"bytes": case["rows"] * (v * size + 8 * case["k"]), "flops": 4 * case["rows"] * v}
    if case["op"] == "beams":
        live = case["batch"] * (case["beams"] - case["finished"])
        return {"bytes": live * v * size + case["batch"] * (5 * case["beams"] + 13 * case["n"]), "flops": 4 * live * v}
    # rows that are left out: their zeros are written, nothing is read
    rows, active = case["rows"], case["rows"] - _left_out(case)
    return {"bytes": (rows + active) * v * size + 8 * active * case["k"] + 8 * rows, "flops": 7 * active * v}


# ------------------------------------------------------------------ the definition in 64 bits
def _blocks(rows, vocab):
    n = max(1, (1 << 25) // vocab)
    return [(a, min(a + n, rows)) for a in range(0, rows, n)]


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    if op == "reorder":
        moved, beams = s["cache"].clone(), case["beams"]
        for b, (count, sources) in enumerate(zip(_lengths(case), s["parents"].tolist())):
            for i, p in enumerate(sources):
                moved[:, b * beams + i].narrow(-2, 0, count).copy_(s["cache"][:, b * beams + p].narrow(-2, 0, count))
        return moved
    x, t = s["logits"], case["temperature"]
    if op == "top":
        return torch.cat([torch.log_softmax(x[a:b].double() / t, 1).topk(case["k"], 1).values for a, b in _blocks(*x.shape)]), None
    if op == "beams":
        batch, beams, n = case["batch"], case["beams"], case["n"]
        best = []
        for a, b in _blocks(*x.shape):
            y = torch.log_softmax(x[a:b].double() / t, 1) + s["scores"].view(-1)[a:b, None].double()
            best.append(y.topk(min(n, case["vocab"]), 1).values)
        best = torch.cat(best).view(batch, beams, -1)
        ended = s["finished_beams"].nonzero()
        best[ended[:, 0], ended[:, 1]] = -math.inf
        best[ended[:, 0], ended[:, 1], 0] = s["scores"][ended[:, 0], ended[:, 1]].double()
        best = best.view(batch, -1)
        if not case["keep"]:
            return best.sort(1, descending=True).values[:, :n], None, None, None
        # each beam's best child in its parent's place, the others by rank in what is left
        placed = torch.full((batch, n), -math.inf, dtype=torch.float64)
        for b, row in enumerate(best.tolist()):
            every = sorted(((v, -(i // (len(row) // beams))) for i, v in enumerate(row) if v > -math.inf), reverse=True)[:n]
            later = []
            for v, minus in every:
                if placed[b, -minus] == -math.inf:
                    placed[b, -minus] = v
                else:
                    later.append(v)
            for i in range(n):
                if placed[b, i] == -math.inf and later:
                    placed[b, i] = later.pop(0)
        return placed.to(best.device), None, None, None
    row_losses, grads = [], []
    for a, b in _blocks(*x.shape):
        y = x[a:b].double().requires_grad_(True)
        lp = torch.log_softmax(y / t, 1)
        at, given = s["teacher_tokens"][a:b].long(), s["teacher_logprobs"][a:b].double()
        w = s["weights"][a:b].double()
        if case["rest"]:
            q = given.exp()
            r = torch.clamp(1 - q.sum(1), min=0)
            unlisted = lp.scatter(1, at, -math.inf).logsumexp(1)
            each = torch.nn.functional.kl_div(lp.gather(1, at), q, reduction="none").sum(1) + torch.nn.functional.kl_div(unlisted, r, reduction="none")
        else:
            q = torch.softmax(given, 1)
            each = (q * (q.log() - lp.gather(1, at))).sum(1)
        each = torch.where(w != 0, each, torch.zeros_like(each))
        (w * each).sum().backward()
        row_losses.append(each.detach())
        grads.append(y.grad)
    row_losses = torch.cat(row_losses)
    return (s["weights"].double() * row_losses).sum(), row_losses, torch.cat(grads)
