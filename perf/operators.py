"""The operators around the decode tail that are measured, in a plain form and as the framework's calls.

* ``token_logprobs``: log-probability of one chosen token per row of logits, and its backward.
* ``policy_loss``: clipped policy loss with a KL term over sampled tokens, with the gradient of the logits.
* ``preference_loss``: paired log-ratio loss over chosen and rejected sequences, with the gradient of the logits.
* ``lm_head_w4``: final RMSNorm and an lm_head whose weight is held in 4 bits with a scale per group, for few tokens.

Where ``own`` is false, ``run`` computes the plain form from elementary torch operations; where it is true, it makes the
framework's calls.
"""
import math

import torch

own = False

VOCAB = 151936  # rows of the lm_head weight and columns of the logits in this repository's configuration
HIDDEN = 1024

_DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the log-probability that goes back with one sampled token of one sequence
        {"name": "logprobs one row", "op": "logprobs", "rows": 1, "vocab": VOCAB, "dtype": "bf16", "temperature": 0.6},
        # a benchmark batch of sampled tokens, scored for a rollout's old log-probabilities
        {"name": "logprobs batch", "op": "logprobs", "rows": 1024, "vocab": VOCAB, "dtype": "bf16", "temperature": 0.7},
        # scoring in fp32, the full-vocabulary sampling configuration's batch
        {"name": "logprobs f32", "op": "logprobs", "rows": 64, "vocab": VOCAB, "dtype": "f32", "temperature": 0.8},
        # a user's own loss over the log-probabilities: its gradient taken back to the logits; odd vocabulary
        {"name": "logprobs backward", "op": "logprobs_backward", "rows": 509, "vocab": 50021, "dtype": "bf16", "temperature": 1.0},
        # the last step of a short answer, eight sequences
        {"name": "policy few rows", "op": "policy", "rows": 8, "vocab": VOCAB, "dtype": "bf16", "kl": 0.05, "temperature": 1.0},
        # a micro-batch of a rollout: 2048 token positions, a quarter of them prompt or padding
        {"name": "policy rollout", "op": "policy", "rows": 2048, "vocab": VOCAB, "dtype": "bf16", "kl": 0.05, "temperature": 0.7},
        # fp32 logits over a small odd vocabulary, no KL term
        {"name": "policy f32 odd", "op": "policy", "rows": 300, "vocab": 37999, "dtype": "f32", "kl": 0.0, "temperature": 1.0},
        # one pair of short answers
        {"name": "preference one pair", "op": "preference", "pairs": 1, "rows": 18, "vocab": VOCAB, "dtype": "bf16", "smoothing": 0.0},
        # a micro-batch of eight ragged pairs with their prompts
        {"name": "preference batch", "op": "preference", "pairs": 8, "rows": 1900, "vocab": VOCAB, "dtype": "bf16", "smoothing": 0.0},
        # one sequence's decode step over this repository's head
        {"name": "lm_head_w4 one token", "op": "w4", "tokens": 1, "vocab": VOCAB, "hidden": HIDDEN, "group": 128, "zeros": False, "scale": "bf16"},
        # a small serving batch, fine groups with zero points
        {"name": "lm_head_w4 batch", "op": "w4", "tokens": 16, "vocab": VOCAB, "hidden": HIDDEN, "group": 32, "zeros": True, "scale": "f16"},
        # a wider model over a small odd vocabulary, five sequences
        {"name": "lm_head_w4 wide", "op": "w4", "tokens": 5, "vocab": 32003, "hidden": 4096, "group": 64, "zeros": True, "scale": "bf16"},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs_backward", "policy", "preference", "w4"])
    vocab = _spread(rng, 1000, VOCAB)
    if op == "w4":
        hidden = 64 * _spread(rng, 4, 64)
        return {"op": op, "tokens": _spread(rng, 1, 32), "vocab": min(vocab, VOCAB * HIDDEN // hidden), "hidden": hidden,
                "group": rng.choice([g for g in (32, 64, 128) if hidden % g == 0]), "zeros": rng.random() < 0.5,
                "scale": rng.choice(["bf16", "f16"])}
    dtype = rng.choice(["bf16", "bf16", "f32"])
    most = (2048 if dtype == "bf16" else 1024) * VOCAB // vocab
    if op == "preference":
        pairs = _spread(rng, 1, 16)
        return {"op": op, "pairs": pairs, "rows": _spread(rng, 8 * pairs, max(8 * pairs + 1, min(1900, most // 2))), "vocab": vocab,
                "dtype": dtype, "smoothing": rng.choice([0.0, 0.1])}
    rows = _spread(rng, 1, min(2048, most // 2 if op == "logprobs_backward" else most))
    case = {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": rng.choice([0.6, 0.7, 1.0])}
    if op == "policy":
        case["kl"] = rng.choice([0.0, 0.02, 0.1])
    return case


# ------------------------------------------------------------------ inputs
def _logits(g, rows, vocab, dtype):
    """Rows between flat and peaked: Gumbel noise of a scale and an offset of the row's own."""
    x = torch.rand((rows, vocab), generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7).log_().neg_().log_().neg_()
    x.mul_(1.0 + 2.0 * torch.rand((rows, 1), generator=g, device="cuda"))
    x.add_(16.0 * torch.rand((rows, 1), generator=g, device="cuda") - 8.0)
    return x.to(_DTYPE[dtype])


def _drawn_tokens(g, logits, temperature):
    """One token per row, drawn from the row's distribution."""
    u = torch.rand(logits.shape, generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)
    return (logits.float() / temperature - torch.log(-torch.log(u))).argmax(1).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "w4":
        t, v, k, group = case["tokens"], case["vocab"], case["hidden"], case["group"]
        s["hidden_rows"] = torch.randn((t, k), generator=g, device="cuda").to(torch.bfloat16)
        s["norm_weight"] = (1.0 + 0.1 * torch.randn((k,), generator=g, device="cuda")).to(torch.bfloat16)
        # codes as rounding normally distributed weights to 16 levels leaves them
        q = torch.randn((v, k), generator=g, device="cuda").mul_(2.6).add_(8.0).round_().clamp_(0, 15).to(torch.uint8)
        s["codes"] = q[:, 0::2] | (q[:, 1::2] << 4)
        del q
        s["scales"] = (0.01 * (0.5 + torch.rand((v, k // group), generator=g, device="cuda"))).to(_DTYPE[case["scale"]])
        s["zero_points"] = torch.randint(5, 12, (v, k // group), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        if own:  # the handle that a program keeps: the weight laid out once, when it is loaded
            from qwen600_engine_b200.w4 import W4Weight
            s["weight"] = W4Weight.pack(s["codes"], s["scales"], s["zero_points"])
        return s
    temperature = case.get("temperature", 1.0)
    if case["op"] == "preference":
        # ragged sequences, the longest at most three times the shortest; what rounding leaves over is padding behind the last
        pairs, rows = case["pairs"], case["rows"]
        share = 0.5 + torch.rand((2 * pairs,), generator=g, device="cuda", dtype=torch.float64)
        lengths = (rows * share / share.sum()).floor().long()
        offsets = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)])
        s["seq_offsets"] = offsets.to(torch.int32)
        of_row = torch.searchsorted(offsets, torch.arange(rows, device="cuda"), right=True) - 1
        at = torch.arange(rows, device="cuda") - offsets[of_row]
        # a third of each sequence is its prompt; neither it nor the padding is scored
        prompt = (of_row >= 2 * pairs) | (at < (lengths // 3)[of_row.clamp(max=2 * pairs - 1)])
    else:
        rows = case["rows"]
        prompt = torch.rand((rows,), generator=g, device="cuda") < (0.25 if case["op"] == "policy" and rows > 8 else 0.0)
    s["logits"] = _logits(g, rows, case["vocab"], case["dtype"])
    s["tokens"] = _drawn_tokens(g, s["logits"], temperature)
    if case["op"] == "logprobs":
        return s
    lp = _rows(s["logits"], s["tokens"], temperature)[0]
    noise = torch.randn((rows,), generator=g, device="cuda", dtype=torch.float64)
    if case["op"] == "logprobs_backward":
        s["grad_logprobs"] = torch.randn((rows,), generator=g, device="cuda")
        s["stats"] = _plain_logprobs(s)[1]  # what the program keeps of the forward call
    elif case["op"] == "policy":
        # the policy moved since the rollout; ratios within 0.002 of a border of the clip range, where rounding would
        # choose the branch, are moved away from it
        step = 0.15 * noise
        ratio = step.exp()
        near = ((ratio - 0.8).abs() < 2e-3) | ((ratio - 1.2).abs() < 2e-3)
        s["old_logprobs"] = (lp - torch.where(near, step + 0.01, step)).float()
        s["ref_logprobs"] = (lp + 0.2 * torch.randn((rows,), generator=g, device="cuda")).float() if case["kl"] else None
        s["advantages"] = torch.randn((rows,), generator=g, device="cuda")
        active = ~prompt
        s["weights"] = active.float() / active.sum().clamp(min=1)  # mean over the answers' tokens
    else:
        s["tokens"] = torch.where(prompt, torch.full_like(s["tokens"], -1), s["tokens"])
        lp = torch.where(prompt, torch.zeros_like(lp), lp)
        s["ref_logprobs"] = (_per_sequence(lp, s["seq_offsets"]) + 5.0 * noise[:1] + 2.0 * torch.randn((2 * pairs,), generator=g, device="cuda")).float()
    return s


# ------------------------------------------------------------------ plain forms
def _rows(logits, tokens, temperature):
    """Log-probability of each row's token in 64 bits from 32-bit terms; rows whose token is outside the vocabulary
    score 0. Also the terms and their sums, for a gradient."""
    x = logits.float()
    top = x.amax(1, keepdim=True)
    terms = ((x - top) / temperature).exp_()
    total = terms.sum(1, keepdim=True, dtype=torch.float64)
    taken = (tokens >= 0) & (tokens < x.shape[1])
    at = torch.where(taken, tokens, torch.zeros_like(tokens)).long()[:, None]
    lp = (x.gather(1, at) - top).double() / temperature - total.log()
    return torch.where(taken, lp[:, 0], torch.zeros_like(lp[:, 0])), terms, total, taken, at


def _grad_rows(terms, total, taken, at, coef, temperature, dtype):
    """coef * (one-hot - softmax) / temperature, rounded once."""
    c = torch.where(taken, coef, torch.zeros_like(coef)).double()[:, None] / temperature
    grad = terms.mul_((-c / total).float())
    grad.scatter_(1, at, (grad.gather(1, at).double() + c).float())
    return grad.to(dtype)


def _per_sequence(lp, offsets):
    run = torch.cat([lp.new_zeros(1), lp.cumsum(0)])
    return run[offsets[1:].long()] - run[offsets[:-1].long()]


def _plain_logprobs(s):
    """The log-probabilities, and for the backward each row's maximum and its sum of exp((x - maximum) / temperature) beyond
    the maximum's own term (a peaked row's sum is 1 and very little, which 32 bits hold only apart from the 1)."""
    lp, _, total, _, _ = _rows(s["logits"], s["tokens"], s["temperature"])
    return lp.float(), torch.cat([s["logits"].amax(1, keepdim=True).float(), (total - 1).float()], dim=1)


def _plain_logprobs_backward(s):
    terms = ((s["logits"].float() - s["stats"][:, :1]) / s["temperature"]).exp_()
    tokens = s["tokens"]
    taken = (tokens >= 0) & (tokens < s["vocab"])
    at = torch.where(taken, tokens, torch.zeros_like(tokens)).long()[:, None]
    return _grad_rows(terms, s["stats"][:, 1:].double() + 1, taken, at, s["grad_logprobs"], s["temperature"], s["logits"].dtype)


def _plain_policy(s):
    lp, terms, total, taken, at = _rows(s["logits"], s["tokens"], s["temperature"])
    adv, w = s["advantages"].double(), s["weights"].double()
    taken = taken & (w != 0)
    ratio = (lp - s["old_logprobs"].double()).exp()
    loss = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv)
    cut = ((adv > 0) & (ratio > 1.2)) | ((adv < 0) & (ratio < 0.8))
    slope = torch.where(cut, torch.zeros_like(adv), -adv * ratio)
    if s["kl"]:
        d = s["ref_logprobs"].double() - lp
        loss = loss + s["kl"] * (d.exp() - d - 1)
        slope = slope + s["kl"] * (1 - d.exp())
    zero = torch.zeros_like(lp)
    total_loss = torch.where(taken, w * loss, zero).sum()
    grad = _grad_rows(terms, total, taken, at, w * slope, s["temperature"], s["logits"].dtype)
    return total_loss.float(), torch.where(taken, lp, zero).float(), grad


def _plain_preference(s):
    lp, terms, total, taken, at = _rows(s["logits"], s["tokens"], 1.0)
    off = s["seq_offsets"]
    seq = _per_sequence(lp, off)
    pairs, beta, smooth = s["pairs"], 0.1, s["smoothing"]
    r = seq - s["ref_logprobs"].double()
    z = beta * (r[:pairs] - r[pairs:])
    # log(1 + exp(-z)) and log(1 + exp(z)), without overflow
    low = (-z).clamp(min=0) + torch.log1p((-z.abs()).exp())
    loss = ((1 - smooth) * low + smooth * (low + z)).mean()
    slope = -beta * ((1 - smooth) / (1 + z.exp()) - smooth / (1 + (-z).exp())) / pairs
    at_row = torch.searchsorted(off, torch.arange(lp.shape[0], device=off.device), right=True) - 1
    coef = torch.cat([slope, -slope, slope.new_zeros(1)])[at_row]  # rows behind the last sequence take no part
    return loss.float(), seq.float(), _grad_rows(terms, total, taken, at, coef, 1.0, s["logits"].dtype)


def _plain_w4(s):
    x = s["hidden_rows"].float()
    # the normed rows are an output in bf16, and the projection takes them as they are
    normed = (x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-6) * s["norm_weight"].float()).to(torch.bfloat16)
    q = torch.stack([s["codes"] & 15, s["codes"] >> 4], dim=2).float()
    q = q.view(s["vocab"], -1, s["group"])
    zero = 8.0 if s["zero_points"] is None else s["zero_points"].float()[:, :, None]
    w = ((q - zero) * s["scales"].float()[:, :, None]).view(s["vocab"], s["hidden"])
    return normed, (normed.float() @ w.t()).to(torch.bfloat16)


def run(state):
    s = state
    op = s["op"]
    if not own:
        return {"logprobs": _plain_logprobs, "logprobs_backward": _plain_logprobs_backward, "policy": _plain_policy,
                "preference": _plain_preference, "w4": _plain_w4}[op](s)
    from qwen600_engine_b200 import losses, w4
    if op == "logprobs":
        r = losses.token_logprobs(s["logits"], s["tokens"], temperature=s["temperature"])
        return r.logprobs, r.stats
    if op == "logprobs_backward":
        return losses.token_logprobs_backward(s["logits"], s["tokens"], s["stats"], s["grad_logprobs"], temperature=s["temperature"])
    if op == "policy":
        r = losses.policy_loss(s["logits"], s["tokens"], s["old_logprobs"], s["advantages"], ref_logprobs=s["ref_logprobs"],
                               weights=s["weights"], clip_low=0.2, clip_high=0.2, kl_coef=s["kl"], temperature=s["temperature"])
        return r.loss, r.logprobs, r.grad
    if op == "preference":
        r = losses.preference_loss(s["logits"], s["tokens"], s["seq_offsets"], s["ref_logprobs"], beta=0.1, label_smoothing=s["smoothing"])
        return r.loss, r.seq_logprobs, r.grad
    return w4.lm_head_w4(s["hidden_rows"], s["weight"], s["norm_weight"])


# ------------------------------------------------------------------ work
def work(case):
    v = case["vocab"]
    if case["op"] == "w4":
        t, k = case["tokens"], case["hidden"]
        groups = v * (k // case["group"])
        return {"bytes": v * k // 2 + groups * (3 if case["zeros"] else 2) + 4 * t * k + 2 * k + 2 * t * v, "flops": 2 * t * v * k}
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "logprobs":
        return {"bytes": case["rows"] * (v * size + 16), "flops": 4 * case["rows"] * v}
    if case["op"] == "logprobs_backward":
        return {"bytes": case["rows"] * (2 * v * size + 16), "flops": 4 * case["rows"] * v}
    if case["op"] == "policy":
        # a quarter of the rows takes no part where there are more than eight: their zeros are written, nothing is read
        rows, active = case["rows"], case["rows"] if case["rows"] <= 8 else 0.75 * case["rows"]
        return {"bytes": (rows + active) * v * size + 24 * rows, "flops": 7 * active * v}
    # two thirds of each sequence is an answer; the other rows' zeros are written, nothing is read
    rows = case["rows"]
    return {"bytes": rows * (1 + 2 / 3) * v * size + 8 * rows, "flops": 7 * rows * 2 / 3 * v}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_scored(x, tokens, temperature):
    """log softmax(x / temperature) at the tokens, for rows that have one."""
    return torch.log_softmax(x / temperature, dim=1)[torch.arange(x.shape[0], device=x.device), tokens.long()]


def _exact_blocks(logits):
    n = max(1, (1 << 25) // logits.shape[1])
    return [(a, min(a + n, logits.shape[0])) for a in range(0, logits.shape[0], n)]


def _exact_grad(s, fn):
    """Runs fn(scored rows' log-probabilities, their row numbers) block by block and differentiates its sum."""
    logits, tokens, temperature = s["logits"], s["tokens"], s.get("temperature", 1.0)
    grad = torch.zeros(logits.shape, dtype=torch.float64, device=logits.device)
    parts = []
    for a, b in _exact_blocks(logits):
        at = a + ((tokens[a:b] >= 0) & (tokens[a:b] < logits.shape[1]) & (s["active"][a:b])).nonzero()[:, 0]
        if not len(at):
            continue
        x = logits[at].double().requires_grad_(True)
        y = fn(_exact_scored(x, tokens[at], temperature), at)
        y.sum().backward()
        grad[at] = x.grad
        parts.append(y.detach().sum())
    return (torch.stack(parts).sum() if parts else grad.new_zeros(())), grad


def _exact_rows(s):
    out = torch.zeros(s["logits"].shape[0], dtype=torch.float64, device=s["logits"].device)
    for a, b in _exact_blocks(s["logits"]):
        at = a + ((s["tokens"][a:b] >= 0) & (s["tokens"][a:b] < s["logits"].shape[1]) & s["active"][a:b]).nonzero()[:, 0]
        out[at] = _exact_scored(s["logits"][at].double(), s["tokens"][at], s.get("temperature", 1.0))
    return out


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    if op == "w4":
        x = s["hidden_rows"].double()
        normed = x / (x.square().sum(1, keepdim=True) / case["hidden"] + 1e-6).sqrt() * s["norm_weight"].double()
        taken = normed.to(torch.bfloat16).double()  # the projection takes the bf16 rows
        group, logits = case["group"], []
        for a in range(0, case["vocab"], 16384):
            c = s["codes"][a:a + 16384].to(torch.int32)
            w = torch.empty((c.shape[0], case["hidden"]), dtype=torch.float64, device=c.device)
            w[:, 0::2], w[:, 1::2] = c % 16, c // 16
            wide = lambda t: t[a:a + 16384].double().repeat_interleave(group, dim=1)  # noqa: E731
            w = (w - (8 if s["zero_points"] is None else wide(s["zero_points"]))) * wide(s["scales"])
            logits.append(taken @ w.t())
        return normed, torch.cat(logits, dim=1)
    s["active"] = s["weights"] != 0 if op == "policy" else torch.ones_like(s["tokens"], dtype=torch.bool)
    if op == "logprobs":
        top = s["logits"].double().amax(1)
        total = [((s["logits"][a:b].double() - top[a:b, None]) / case["temperature"]).logsumexp(1).expm1() for a, b in _exact_blocks(s["logits"])]
        return _exact_rows(s), torch.stack([top, torch.cat(total)], dim=1)
    if op == "logprobs_backward":
        return _exact_grad(s, lambda lp, at: lp * s["grad_logprobs"][at].double())[1]
    if op == "policy":
        def each(lp, at):
            ratio = torch.exp(lp - s["old_logprobs"][at].double())
            a = s["advantages"][at].double()
            y = -torch.minimum(ratio * a, torch.clamp(ratio, 0.8, 1.2) * a)
            if case["kl"]:
                d = s["ref_logprobs"][at].double() - lp
                y = y + case["kl"] * (torch.expm1(d) - d)
            return s["weights"][at].double() * y
        loss, grad = _exact_grad(s, each)
        return loss, _exact_rows(s), grad
    lp = _exact_rows(s)
    off = s["seq_offsets"].tolist()
    seq = torch.stack([lp[a:b].sum() for a, b in zip(off, off[1:])]).requires_grad_(True)
    r = seq - s["ref_logprobs"].double()
    z = 0.1 * (r[:case["pairs"]] - r[case["pairs"]:])
    smooth = case["smoothing"]
    loss = -((1 - smooth) * torch.nn.functional.logsigmoid(z) + smooth * torch.nn.functional.logsigmoid(-z)).mean()
    loss.backward()
    of_row = torch.zeros_like(lp)
    for i, (a, b) in enumerate(zip(off, off[1:])):
        of_row[a:b] = seq.grad[i]
    return loss.detach(), seq.detach(), _exact_grad(s, lambda p, at: p * of_row[at])[1]
