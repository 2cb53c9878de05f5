"""The search that the documents show, run as it stands there, against one on the
host.  The model writes each token's place in the cache as decoders do, gives
logits that depend on all that the cache holds of a row, and takes no token
outside the vocabulary."""
import glob
import math
import os
import re

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
V, EOS, LIMIT, BATCH, WIDTH = 50, 7, 8, 5, 4
INF = float("inf")
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def documented():
    blocks = []
    for path in sorted(glob.glob(os.path.join(ROOT, "*.md"))):
        with open(path) as f:
            blocks += re.findall(r"```python\n(.*?)```", f.read(), re.S)
    return [b for b in blocks if "beam_select(" in b]


def logits_of(path, masked):
    """Of a sequence of tokens; masked: two tokens are allowed where its number is even, none where 6 divides it."""
    number = 0
    for t in path:
        number = (number * 31 + t + 1) % 2147483647
    g = torch.Generator().manual_seed(number)
    x = 2 * torch.randn(V, generator=g)
    x[EOS] += 1
    if masked and number % 2 == 0:
        allowed = torch.randperm(V, generator=g)[:0 if number % 6 == 0 else 2]
        x = torch.full((V,), -INF).scatter(0, allowed, x[allowed])
    return x


def search(prompt, masked):
    """[(score, tokens)] of the beams that are left, on the host."""
    held = [(0.0, (), False)]
    for _ in range(LIMIT):
        c = []
        for s, toks, done in held:
            if done:
                c.append((s, toks + (EOS,), True))
                continue
            lp = torch.log_softmax(logits_of(prompt + toks, masked).double(), 0)
            c += [(s + float(lp[t]), toks + (t,), t == EOS) for t in range(V) if float(lp[t]) > -INF]
        c.sort(key=lambda e: -e[0])
        assert all(a[0] - b[0] > 1e-4 for a, b in zip(c[:WIDTH], c[1:WIDTH + 1])), "inputs nearer than rounding"
        held = c[:WIDTH]
    return [(s, toks) for s, toks, _ in held]


@pytest.mark.parametrize("masked", [False, True])
def test_search_as_documented(masked):
    from qwen600_engine_b200.sampler import Sampler
    blocks = documented()
    assert blocks
    # masked: the third and fourth begin with fewer continuations than beams, the last with none
    prompts = [(1, 2, 3), (4, 8, 15, 16, 23), (10, 2), (10, 4), (9, 4, 2)]
    assert [len(search(p, masked)) for p in prompts] == ([WIDTH, WIDTH, WIDTH, 1, 0] if masked else [WIDTH] * BATCH)
    for block in blocks:
        cache = torch.zeros((2, BATCH * WIDTH, 24, 3), device="cuda")
        for b, p in enumerate(prompts):  # all of the prompt but its last token, as a pass over it leaves
            for i, t in enumerate(p[:-1]):
                cache[:, b * WIDTH:(b + 1) * WIDTH, i] = t
        filled = []

        def model(tokens, cache, lengths):
            given, at = tokens.tolist(), lengths.tolist()
            assert all(0 <= t < V for t in given), "an embedding has no such token"
            rows = []
            for row, t in enumerate(given):
                cache[:, row, at[row // WIDTH]] = t
                path = cache[0, row, :at[row // WIDTH] + 1, 0].int().tolist()
                rows.append(logits_of(tuple(path), masked))
            filled.append(at)
            return torch.stack(rows).cuda()

        names = {"batch": BATCH, "width": WIDTH, "limit": LIMIT, "eos": EOS, "cache": cache, "model": model,
                 "tokens": torch.tensor([p[-1] for p in prompts], dtype=torch.int32, device="cuda").repeat_interleave(WIDTH),
                 "lengths": torch.tensor([len(p) - 1 for p in prompts], dtype=torch.int32, device="cuda"),
                 "sequences": torch.full((BATCH * WIDTH, LIMIT), -1, dtype=torch.int32, device="cuda"),
                 "sampler": Sampler(0.0, 1.0, 0.0, 0, 1.3, 0.4, 0.2, 5, 1, max_batch=BATCH * WIDTH, vocab=V)}
        exec(compile(block, "documented search", "exec"), names)
        assert filled == [[len(p) - 1 + step for p in prompts] for step in range(LIMIT)]
        scores, sequences = names["scores"].tolist(), names["sequences"].tolist()
        for b, p in enumerate(prompts):
            got = sorted(((s, tuple(sequences[b * WIDTH + i])) for i, s in enumerate(scores[b]) if s > -INF), reverse=True)
            want = search(p, masked)
            assert [toks for _, toks in got] == [toks for _, toks in want]
            for (s, _), (t, _) in zip(got, want):
                # a step's sum of terms (as for the lists of best tokens), and the rounding of the score so far
                assert abs(s - t) <= LIMIT * ((4 + 6 * math.log(V) + 22) * U + U * abs(t))
