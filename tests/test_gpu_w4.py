"""The lm_head with 4-bit weights against its formula in 64 bits.

Tolerance of a logit: a product of a code minus its zero point (an integer
below 16) and a bf16 value is exact in fp32; each of the K additions and each
group's scaling may lose a whole step of fp32 (tensor-core sums may truncate),
2^-23 of the sum of magnitudes; the output is rounded to bf16, 2^-8 of its
value at most."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def plain_weight(V, K, group, zeros, scale, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    q = torch.randint(0, 16, (V, K), generator=g, device="cuda", dtype=torch.uint8)
    codes = q[:, 0::2] | (q[:, 1::2] << 4)
    scales = (0.001 + 0.02 * torch.rand((V, K // group), generator=g, device="cuda")).to(scale)
    scales *= (torch.rand((V, K // group), generator=g, device="cuda") < 0.9).to(scale) * 2 - 1  # some negative
    z = torch.randint(0, 16, (V, K // group), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return codes.contiguous(), scales, z, g


def dense(codes, scales, zeros):
    """The weight in 64 bits."""
    V, K = codes.shape[0], 2 * codes.shape[1]
    q = torch.stack([codes & 15, codes >> 4], dim=2).view(V, scales.shape[1], -1).double()
    z = 8.0 if zeros is None else zeros.double()[:, :, None]
    return ((q - z) * scales.double()[:, :, None]).view(V, K)


def check_logits(normed, w, logits):
    K = w.shape[1]
    for a in range(0, w.shape[0], 1 << 15):
        b = w[a:a + (1 << 15)]
        ref = normed.double() @ b.t()
        tol = 2.0 ** -8 * ref.abs() + (K + 8) * 2.0 ** -23 * (normed.double().abs() @ b.abs().t()) * 1.01 + 1e-38
        off = (logits[:, a:a + (1 << 15)].double() - ref).abs()
        assert (off <= tol).all(), f"off by {float((off / tol).max()):.3g} tolerances"


def inputs(g, B, K):
    h = torch.randn((B, K), generator=g, device="cuda").to(torch.bfloat16)
    nw = (1.0 + 0.1 * torch.randn((K,), generator=g, device="cuda")).to(torch.bfloat16)
    return h, nw


@pytest.mark.parametrize("B,V,K,group", [
    (1, 1, 64, 32), (1, 151936, 1024, 128), (1, 1003, 1024, 64), (2, 16, 128, 128), (3, 17, 192, 64), (5, 4099, 320, 32),
    (7, 33, 8192, 128), (8, 1000, 1024, 32), (9, 1000, 1024, 128), (16, 32003, 4096, 64), (17, 257, 2048, 128),
    (31, 75968, 1024, 128), (32, 5000, 1024, 32), (33, 2500, 4096, 128), (70, 1003, 1024, 64), (130, 300, 256, 128)])
@pytest.mark.parametrize("zeros,scale", [(False, torch.bfloat16), (True, torch.float16)])
def test_lm_head_w4(B, V, K, group, zeros, scale):
    from qwen600_engine_b200.sampler import lm_head
    from qwen600_engine_b200.w4 import W4Weight, lm_head_w4
    codes, scales, z, g = plain_weight(V, K, group, zeros, scale, seed=V + K)
    w = W4Weight.pack(codes, scales, z)
    assert (w.vocab, w.hidden_dim, w.group) == (V, K, group)
    h, nw = inputs(g, B, K)
    normed, logits = lm_head_w4(h, w, nw)
    assert normed.shape == (B, K) and logits.shape == (B, V) and logits.dtype == torch.bfloat16
    assert torch.equal(normed, lm_head(h, torch.zeros((8, K), dtype=torch.bfloat16, device="cuda"), nw)[0])
    check_logits(normed, dense(codes, scales, z), logits)
    plain = lm_head_w4(h, w)[0]  # no norm weight: ones
    assert torch.equal(plain, lm_head(h, torch.zeros((8, K), dtype=torch.bfloat16, device="cuda"))[0])


def test_every_code_at_every_place():
    """One weight column at a time: each code and zero point reaches its own product, at full precision."""
    from qwen600_engine_b200.w4 import W4Weight, lm_head_w4
    for group in (32, 64, 128):
        K, V = 256, 256
        g = torch.Generator(device="cuda")
        g.manual_seed(group)
        q = torch.randint(0, 16, (V, K), generator=g, device="cuda", dtype=torch.uint8)
        codes = (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous()
        scales = torch.full((V, K // group), 0.5, dtype=torch.bfloat16, device="cuda")
        scales *= 2.0 ** torch.randint(-3, 4, scales.shape, generator=g, device="cuda").to(torch.bfloat16)
        z = torch.randint(0, 16, (V, K // group), generator=g, device="cuda", dtype=torch.uint8)
        w = W4Weight.pack(codes, scales, z)
        h = torch.eye(K, device="cuda").to(torch.bfloat16)  # row k picks column k, scaled by the norm to 16
        normed, logits = lm_head_w4(h, w)
        ref = normed.double() @ dense(codes, scales, z).t()
        assert torch.equal(logits.double(), ref.to(torch.bfloat16).double())


def test_one_row_does_not_depend_on_the_batch():
    """The rows of a batch are independent: values that are not numbers in one leave the others as they are."""
    from qwen600_engine_b200.w4 import W4Weight, lm_head_w4
    codes, scales, z, g = plain_weight(3001, 1024, 64, True, torch.bfloat16, seed=5)
    w = W4Weight.pack(codes, scales, z)
    h, nw = inputs(g, 13, 1024)
    a = lm_head_w4(h, w, nw)[1]
    h[4] = float("nan")
    h[7, 3] = float("inf")
    b = lm_head_w4(h, w, nw)[1]
    keep = [r for r in range(13) if r not in (4, 7)]
    assert torch.equal(a[keep], b[keep])
    assert torch.isnan(b[[4, 7]]).all()


def test_rows_of_any_magnitude():
    """Rows whose values differ by up to 2^24, tiny and huge rows, a row of zeros."""
    from qwen600_engine_b200.w4 import W4Weight, lm_head_w4
    K, V = 512, 1000
    for group, zeros in ((32, True), (128, False)):
        codes, scales, z, g = plain_weight(V, K, group, zeros, torch.bfloat16, seed=group)
        w = W4Weight.pack(codes, scales, z)
        h, nw = inputs(g, 10, K)
        h[1] = (h[1].float() * torch.exp2(torch.randint(-12, 13, (K,), generator=g, device="cuda").float())).to(torch.bfloat16)
        h[2] = 0.0
        h[3] *= 2.0 ** -80
        h[4, 5] = 3.0e4
        h[5, 1:] = 0.0
        big = (nw.float() * 2.0 ** 90).to(torch.bfloat16)
        small = (nw.float() * 2.0 ** -100).to(torch.bfloat16)
        for weight in (nw, big, small):
            normed, logits = lm_head_w4(h, w, weight)
            assert torch.isfinite(logits).all() and (logits[2] == 0).all()
            check_logits(normed, dense(codes, scales, z), logits)


def test_quantize():
    from qwen600_engine_b200.w4 import W4Weight, lm_head_w4, quantize_w4
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    V, K = 1003, 512
    wt = (0.02 * torch.randn((V, K), generator=g, device="cuda")).to(torch.bfloat16)
    wt[5] = 0.0
    wt[6, :128] = 0.25      # one sign only: the range holds zero too
    wt[7, :128] = -0.25
    for group in (32, 64, 128):
        codes, scales, z = quantize_w4(wt, group)
        d = dense(codes, scales, z)
        x = wt.double().view(V, -1, group)
        lo, hi = x.amin(2).clamp(max=0), x.amax(2).clamp(min=0)
        assert torch.equal(scales, ((hi - lo).float() / 15).to(torch.bfloat16))
        # half a step, and what rounding the scale (2^-8 of 15 steps) and the zero point to whole numbers takes from the ends
        step = scales.double()[:, :, None]
        off = (d.view(V, -1, group) - x).abs()
        assert (off <= step * (0.5 + 0.5 + 15 * 2.0 ** -8 + 1e-6)).all()
        inner = (x > lo[:, :, None] + 1.1 * step) & (x < hi[:, :, None] - 1.1 * step)
        assert (off[inner] <= (0.5 + 1e-4) * step.expand_as(off)[inner]).all()
        assert (d[5] == 0).all()
    h, nw = inputs(g, 4, K)
    codes, scales, z = quantize_w4(wt, 128)
    normed, logits = lm_head_w4(h, W4Weight.quantize(wt, 128), nw)
    check_logits(normed, dense(codes, scales, z), logits)


@pytest.mark.parametrize("B,V,params", [
    (1, 151936, (0.6, 0.95, 0.05, 20, 1.1, 0.5, 0.3)), (8, 50021, (0.8, 0.9, 0.0, 0, 1.2, 0.0, 0.0)),
    (40, 4096, (0.0, 1.0, 0.0, 0, 1.3, 0.0, 0.2)), (5, 1003, (0.7, 0.95, 0.1, 50, 1.15, 0.0, 0.0)),
    (300, 1000, (0.7, 0.95, 0.1, 50, 1.15, 0.0, 0.0))])
def test_sample_from_4_bit_weights(B, V, params):
    """lm_head_sample with such a weight draws what sample() draws from lm_head_w4's logits, step after step."""
    from qwen600_engine_b200.sampler import Sampler
    from qwen600_engine_b200.w4 import W4Weight, lm_head_w4
    codes, scales, z, g = plain_weight(V, 1024, 64, True, torch.bfloat16, seed=V)
    w = W4Weight.pack(codes, scales, z)
    T, topp, minp, k, rp, fp, pp = params
    fused, apart = (Sampler(T, topp, minp, k, rp, fp, pp, 64, 7, max_batch=B, vocab=V) for _ in range(2))
    for step in range(4):
        h, nw = inputs(g, B, 1024)
        tok = fused.lm_head_sample(h, w, nw)
        logits = lm_head_w4(h, w, nw)[1]
        assert torch.equal(fused.lm_head_logits(B), logits)
        want = apart.sample(logits)
        torch.cuda.synchronize()
        np.testing.assert_array_equal(tok.cpu().numpy(), want.cpu().numpy(), err_msg=f"step {step}")
    np.testing.assert_array_equal(fused.rng_state, apart.rng_state)
    # the same handle goes on with a bf16 weight
    wt = (0.02 * torch.randn((V, 1024), generator=g, device="cuda")).to(torch.bfloat16)
    tok = fused.lm_head_sample(h, wt, nw)
    want = apart.sample(fused.lm_head_logits(B).clone())
    assert torch.equal(tok, want)
    fused.free()
    apart.free()


def test_sample_on_a_stream_into_the_callers_buffer():
    from qwen600_engine_b200._lib import SamplerError
    from qwen600_engine_b200.sampler import Sampler
    from qwen600_engine_b200.w4 import W4Weight
    codes, scales, z, g = plain_weight(2003, 256, 32, True, torch.float16, seed=12)
    w = W4Weight.pack(codes, scales, z)
    a, b = (Sampler(0.8, 0.9, 0.0, 10, 1.1, 0.0, 0.0, 16, 3, max_batch=5, vocab=2003) for _ in range(2))
    side = torch.cuda.Stream()
    for _ in range(3):
        h, nw = inputs(g, 5, 256)
        want = a.lm_head_sample(h, w, nw)
        out = torch.full((7,), -5, dtype=torch.int32, device="cuda")
        side.wait_stream(torch.cuda.current_stream())
        got = b.lm_head_sample(h, w, nw, out=out, stream=side)
        del h, nw  # kept until the stream is done with them
        torch.cuda.synchronize()
        assert got is out and torch.equal(out[:5], want) and (out[5:] == -5).all()
    h, nw = inputs(g, 1, 256)
    assert b.lm_head_sample(h[0], w, nw).shape == (1,)  # one row without a batch dimension
    for bad in (out[:3], out.long(), out.cpu()):
        with pytest.raises(SamplerError, match="out must be"):
            b.lm_head_sample(torch.zeros((5, 256), dtype=torch.bfloat16, device="cuda"), w, out=bad)
    a.free()
    b.free()


def test_streams_and_graphs():
    from qwen600_engine_b200.w4 import W4Weight, lm_head_w4
    codes, scales, z, g = plain_weight(50021, 1024, 128, False, torch.bfloat16, seed=3)
    w = W4Weight.pack(codes, scales, z)
    rows = [inputs(g, b, 1024) for b in (1, 6)]
    want = [lm_head_w4(h, w, nw) for h, nw in rows]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = [lm_head_w4(h, w, nw, stream=s) for (h, nw), s in zip(rows, streams)]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    graphs, outs = [], []
    for h, nw in rows:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(lm_head_w4(h, w, nw))
        graphs.append(gr)
    for h, nw in rows:
        h.copy_(h.flip(1))
    want = [lm_head_w4(h, w, nw) for h, nw in rows]
    torch.cuda.synchronize()
    for gr, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            gr.replay()
            gr.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for gr in graphs:
        gr.reset()


def test_refused_on_the_gpu():
    from qwen600_engine_b200._lib import SamplerError
    from qwen600_engine_b200.sampler import Sampler
    from qwen600_engine_b200.w4 import W4Weight, lm_head_w4
    codes, scales, z, g = plain_weight(1000, 1024, 64, True, torch.bfloat16, seed=1)
    w = W4Weight.pack(codes, scales, z)
    h, nw = inputs(g, 2, 1024)
    with pytest.raises(SamplerError, match="columns"):
        lm_head_w4(h[:, :512].contiguous(), w)
    with pytest.raises(SamplerError, match="bf16"):
        lm_head_w4(h.float(), w)
    with pytest.raises(SamplerError, match="norm_weight has"):
        lm_head_w4(h, w, nw[:64].contiguous())
    with pytest.raises(SamplerError, match="group"):
        W4Weight.pack(codes, scales[:, :1].contiguous())
    assert lm_head_w4(h[:0], w)[1].shape == (0, 1000)
    s = Sampler(max_batch=1, vocab=1000)
    with pytest.raises(SamplerError, match="max_batch"):
        s.lm_head_sample(h, w, nw)
    s.free()
    s = Sampler(max_batch=2, vocab=999)
    with pytest.raises(SamplerError, match="vocabulary rows"):
        s.lm_head_sample(h, w, nw)
    s.free()


def test_rollout_and_learning_step():
    """The operators together: the 4-bit tail answers, its tokens are scored, and the losses over them take a step on
    the bf16 logits of the same rows; gradients against the formula."""
    from qwen600_engine_b200 import losses
    from qwen600_engine_b200.sampler import Sampler, lm_head
    from qwen600_engine_b200.w4 import W4Weight
    g = torch.Generator(device="cuda")
    g.manual_seed(77)
    B, V, K, steps = 6, 5003, 256, 4
    wt = (0.05 * torch.randn((V, K), generator=g, device="cuda")).to(torch.bfloat16)
    w = W4Weight.quantize(wt, 64)
    nw = torch.ones(K, dtype=torch.bfloat16, device="cuda")
    s = Sampler(1.0, 1.0, 0.0, 0, 1.0, 0.0, 0.0, 0, 5, max_batch=B, vocab=V)
    hs, toks, old = [], [], []
    for _ in range(steps):
        h = torch.randn((B, K), generator=g, device="cuda").to(torch.bfloat16)
        t = s.lm_head_sample(h, w, nw)
        old.append(losses.token_logprobs(s.lm_head_logits(B), t).logprobs)
        hs.append(h)
        toks.append(t)
    s.free()
    h = torch.stack(hs, 1).view(B * steps, K)           # sequence by sequence
    tok = torch.stack(toks, 1).reshape(-1).contiguous()
    old = torch.stack(old, 1).reshape(-1).contiguous()
    assert (old < 0).all() and torch.isfinite(old).all()
    logits = lm_head(h, wt, nw)[1]                      # the learner's weights are not rounded
    ref = losses.token_logprobs(logits, tok).logprobs
    adv = torch.randn((B * steps,), generator=g, device="cuda")
    r = losses.policy_loss(logits, tok, old, adv, ref_logprobs=ref, kl_coef=0.1)
    assert torch.equal(r.logprobs, ref)                 # the same rows score the same bits
    x = logits.double().requires_grad_(True)
    lp = torch.log_softmax(x, 1).gather(1, tok.long()[:, None])[:, 0]
    ratio = (lp - old.double()).exp()
    d = ref.double() - lp
    border = (((ratio - 0.8).abs() < 1e-4) | ((ratio - 1.2).abs() < 1e-4)).any()
    assert not border
    l = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv) + 0.1 * (d.exp() - d - 1)
    l.mean().backward()
    assert abs(float(r.loss) - float(l.mean())) < 1e-5
    # bf16 half a step, and log-probabilities good to 1e-5 in the coefficients
    off = (r.grad.double() - x.grad).abs()
    assert (off <= 2.0 ** -8 * x.grad.abs() + 2e-5 * adv.abs().max() / (B * steps)).all()
    offsets = torch.arange(0, B * steps + 1, steps, dtype=torch.int32, device="cuda")
    seq_ref = ref.view(B, steps).sum(1)
    p = losses.preference_loss(logits, tok, offsets, seq_ref, beta=0.2)
    assert abs(float(p.loss) - float(np.log(2.0))) < 1e-5  # the model is its own reference
    y = logits.double().requires_grad_(True)
    sl = torch.log_softmax(y, 1).gather(1, tok.long()[:, None])[:, 0].view(B, steps).sum(1) - seq_ref.double()
    (-torch.nn.functional.logsigmoid(0.2 * (sl[:3] - sl[3:]))).mean().backward()
    assert ((p.grad.double() - y.grad).abs() <= 2.0 ** -8 * y.grad.abs() + 1e-6).all()


def test_captured_sampling_outlives_a_larger_hidden_size():
    # the handle's buffers grow in between; the graph keeps the ones it was captured with
    from qwen600_engine_b200.sampler import Sampler
    from qwen600_engine_b200.w4 import W4Weight
    codes, scales, z, g = plain_weight(2003, 256, 64, True, torch.bfloat16, seed=21)
    small = W4Weight.pack(codes, scales, z)
    large = W4Weight.pack(*plain_weight(2003, 1024, 128, False, torch.float16, seed=22)[:3])
    a, b = (Sampler(0.8, 0.9, 0.0, 10, 1.1, 0.0, 0.0, 16, 3, max_batch=3, vocab=2003) for _ in range(2))
    h, nw = inputs(g, 3, 256)
    hl, nl = inputs(g, 3, 1024)
    want = [a.lm_head_sample(x, w, n) for x, w, n in
            [(h, small, nw), (h, small, nw), (hl, large, nl), (h, small, nw), (hl, large, nl)]]
    got = [b.lm_head_sample(h, small, nw)]
    out = torch.empty(3, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.lm_head_sample(h, small, nw, out=out)
    logits = b.lm_head_logits(3).data_ptr()
    for x in (None, (hl, large, nl), None, (hl, large, nl)):
        if x is None:
            graph.replay()
            got.append(out.clone())
        else:
            got.append(b.lm_head_sample(*x))
    torch.cuda.synchronize()
    assert b.lm_head_logits(3).data_ptr() == logits
    for i, j in zip(got, want):
        assert torch.equal(i, j)
    graph.reset()
    a.free()
    b.free()


@pytest.mark.parametrize("four_bits", [True, False])
def test_first_call_on_a_stream_beside_a_busy_default_stream(four_bits):
    """A handle's first call makes and clears its buffers; work queued on another stream must not delay the clear."""
    from qwen600_engine_b200.sampler import Sampler
    from qwen600_engine_b200.w4 import W4Weight
    V, K, B = 50021, 1024, 4
    codes, scales, z, g = plain_weight(V, K, 64, True, torch.bfloat16, seed=41)
    w = W4Weight.pack(codes, scales, z) if four_bits else (0.02 * torch.randn((V, K), generator=g, device="cuda")).to(torch.bfloat16)
    h, nw = inputs(g, B, K)
    a = torch.empty(1 << 30, dtype=torch.uint8, device="cuda")
    b = torch.empty_like(a)
    for trial in range(4):
        first, second = (Sampler(0.8, 0.9, 0.0, 20, 1.1, 0.0, 0.0, 16, 3 + trial, max_batch=B, vocab=V) for _ in range(2))
        want = [first.lm_head_sample(h, w, nw).clone() for _ in range(3)]
        side = torch.cuda.Stream()
        out = [torch.empty(B, dtype=torch.int32, device="cuda") for _ in range(3)]
        torch.cuda.synchronize()
        for _ in range(60):  # some 20 ms
            b.copy_(a)
        for o in out:
            second.lm_head_sample(h, w, nw, out=o, stream=side)
        torch.cuda.synchronize()
        for i, (o, t) in enumerate(zip(out, want)):
            assert torch.equal(o, t), f"trial {trial}, step {i}"
        first.free()
        second.free()


def test_a_failed_call_leaves_no_error_for_the_next():
    """Allocations that the device refuses (more than it has), then ordinary calls."""
    import ctypes as C
    from qwen600_engine_b200 import _lib
    from qwen600_engine_b200._lib import SamplerError
    from qwen600_engine_b200.sampler import Sampler, lm_head
    from qwen600_engine_b200.w4 import W4Weight, lm_head_w4
    codes, scales, z, g = plain_weight(1003, 256, 64, True, torch.bfloat16, seed=51)
    w = W4Weight.pack(codes, scales, z)
    h, nw = inputs(g, 2, 256)
    want = lm_head_w4(h, w, nw)

    def refused_bytes():
        p, handle = C.c_void_p(), C.create_string_buffer(64)
        assert _lib.lib.qs_ipc_alloc(1 << 45, C.byref(p), handle) < 0 and p.value is None

    def refused_handle():
        with pytest.raises(SamplerError):
            Sampler(max_batch=1 << 30, vocab=151936)

    s = Sampler(0.0, 1.0, 0.0, 0, 1.0, 0.0, 0.0, 0, 3, max_batch=2, vocab=1003)
    for refused in (refused_bytes, refused_handle):
        for call in (lambda: lm_head_w4(h, w, nw), lambda: W4Weight.pack(codes, scales, z),
                     lambda: lm_head(h, torch.zeros((8, 256), dtype=torch.bfloat16, device="cuda"), nw),
                     lambda: s.lm_head_sample(h, w, nw), lambda: s.sample(want[1])):
            refused()
            assert _lib.lib.qs_last_error()
            call()
    assert torch.equal(lm_head_w4(h, w, nw)[1], want[1])
    s.free()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_keeps_what_is_not_a_number(group):
    """A NaN or an infinity in a weight shows in its own rows' logits, and in no others."""
    from qwen600_engine_b200.w4 import W4Weight, lm_head_w4, quantize_w4
    g = torch.Generator(device="cuda")
    g.manual_seed(61)
    V, K = 300, 256
    wt = (0.02 * torch.randn((V, K), generator=g, device="cuda")).to(torch.bfloat16)
    h, nw = inputs(g, 3, K)
    want = lm_head_w4(h, W4Weight.quantize(wt, group), nw)[1]
    spoiled = {3: float("nan"), 40: float("inf"), 77: -float("inf"), 299: float("nan")}
    for r, v in spoiled.items():
        wt[r, (37 * r) % K] = v
    wt[120, :] = float("nan")
    codes, scales, z = quantize_w4(wt, group)
    assert int((~torch.isfinite(scales)).sum()) == 4 + K // group
    got = lm_head_w4(h, W4Weight.pack(codes, scales, z), nw)[1]
    bad = torch.zeros(V, dtype=torch.bool, device="cuda")
    bad[list(spoiled) + [120]] = True
    assert torch.isnan(got[:, bad]).all() and torch.equal(got[:, ~bad], want[:, ~bad])
