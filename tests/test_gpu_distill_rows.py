"""Rows of the distillation whose logits are no distribution: loss and gradient
agree that they are none, whatever the teacher gives the list.  And batches of
nothing but rows that are left out, with their inputs written again at once."""
import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")
NAN = float("nan")


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("given", [-INF, -2000.0, -1.0])
@pytest.mark.parametrize("listed", [-INF, NAN, INF])
@pytest.mark.parametrize("V", [3, 40, 5003])
def test_no_distribution_and_a_list_of_nothing(dtype, given, listed, V):
    """Row 1: all unlisted tokens masked, and the listed ones masked, NaN or +inf.  Probabilities of the teacher that
    are 0 (or come out as 0: exp(-2000)) leave nothing that the loss sums, and still the row has no distribution."""
    from qwen600_engine_b200 import losses
    g = torch.Generator(device="cuda")
    g.manual_seed(V)
    x = torch.randn((3, V), generator=g, device="cuda").to(dtype)
    tok = torch.tensor([[0, V - 1]] * 3, dtype=torch.int32, device="cuda")
    lps = torch.full((3, 2), -1.0, device="cuda")
    clean = losses.distill_loss(x, tok, lps)
    x[1] = -INF
    x[1, V - 1] = listed
    lps[1] = given
    r = losses.distill_loss(x, tok, lps)
    assert r.loss.isnan() and r.row_losses[1].isnan() and r.grad[1].isnan().all()
    alone = losses.distill_loss(x, tok, lps, grad=False)
    assert alone.loss.isnan() and alone.row_losses[1].isnan()
    for i in (0, 2):
        assert torch.equal(r.row_losses[i], clean.row_losses[i]) and torch.equal(r.grad[i], clean.grad[i])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_distribution_and_a_list_of_nothing(dtype):
    """All unlisted tokens masked, the listed ones not: the loss sums nothing and the gradient is zero."""
    from qwen600_engine_b200 import losses
    x = torch.full((1, 40), -INF, device="cuda", dtype=dtype)
    x[0, :2] = 1.5
    tok = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    r = losses.distill_loss(x, tok, torch.full((1, 2), -INF, device="cuda"))
    assert float(r.loss) == 0 and not r.grad.any()


@pytest.mark.parametrize("N,V,k", [(1, 5, 1), (8, 4003, 20), (3000, 40, 256), (300, 3001, 256)])
def test_every_row_left_out_and_the_inputs_written_again(N, V, k):
    """The next writes on the stream come behind all of the call's reads."""
    from qwen600_engine_b200 import losses
    g = torch.Generator(device="cuda")
    g.manual_seed(N)
    x = torch.randn((N, V), generator=g, device="cuda")
    tok = torch.randint(0, V, (N, k), generator=g, device="cuda").int()
    lps = torch.full((N, k), -6.0, device="cuda")
    some = torch.rand((N,), generator=g, device="cuda") + 0.5
    want = losses.distill_loss(x, tok, lps, weights=some)
    w = torch.zeros((N,), device="cuda")
    tokens = tok.clone()
    for i in range(40):
        out = torch.full_like(x, 3.0)
        w.zero_()
        r = losses.distill_loss(x, tokens, lps, weights=w, out=out)
        w.copy_(some)
        tokens.fill_(-1)
        filler = torch.full((4 * N * k,), 7, dtype=torch.int32, device="cuda")  # where the call's workspace may have been
        tokens.copy_(tok)
        again = losses.distill_loss(x, tokens, lps, weights=w)
        assert float(r.loss) == 0 and not r.row_losses.any() and not out.any()
        assert torch.equal(again.grad, want.grad) and torch.equal(again.row_losses, want.row_losses)
        assert (filler == 7).all()
