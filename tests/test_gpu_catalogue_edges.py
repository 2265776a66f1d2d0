"""GPU tests of the catalogue operators at the edges of what they take: empty batches before full ones, factors and scales near the ends
of their ranges, the tile forms of large batches.  U = 2^-24 is half a step of fp32 relative to the value, B = 2^-8 of bf16."""
import pytest

pytestmark = pytest.mark.gpu
U, B = 2.0 ** -24, 2.0 ** -8


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


@pytest.fixture(scope="module")
def sc(torch):
    from recommenders_amd import HipScorer
    return HipScorer(0)


def _gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("n,width", [(0, 5), (3, 0), (0, 0)])
def test_policy_batch_after_an_empty_one(torch, n, width):
    """A scorer whose first call with a mask and the batch's mean has no place takes full batches afterwards."""
    from recommenders_amd import HipScorer
    sc = HipScorer(0)
    empty = torch.zeros((n, width), device="cuda")
    p = sc.policy_loss(empty, empty, torch.ones(n, device="cuda"), mask=torch.ones((n, width), dtype=torch.bool, device="cuda"), reduction="batch")
    assert p.loss.shape == (n,) and (p.loss == 0).all() and p.d_logp.shape == (n, width)
    logp = torch.zeros((2, 3), device="cuda")
    mask = torch.tensor([[True, True, False], [True, False, False]], device="cuda")
    p = sc.policy_loss(logp, logp, torch.tensor([3.0, 6.0], device="cuda"), mask=mask, reduction="batch")
    assert p.loss.tolist() == [-2.0, -2.0] and p.d_logp.tolist() == [[-1.0, -1.0, 0.0], [-2.0, 0.0, 0.0]]
    sc.close()


@pytest.mark.parametrize("beta", [1e-30, 1e-25, 1e-10, 1.0, 1e25, 1e30])
def test_squared_preference_over_the_range_of_beta(torch, sc, beta):
    """d loss / dh times beta is 2 (h - 1/2) / beta, which fp32 holds where the factors 2 (h - 1/2) / beta^2 and beta leave it."""
    D = torch.tensor([[0.0], [1.0], [-3.0], [1e-3]], device="cuda")
    p = sc.preference_loss(D, torch.zeros_like(D), beta=beta, kind="squared")
    h = (beta * D.double()[:, 0])
    # h rounds to fp32 (and to a multiple of 2^-149), then a difference, a quotient and a product
    want = 2 * (h - 0.5) / beta
    tol = 8 * U * want.abs() + 2 * (U * h.abs() + 2.0 ** -149) / beta
    assert ((p.d_chosen.double()[:, 0] - want).abs() <= tol).all() and torch.equal(p.d_rejected, -p.d_chosen)


@pytest.mark.parametrize("up,down", [(118, 118), (124, 124), (126, 120)])
def test_logprob_of_4bit_rows_whose_scales_cancel(torch, sc, up, down):
    """Users near the top of fp32 and items as far below 1: scores are ordinary numbers, and so is every log-probability."""
    g = _gen(torch, up)
    X, V = torch.randn((5, 96), generator=g, device="cuda") * 0.3, torch.randn((70, 96), generator=g, device="cuda") * 0.3
    ids = torch.randint(0, 70, (5, 4), generator=g, device="cuda", dtype=torch.int32)
    xq, vq = sc.quantize_mxfp4(X * 2.0 ** up), sc.quantize_mxfp4(V * 2.0 ** -down)
    scale = 2.0 ** (down - up)
    logp, lse = sc.catalogue_logprob(xq, vq, ids, scale=scale)
    x, v = sc.dequantize_mxfp4(xq).double(), sc.dequantize_mxfp4(vq).double()
    z, room = scale * x @ v.t(), float((scale * x.abs() @ v.abs().t()).max())
    want = torch.logsumexp(z, 1)
    # exact products, at most 96 additions in fp32, and the roundings of scale, exponent (twice |z| and |lse|), v_exp_f32 and the sum of 70
    score = 100 * U * room
    e_lse = score + 6 * U * (float(z.abs().max()) + float(want.abs().max()) + 8) + 2.0 ** -21 + 99 * U
    assert float((lse.double() - want).abs().max()) <= e_lse
    assert float((logp.double() - (z.gather(1, ids.long()) - want[:, None])).abs().max()) <= score + 2 * e_lse


@pytest.mark.parametrize("n,items", [(513, 32800), (700, 24001), (1030, 16404)])
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("k", [33, 200])
def test_scores_of_a_large_batch(torch, sc, n, items, out, k):
    """Enough tiles of 32 x 32 for the form that keeps 128 or 256 items a wave; rows at 16-byte borders and others, widths that end inside a tile."""
    g = _gen(torch, n + k)
    X, V = torch.randn((n, k), generator=g, device="cuda"), torch.randn((items, k), generator=g, device="cuda") * 0.1
    ib, ub = torch.randn(items, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda")
    xq, vq = sc.quantize_mxfp4(X), sc.quantize_mxfp4(V)
    x, v = sc.dequantize_mxfp4(xq).double(), sc.dequantize_mxfp4(vq).double()
    ref = x @ v.t() + ib.double() + ub.double()[:, None]
    # k products (exact) and two bases: at most k + 2 additions in fp32, then one rounding to the output's type
    tol = (k + 2) * U * (x.abs() @ v.abs().t() + ib.double().abs() + ub.double().abs()[:, None]) + (B * (1 + 1e-3) * ref.abs() if out == "bfloat16" else 0) + 1e-30
    s = sc.score_mxfp4(xq, vq, ubase=ub, ibase=ib, dtype=getattr(torch, out))
    assert ((s.double() - ref).abs() <= tol).all()
    wide = torch.full((n, items + 5), 5.0, dtype=s.dtype, device="cuda")
    sc.score_mxfp4(xq, vq, ubase=ub, ibase=ib, out=wide[:, :items])
    assert torch.equal(wide[:, :items], s) and (wide[:, items:] == 5).all()
