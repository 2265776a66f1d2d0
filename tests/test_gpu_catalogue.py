"""GPU tests of the catalogue operators (recommenders_amd/catalogue.py) against plain implementations in 64 bits.

Tolerances are worst-case bounds, written beside each check.  U = 2^-24 is half a step of fp32 relative to the value, B = 2^-8 of bf16.
Split fp32 operands (two fp16 parts) are off by at most 2^-22 of a value or 2^-39 of the matrix's largest; the product leaves out
lo * lo, at most 2^-22 of a term: 3 * 2^-22 of sum |x v| a score beside the rounding of its sums."""
import math

import numpy as np
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


# ---------------------------------------------------------------- 4 bits
GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


def quantize_np(x):
    """Codes, scales and values by the definition, element by element in float64."""
    n, k = x.shape
    kb = (k + 31) // 32
    y = np.zeros((n, kb * 32))
    y[:, :k] = x
    y = y.reshape(n, kb, 32)
    codes, scales, vals = np.zeros(y.shape, np.uint8), np.zeros((n, kb), np.uint8), np.zeros(y.shape)
    for r in range(n):
        for b in range(kb):
            blk = y[r, b]
            if not np.isfinite(blk).all():
                scales[r, b], vals[r, b] = 255, np.nan
                continue
            top = np.abs(blk).max()
            e = max(math.frexp(top)[1] - 1 - 2, -127) if top > 0 else -127
            scales[r, b] = e + 127
            t = np.abs(blk) * 2.0 ** -e
            d = np.abs(t[:, None] - GRID[None, :])
            near = d.min(1, keepdims=True)
            tied = d == near
            even = np.where(tied[:, ::2].any(1), 2 * np.argmax(tied[:, ::2], 1), 2 * np.argmax(tied[:, 1::2], 1) + 1)
            codes[r, b] = even + 8 * np.signbit(blk)
            vals[r, b] = np.where(np.signbit(blk), -GRID[even], GRID[even]) * 2.0 ** e
    packed = codes.reshape(n, -1)
    return packed[:, ::2] | (packed[:, 1::2] << 4), scales, vals.reshape(n, -1)[:, :k]


def _awkward(rng, n, k):
    """Ties, borders, subnormals, the largest values, zero blocks, both zeros."""
    x = rng.normal(0, 1, (n, k))
    x[0] = np.resize(np.concatenate([GRID, -GRID, [.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7, 7.9, -.25, -2.5, -5, -7]]), k)
    if n > 1:
        x[1] = 0.0
        x[1, ::2] = -0.0
    if n > 2:
        x[2] = rng.normal(0, 1e-40, k)
    if n > 3:
        x[3] = rng.choice([3.4028234e38, -1.7e38, 1e30], k)
    if n > 4:
        x[4] = np.exp2(rng.integers(-140, 100, k).astype(float)) * 1.5
    return x


@pytest.mark.parametrize("n,k", [(1, 1), (5, 31), (7, 32), (9, 33), (6, 50), (33, 128), (5, 200), (6, 256), (6, 777)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_quantize_and_back_exact(torch, sc, n, k, dtype):
    x = torch.as_tensor(_awkward(np.random.default_rng(n * 1000 + k), n, k).astype(np.float32)).to(getattr(torch, dtype))
    codes, scales, vals = quantize_np(x.float().numpy().astype(np.float64))
    q = sc.quantize_mxfp4(x.cuda())
    np.testing.assert_array_equal(q.scales.cpu().numpy(), scales)
    np.testing.assert_array_equal(q.codes.cpu().numpy(), codes)
    back = sc.dequantize_mxfp4(q)
    np.testing.assert_array_equal(back.cpu().numpy(), vals.astype(np.float32))
    assert q.shape == (n, k) and back.shape == (n, k)


def test_quantize_nonfinite_blocks_and_strides(torch, sc):
    x = torch.randn((9, 100), generator=_gen(torch, 1), device="cuda")
    x[2, 40] = float("inf")
    x[3, 99] = float("nan")
    x[4, 0] = float("-inf")
    q = sc.quantize_mxfp4(x)
    s = q.scales.cpu().numpy()
    assert s[2, 1] == 255 and s[3, 3] == 255 and s[4, 0] == 255 and (s == 255).sum() == 3
    v = sc.dequantize_mxfp4(q).cpu().numpy()
    assert np.isnan(v[2, 32:64]).all() and np.isnan(v[3, 96:]).all() and np.isnan(v[4, :32]).all() and np.isnan(v).sum() == 32 + 4 + 32
    # the same values from a slice whose rows are neither aligned nor contiguous, from a transpose, and from one expanded row
    wide = torch.zeros((9, 203), device="cuda")
    wide[:, 1:101] = x
    for other in (wide[:, 1:101], x.t().contiguous().t()):
        w = sc.quantize_mxfp4(other)
        assert torch.equal(w.codes, q.codes) and torch.equal(w.scales, q.scales)
    e = sc.quantize_mxfp4(x[0:1].expand(5, 100))
    assert torch.equal(e.codes, q.codes[0:1].expand(5, -1))
    out = torch.full((9, 105), 7.0, device="cuda")
    sc.dequantize_mxfp4(q, out=out[:, :100])
    assert (out[:, 100:] == 7).all()
    assert sc.quantize_mxfp4(x[:0]).shape == (0, 100) and sc.dequantize_mxfp4(sc.quantize_mxfp4(x[:0])).shape == (0, 100)


@pytest.mark.parametrize("n,items,k", [(1, 1, 1), (1, 700, 128), (3, 65, 33), (31, 100, 50), (33, 257, 64), (70, 1000, 128), (65, 129, 200), (129, 500, 256),
                                       (200, 31, 100)])
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("bases", [0, 1, 2])
def test_scores_of_a_4bit_model(torch, sc, n, items, k, out, bases):
    g = _gen(torch, n + items + k)
    X, V = torch.randn((n, k), generator=g, device="cuda"), torch.randn((items, k), generator=g, device="cuda") * 0.1
    ib = torch.randn(items, generator=g, device="cuda") if bases else None
    ub = torch.randn(n, generator=g, device="cuda") if bases == 2 else None
    xq, vq = sc.quantize_mxfp4(X), sc.quantize_mxfp4(V)
    x, v = sc.dequantize_mxfp4(xq).double(), sc.dequantize_mxfp4(vq).double()
    ref, room = x @ v.t(), x.abs() @ v.abs().t()
    if ib is not None:
        ref, room = ref + ib.double(), room + ib.double().abs()
    if ub is not None:
        ref, room = ref + ub.double()[:, None], room + ub.double().abs()[:, None]
    wide = torch.full((n, items + 3), 5.0, dtype=getattr(torch, out), device="cuda")
    s = sc.score_mxfp4(xq, vq, ubase=ub, ibase=ib, out=wide[:, :items])
    # k products (exact) and two bases: at most k + 2 additions in fp32, then one rounding to the output's type
    tol = (k + 2) * U * room + (B * ref.abs() if out == "bfloat16" else 0) * (1 + 1e-3) + 1e-30
    assert ((s.double() - ref).abs() <= tol).all()
    assert (wide[:, items:] == 5).all()
    assert torch.equal(sc.score_mxfp4(xq, vq, ubase=ub, ibase=ib, dtype=getattr(torch, out)), s)


def test_scores_nan_blocks_stay_in_their_rows(torch, sc):
    g = _gen(torch, 3)
    X, V = torch.randn((40, 96), generator=g, device="cuda"), torch.randn((70, 96), generator=g, device="cuda")
    X[5, 3] = float("nan")
    V[11, 95] = float("inf")
    s = sc.score_mxfp4(sc.quantize_mxfp4(X), sc.quantize_mxfp4(V)).cpu().numpy()
    bad = np.isnan(s)
    assert bad[5].all() and bad[:, 11].all() and bad.sum() == 70 + 40 - 1


# ---------------------------------------------------------------- log-probabilities
def _case(torch, n, items, k, m, dtype, bias, seed, spread=0.4):
    g = _gen(torch, seed)
    dt = getattr(torch, dtype)
    X = (torch.randn((n, k), generator=g, device="cuda") * spread).to(dt)
    V = (torch.randn((items, k), generator=g, device="cuda") * spread).to(dt)
    b = torch.randn(items, generator=g, device="cuda") if bias else None
    ids = torch.randint(-1, items, (n, m), generator=g, device="cuda", dtype=torch.int32)
    dlogp = torch.randn((n, m), generator=g, device="cuda")
    return X, V, b, ids, dlogp


def _reference(torch, X, V, b, ids, dlogp, scale):
    """Forward and gradient in float64, with the sums of magnitudes that the bounds need."""
    x, v = X.double(), V.double()
    s, room = x @ v.t(), x.abs() @ v.abs().t()
    if b is not None:
        s, room = s + b.double(), room + b.double().abs().nan_to_num(posinf=0.0)
    z, room = scale * s, scale * room
    lse = torch.logsumexp(z, 1)
    held = ids >= 0
    at = ids.long().clamp(min=0)
    logp = torch.where(held, z.gather(1, at) - lse[:, None], 0.0) if ids.shape[1] else z[:, :0]
    g = torch.where(held, dlogp.double(), 0.0)
    G = g.sum(1)
    P = torch.where(torch.isfinite(lse)[:, None], torch.exp(z - lse[:, None]), 0.0)
    hot = torch.zeros_like(z).scatter_add_(1, at, g)
    hot_abs = torch.zeros_like(z).scatter_add_(1, at, g.abs())
    dz = hot - G[:, None] * P
    mass = G.abs()[:, None] * P
    return dict(z=z, room=room, lse=lse, logp=logp, dX=scale * dz @ v, dV=scale * dz.t() @ x, db=scale * dz.sum(0),
                pX=scale * mass @ v.abs(), pV=scale * mass.t() @ x.abs(), pb=scale * mass.sum(0),
                tX=scale * hot_abs @ v.abs(), tV=scale * hot_abs.t() @ x.abs(), tb=scale * hot_abs.sum(0), gabs=g.abs().sum(1))


def _bounds(r, items, n, k, m, dtype):
    """(score, lse, relative error of a probability): scores by operands (3 * 2^-22, split only) and at most 3 k additions of the
    products of the parts, plus the roundings of the scaling, the base and log2(e); lse adds the exponent's rounding (|z| and
    |lse| up to Z in units of 2^-24, twice), v_exp_f32 (2^-22) and at most items / 2 + 64 additions of positive numbers."""
    room, Z = float(r["room"].max()), float(r["z"].abs().nan_to_num(posinf=0.0).max()) + float(r["lse"].abs().nan_to_num(posinf=0.0).max()) + 32
    score = (3 * 2.0 ** -22 if dtype == "float32" else 0.0) * room + (3 * k + 4) * U * room
    lse = score + 6 * Z * U + 2.0 ** -21 + (items / 2 + 64) * U
    return score, lse, score + lse + 6 * Z * U + 2.0 ** -21


SIZES = [(1, 1, 1, 1), (1, 33, 5, 3), (3, 1000, 128, 7), (31, 31, 64, 1), (33, 129, 50, 4), (130, 700, 128, 20), (129, 257, 192, 2), (64, 1500, 200, 9),
         (260, 333, 256, 5), (5, 40, 100, 0)]


@pytest.mark.parametrize("n,items,k,m", SIZES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("bias,scale", [(False, 1.0), (True, 1.0), (True, 2.5)])
def test_logprob_and_gradient(torch, sc, n, items, k, m, dtype, bias, scale):
    X, V, b, ids, dlogp = _case(torch, n, items, k, m, dtype, bias, n * 7 + items)
    r = _reference(torch, X, V, b, ids, dlogp, scale)
    logp, lse = sc.catalogue_logprob(X, V, ids, ibase=b, scale=scale)
    score, e_lse, e_p = _bounds(r, items, n, k, m, dtype)
    assert float((lse.double() - r["lse"]).abs().max()) <= e_lse
    if m:
        assert float((logp.double() - r["logp"]).abs().max()) <= score + e_lse
    dX, dV, db = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b, scale=scale)
    assert dX.dtype == X.dtype and dV.dtype == V.dtype and (db is None) == (b is None)
    # the probabilities' part: their error, the split or the rounding of the probability and of the other operand (G x), and at most
    # 3 additions a term; the items' part: m (n m) additions and products in fp32; G itself m additions; the result one rounding
    half, low = (2 * 2.0 ** -22, U) if dtype == "float32" else (2 * B, B)
    # split probabilities also have an absolute step: 2^-39, against operands of at most max |v| (max |G x|)
    step = 2.0 ** -39 if dtype == "float32" else 0.0
    big = float(r["gabs"].max()) if n and m else 0.0
    grow = lambda terms: e_p + half + 3 * terms * U + m * U
    for name, got, ref, p, t, terms, other in (("dX", dX, r["dX"], r["pX"], r["tX"], items, V), ("dV", dV, r["dV"], r["pV"], r["tV"], n, X)):
        tol = grow(terms) * p + (n * m + 4) * U * t + (low + 2 * U) * ref.abs() + scale * big * float(other.float().abs().max()) * terms * step * 4 + 1e-30
        # cancellation in G: |G| may be far below the sum of its parts, each addition of which rounds
        tol = tol + m * U * scale * big * float(other.float().abs().max()) * (1 if name == "dX" else n)
        assert ((got.double() - ref).abs() <= tol).all(), (name, float(((got.double() - ref).abs() / tol).max()))
    if db is not None:
        tol = grow(n) * r["pb"] + (n * m + 4) * U * r["tb"] + 3 * U * r["db"].abs() + scale * big * (n * step * 4 + m * U * n) + 1e-30
        assert ((db.double() - r["db"]).abs() <= tol).all()
    again = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b, scale=scale)
    assert all(a is None and c is None or torch.equal(a, c) for a, c in zip((dX, dV, db), again))


@pytest.mark.parametrize("n,items,k,m", [(600, 150, 40, 40), (700, 3, 128, 30), (300, 70001, 32, 20), (90, 66000, 200, 3), (200, 40000, 128, 64)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logprob_gradient_of_items_that_everybody_names(torch, sc, n, items, k, m, dtype):
    """More places than one pass over them holds, one item in half of them, catalogues of few and of many rows."""
    X, V, b, ids, dlogp = _case(torch, n, items, k, m, dtype, True, 21, spread=0.2)
    g = _gen(torch, 22)
    pick = torch.rand((n, m), generator=g, device="cuda")
    ids = torch.where(pick < 0.5, torch.full_like(ids, items // 2), torch.where(pick < 0.6, torch.full_like(ids, items - 1), ids))
    dlogp /= n
    _, lse = sc.catalogue_logprob(X, V, ids, ibase=b)
    r = _reference(torch, X, V, b, ids, dlogp, 1.0)
    got = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b)
    # the norm of the error: rounding of the result, operands and probabilities in 16 bits (their errors are independent and add up
    # like at most sqrt(3) steps), or 22 bits and up to n m additions of one item's places, errors again independent
    bound = 3 * B if dtype == "bfloat16" else 8 * 2.0 ** -22 + math.sqrt(n * m) * U
    for a, ref in zip(got, (r["dX"], r["dV"], r["db"])):
        assert float((a.double() - ref).norm() / ref.norm()) <= (bound if a.dtype != torch.float32 or dtype == "float32" else 2.0 ** -18)
    again = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.parametrize("n,items,k,m", [(700, 5000, 33, 100), (4100, 2048, 64, 16), (1100, 9000, 130, 64), (70000, 2111, 32, 1)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logprob_gradient_of_many_places(torch, sc, n, items, k, m, dtype):
    """Places enough to be dealt into buckets first: one item in half of them, empty ones, catalogues of 16 to 71 blocks of 128 rows."""
    X, V, b, ids, dlogp = _case(torch, n, items, k, m, dtype, True, 21, spread=0.2)
    g = _gen(torch, 22)
    pick = torch.rand((n, m), generator=g, device="cuda")
    ids = torch.where(pick < 0.5, torch.full_like(ids, items // 2), torch.where(pick < 0.6, torch.full_like(ids, items - 1), ids))
    dlogp /= n
    _, lse = sc.catalogue_logprob(X, V, ids, ibase=b)
    r = _reference(torch, X, V, b, ids, dlogp, 1.0)
    got = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b)
    # the norm of the error: rounding of the result, operands and probabilities in 16 bits (their errors are independent and add up
    # like at most sqrt(3) steps), or 22 bits and up to n m additions of one item's places, errors again independent
    bound = 3 * B if dtype == "bfloat16" else 8 * 2.0 ** -22 + math.sqrt(n * m) * U
    for a, ref in zip(got, (r["dX"], r["dV"], r["db"])):
        assert float((a.double() - ref).norm() / ref.norm()) <= (bound if a.dtype != torch.float32 or dtype == "float32" else 2.0 ** -18 + math.sqrt(n * m) * U)
    again = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logprob_parts_that_are_not_wanted(torch, sc, dtype):
    X, V, b, ids, dlogp = _case(torch, 50, 300, 70, 3, dtype, True, 5)
    _, lse = sc.catalogue_logprob(X, V, ids, ibase=b)
    whole = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b)
    for at, name in enumerate(("X", "V", "ibase")):
        part = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b, want=(name,))
        assert [p is None for p in part] == [i != at for i in range(3)]
        assert torch.equal(part[at], whole[at])
    assert sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b, want=()) == (None, None, None)


def test_logprob_gradient_against_differences(torch, sc):
    X, V, b, ids, dlogp = _case(torch, 20, 150, 40, 4, "float32", True, 8, spread=0.3)
    _, lse = sc.catalogue_logprob(X, V, ids, ibase=b)
    grads = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b)
    held = ids >= 0

    def value(X, V, b):
        logp, _ = sc.catalogue_logprob(X, V, ids, ibase=b)
        return float((logp.double() * dlogp.double())[held].sum())

    h = 2.0 ** -6
    for at in range(3):
        args = [X, V, b]
        d = torch.randn(args[at].shape, generator=_gen(torch, at), device="cuda")
        d /= float(d.abs().max())
        up, down = list(args), list(args)
        up[at], down[at] = args[at] + h * d, args[at] - h * d
        slope = (value(*up) - value(*down)) / (2 * h)
        want = float((grads[at].double() * d.double()).sum())
        # the third derivative of a log-sum-exp along a line is at most the cube of the range of the scores' slopes
        reach = 2 * float((d.double() @ V.double().t() if at == 0 else X.double() @ d.double().t() if at == 1 else d.double()).abs().max())
        weight = float(dlogp.abs().sum())
        tol = weight * (reach ** 3 * h * h / 6 + 4e-6 / h)                # 4e-6: error of a log-probability here (|logp| < 16, 2^-22 steps)
        assert abs(slope - want) <= tol, (at, slope, want, tol)


def test_logprob_masks_and_awkward_places(torch, sc):
    X, V, b, ids, dlogp = _case(torch, 70, 200, 64, 6, "float32", True, 11)
    b[10:50] = float("-inf")                      # taken out of the catalogue
    b[60] = torch.finfo(torch.float32).min        # as good as out
    ids[0] = -1                                   # a slate without an item
    ids[1] = 7                                    # the same item six times
    ids[2, 0] = 12                                # an item that is out
    ids[3, 1] = -2147483648
    dlogp[0] = float("nan")                       # nothing flows through empty places, whatever stands there
    dlogp[3, 1] = float("inf")
    clean = dlogp.clone()
    clean[ids < 0] = 0
    logp, lse = sc.catalogue_logprob(X, V, ids, ibase=b)
    r = _reference(torch, X, V, b, ids, clean, 1.0)
    assert (logp[0] == 0).all() and logp[2, 0] == float("-inf") and logp[3, 1] == 0
    fin = torch.isfinite(r["logp"])
    assert torch.equal(torch.isfinite(logp), fin)
    assert float((logp.double() - r["logp"])[fin].abs().max()) < 1e-4 and float((lse.double() - r["lse"]).abs().max()) < 1e-4
    dX, dV, db = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b)
    for got, ref in ((dX, r["dX"]), (dV, r["dV"]), (db, r["db"])):
        assert float((got.double() - ref).abs().max()) < 1e-4 * max(1.0, float(ref.abs().max()))
    assert (dX[0] == 0).all()
    # every item out: no probabilities, -inf, and a gradient through the named items alone
    out = torch.full_like(b, torch.finfo(torch.float32).min)
    _, lse = sc.catalogue_logprob(X, V, ids, ibase=out, scale=2.0)
    assert (lse == float("-inf")).all()
    out = torch.full_like(b, float("-inf"))
    logp, lse = sc.catalogue_logprob(X, V, ids, ibase=out)
    assert (lse == float("-inf")).all() and (logp[ids >= 0] == float("-inf")).all() and (logp[ids < 0] == 0).all()
    dX, dV, db = sc.catalogue_logprob_backward(X, V, ids, lse, clean, ibase=out)
    assert all(torch.isfinite(t).all() for t in (dX, dV, db))
    want = torch.zeros_like(b.double()).index_add_(0, ids[ids >= 0].long(), clean[ids >= 0].double())
    assert float((db.double() - want).abs().max()) < 1e-4
    # an id behind the catalogue is seen in the result
    ids[5, 2] = 200
    logp, _ = sc.catalogue_logprob(X, V, ids, ibase=b)
    assert torch.isnan(logp[5, 2]) and torch.isnan(logp).sum() == 1


@pytest.mark.parametrize("dtype,k", [("float32", 50), ("float32", 128), ("bfloat16", 64), ("bfloat16", 61)])
def test_a_padded_batch(torch, sc, dtype, k):
    """Users without an item, with NaN and infinities in their rows, gradients and lse: the others' results are those of a batch without them."""
    X, V, b, ids, dlogp = _case(torch, 90, 300, k, 4, dtype, True, 31)
    ids.clamp_(min=0)
    real = torch.ones(90, dtype=torch.bool, device="cuda")
    real[5::7] = False
    want = sc.catalogue_logprob(X[real], V, ids[real], ibase=b)
    Xp, ip, dp = X.clone(), ids.clone(), dlogp.clone()
    Xp[~real], ip[~real], dp[~real] = float("nan"), -1, float("nan")
    Xp[5] = float("inf")
    logp, lse = sc.catalogue_logprob(Xp, V, ip, ibase=b)
    assert (logp[~real] == 0).all() and torch.isnan(lse[~real]).all()
    score, e_lse, _ = _bounds(_reference(torch, X[real], V, b, ids[real], dlogp[real], 1.0), 300, 90, k, 4, dtype)
    assert float((logp[real] - want[0]).abs().max()) <= 2 * (score + e_lse) and float((lse[real] - want[1]).abs().max()) <= 2 * e_lse
    dX, dV, db = sc.catalogue_logprob_backward(Xp, V, ip, lse, dp, ibase=b)
    r = _reference(torch, X[real], V, b, ids[real], dlogp[real], 1.0)
    assert (dX[~real] == 0).all()
    for got, ref in ((dX[real], r["dX"]), (dV, r["dV"]), (db, r["db"])):
        # the norm of the error: a step of 16 bits for operand, probability and result, or 22 bits and the sums' rounding
        bound = 3 * B if got.dtype == torch.bfloat16 else 2.0 ** -18
        assert float((got.double() - ref).norm() / ref.norm()) <= bound


def test_logprob_nan_stays_in_its_row(torch, sc):
    X, V, b, ids, dlogp = _case(torch, 70, 200, 64, 3, "float32", False, 12)
    ids.clamp_(min=0)
    X[9, 1] = float("nan")
    logp, lse = sc.catalogue_logprob(X, V, ids)
    bad = torch.isnan(lse)
    assert bad[9] and bad.sum() == 1 and torch.isnan(logp[9]).all() and torch.isnan(logp).sum() == 3


@pytest.mark.parametrize("spread", [1e-20, 1e-3, 1e4])
def test_logprob_magnitudes(torch, sc, spread):
    """fp32 operands far from 1: the scaling of the split follows the largest magnitude."""
    X, V, _, ids, dlogp = _case(torch, 40, 100, 50, 2, "float32", False, 13)
    big = X * (1 / spread)
    logp, lse = sc.catalogue_logprob(big, V * spread, ids)
    r = _reference(torch, big, V * spread, None, ids, dlogp, 1.0)
    score, e_lse, _ = _bounds(r, 100, 40, 50, 2, "float32")
    assert float((lse.double() - r["lse"]).abs().max()) <= e_lse and float((logp.double() - r["logp"]).abs().max()) <= score + e_lse
    dX, dV, _ = sc.catalogue_logprob_backward(big, V * spread, ids, lse, dlogp)
    assert float(((dX.double() - r["dX"]) / spread).abs().max()) < 1e-4 and float(((dV.double() - r["dV"]) * spread).abs().max()) < 1e-3
    zero = torch.zeros_like(V)
    logp, lse = sc.catalogue_logprob(X, zero, ids)
    assert float((lse - math.log(100)).abs().max()) <= 4 * U * 8
    dX, dV, _ = sc.catalogue_logprob_backward(X, zero, ids, lse, dlogp)
    assert (dX == 0).all() and torch.isfinite(dV).all()


def test_logprob_strides_and_empty_batches(torch, sc):
    X, V, b, ids, dlogp = _case(torch, 45, 120, 37, 5, "bfloat16", True, 14)
    want = sc.catalogue_logprob(X, V, ids, ibase=b)
    grads = sc.catalogue_logprob_backward(X, V, ids, want[1], dlogp, ibase=b)
    Xw, Vw = torch.full((45, 41), 9, dtype=X.dtype, device="cuda"), torch.full((120, 40), 9, dtype=X.dtype, device="cuda")
    iw, dw = torch.full((45, 9), 3, dtype=torch.int32, device="cuda"), torch.full((45, 11), 3.0, device="cuda")
    Xw[:, 3:40], Vw[:, 1:38], iw[:, 2:7], dw[:, 1:6] = X, V, ids, dlogp
    args = (Xw[:, 3:40], Vw[:, 1:38], iw[:, 2:7])
    assert all(torch.equal(a, c) for a, c in zip(sc.catalogue_logprob(*args, ibase=b), want))
    assert all(torch.equal(a, c) for a, c in zip(sc.catalogue_logprob_backward(*args, want[1], dw[:, 1:6], ibase=b), grads))
    # rows of whole pieces (read as they lie) and the same rows at an odd place (put in order first), in turn
    X, V, b, ids, dlogp = _case(torch, 150, 300, 64, 5, "bfloat16", True, 24)
    Xo, Vo = torch.zeros((150, 67), dtype=X.dtype, device="cuda"), torch.zeros((300, 65), dtype=X.dtype, device="cuda")
    Xo[:, 3:], Vo[:, 1:] = X, V
    want = sc.catalogue_logprob(X, V, ids, ibase=b)
    grads = sc.catalogue_logprob_backward(X, V, ids, want[1], dlogp, ibase=b)
    for args in ((Xo[:, 3:], Vo[:, 1:], ids), (X, Vo[:, 1:], ids), (Xo[:, 3:], V, ids), (X, V, ids)):
        assert all(torch.equal(a, c) for a, c in zip(sc.catalogue_logprob(*args, ibase=b), want))
        assert all(torch.equal(a, c) for a, c in zip(sc.catalogue_logprob_backward(*args, want[1], dlogp, ibase=b), grads))
    X, V, b, ids, _ = _case(torch, 45, 120, 37, 5, "bfloat16", True, 14)
    want = sc.catalogue_logprob(X, V, ids, ibase=b)
    # one user repeated by a broadcast, ids of another order
    e = sc.catalogue_logprob(X[:1].expand(45, 37), V, ids.t().contiguous().t(), ibase=b)
    assert float((e[1] - want[1][0]).abs().max()) == 0
    logp, lse = sc.catalogue_logprob(X[:0], V, ids[:0], ibase=b)
    assert logp.shape == (0, 5) and lse.shape == (0,)
    dX, dV, db = sc.catalogue_logprob_backward(X[:0], V, ids[:0], lse, dlogp[:0], ibase=b)
    assert dX.shape == (0, 37) and (dV == 0).all() and (db == 0).all()


@pytest.mark.parametrize("n,items,k,m", [(1, 1, 1, 1), (3, 100, 33, 4), (130, 1000, 128, 5), (40, 260, 200, 3), (65, 90, 256, 2)])
def test_logprob_of_a_4bit_model(torch, sc, n, items, k, m):
    X, V, b, ids, dlogp = _case(torch, n, items, k, m, "float32", True, 15 + n)
    xq, vq = sc.quantize_mxfp4(X), sc.quantize_mxfp4(V)
    x, v = sc.dequantize_mxfp4(xq), sc.dequantize_mxfp4(vq)
    r = _reference(torch, x, v, b, ids, dlogp, 1.5)
    logp, lse = sc.catalogue_logprob(xq, vq, ids, ibase=b, scale=1.5)
    score, e_lse, _ = _bounds(r, items, n, k, m, "bfloat16")               # products are exact, as those of bf16 operands
    assert float((lse.double() - r["lse"]).abs().max()) <= e_lse and float((logp.double() - r["logp"]).abs().max()) <= score + e_lse
    with pytest.raises(TypeError, match="no gradient"):
        sc.catalogue_logprob_backward(xq, vq, ids, lse, dlogp, ibase=b)


# ---------------------------------------------------------------- preference
def _preference_ref(torch, c, r, rc, rr, mc, mr, beta, kind, eps, margin, average, w):
    c, r = c.double(), r.double()
    x, y = (c, r) if rc is None else (c - rc.double(), r - rr.double())
    mc = torch.ones_like(c, dtype=torch.bool) if mc is None else mc.bool()
    mr = torch.ones_like(r, dtype=torch.bool) if mr is None else mr.bool()
    x, y = torch.where(mc, x, 0.0), torch.where(mr, y, 0.0)
    nc = mc.sum(1).clamp(min=1).double() if average else torch.ones(len(c), device=c.device).double()
    nr = mr.sum(1).clamp(min=1).double() if average else torch.ones(len(c), device=c.device).double()
    h = beta * (x.sum(1) / nc - y.sum(1) / nr) - margin
    if kind == "logistic":
        sp = torch.nn.functional.softplus
        loss, slope = (1 - eps) * sp(-h) + eps * sp(h), eps * torch.sigmoid(h) - (1 - eps) * torch.sigmoid(-h)
    elif kind == "hinge":
        loss, slope = (1 - h).clamp(min=0), -(h < 1).double()
    else:
        loss, slope = ((h - .5) / beta) ** 2, 2 * (h - .5) / beta ** 2
    g = slope * beta * (1.0 if w is None else w.double())
    return loss, h, mc * (g / nc)[:, None], mr * (-g / nr)[:, None]


@pytest.mark.parametrize("n,lc,lr", [(1, 1, 1), (3, 7, 0), (5, 0, 0), (2, 64, 65), (300, 10, 10), (70, 257, 1000), (4, 5000, 3)])
@pytest.mark.parametrize("kind,eps,margin,average,masked,ref", [("logistic", 0, 0, False, False, False), ("logistic", 0.1, 0.3, True, True, True),
                                                                ("hinge", 0, 0.5, False, True, True), ("squared", 0, 0, True, True, False)])
def test_preference_loss(torch, sc, n, lc, lr, kind, eps, margin, average, masked, ref):
    g = _gen(torch, n + lc)
    rand = lambda w: -torch.rand((n, w), generator=g, device="cuda") * 9 - 1
    both = torch.full((n, lc + lr + 3), float("nan"), device="cuda")                 # slates as columns of one tensor
    both[:, :lc], both[:, lc:lc + lr] = rand(lc), rand(lr)
    c, r = both[:, :lc], both[:, lc:lc + lr]
    rc, rr = (c + torch.randn((n, lc), generator=g, device="cuda"), r + torch.randn((n, lr), generator=g, device="cuda")) if ref else (None, None)
    mc = torch.rand((n, lc), generator=g, device="cuda") < 0.6 if masked else None
    mr = torch.rand((n, lr), generator=g, device="cuda") < 0.6 if masked else None
    if masked and n > 1:
        mc[1] = False                                                                # a slate without an item
        c[mc == 0] = float("nan")                                                    # nothing behind the mask counts
        r[mr == 0] = float("inf")
    w = torch.rand(n, generator=g, device="cuda") if average else None
    beta = 0.1
    got = sc.preference_loss(c, r, rc, rr, mc, mr, beta=beta, kind=kind, label_smoothing=eps, margin=margin, average=average, weight=w)
    want = _preference_ref(torch, c, r, rc, rr, mc, mr, beta, kind, eps, margin, average, w)
    # sums in fp64: h rounds once; the slope moves by at most 2 / beta^2 of that and a handful of fp32 operations
    eh = U * want[1].abs() + 1e-12
    steep = {"logistic": 1.0, "hinge": 1.0, "squared": 2 / beta ** 2 * float((want[1] - .5).abs().max() + 1)}[kind]
    assert ((got.h.double() - want[1]).abs() <= eh).all()
    assert ((got.loss.double() - want[0]).abs() <= 16 * U * (want[0].abs() + 1) * (1 if kind != "squared" else steep) + steep * eh).all()
    clear = ((want[1] - 1).abs() > 1e-5) if kind == "hinge" else torch.ones_like(want[1], dtype=torch.bool)
    top = float((w if w is not None else torch.ones(1)).abs().max())
    for a, b in ((got.d_chosen, want[2]), (got.d_rejected, want[3])):
        tol = (16 * U * (b.abs() + beta * top) + 2 / beta ** 2 * beta * top * eh[:, None] * (1 if kind == "squared" else beta ** 2)) * (1 + 0 * b)
        if kind == "squared":
            tol = tol + 16 * U * b.abs() + 2 / beta * top * U
        assert ((a.double() - b).abs() <= tol)[clear].all()
        assert (a[b == 0] == 0).all()


def test_preference_extremes_and_differences(torch, sc):
    one = lambda *v: torch.tensor(v, device="cuda").reshape(-1, 1)
    c, r = one(0.0, -1e4, 300.0, float("inf"), float("nan")), one(-1e4, 0.0, 0.0, 0.0, 0.0)
    p = sc.preference_loss(c, r, beta=1.0)
    assert p.loss[0] == 0 and p.loss[1] == 1e4 and 0 <= p.loss[2] < 1e-30 and p.loss[3] == 0 and torch.isnan(p.loss[4])
    assert p.d_chosen[0] == 0 and p.d_chosen[1] == -1 and p.d_rejected[1] == 1 and p.d_chosen[3] == 0 and torch.isnan(p.d_chosen[4])
    # BPR's criterion: slates of one item
    g = _gen(torch, 2)
    c, r = torch.randn((50, 1), generator=g, device="cuda"), torch.randn((50, 1), generator=g, device="cuda")
    p = sc.preference_loss(c, r, beta=1.0)
    want = -torch.nn.functional.logsigmoid((c - r).double()[:, 0])
    assert float((p.loss.double() - want).abs().max()) <= 16 * U * float(want.max() + 1)
    # differences along a random direction, for every kind
    c, r = torch.randn((30, 6), generator=g, device="cuda"), torch.randn((30, 4), generator=g, device="cuda")
    dc, dr = torch.randn((30, 6), generator=g, device="cuda"), torch.randn((30, 4), generator=g, device="cuda")
    h = 2.0 ** -6
    for kind, eps in (("logistic", 0.2), ("squared", 0.0), ("hinge", 0.0)):
        kw = dict(beta=0.7, kind=kind, label_smoothing=eps, average=True)
        p = sc.preference_loss(c, r, **kw)
        slope = (sc.preference_loss(c + h * dc, r + h * dr, **kw).loss.double() - sc.preference_loss(c - h * dc, r - h * dr, **kw).loss.double()) / (2 * h)
        want = (p.d_chosen.double() * dc).sum(1) + (p.d_rejected.double() * dr).sum(1)
        reach = 0.7 * ((dc.double().mean(1)) - dr.double().mean(1)).abs()
        smooth = (p.h.double() - 1).abs() > 2 * h * reach if kind == "hinge" else torch.ones_like(p.h, dtype=torch.bool)
        # third derivative of the logistic loss in h: at most 0.1; the others have none.  fp32 losses: 16 U (loss + 1)
        tol = 0.1 * reach ** 3 * h * h / 6 + 32 * U * (p.loss.double() + 4) * (1 if kind != "squared" else 10) / h
        assert ((slope - want).abs() <= tol)[smooth].all()


# ---------------------------------------------------------------- policy
def _policy_ref(torch, logp, old, A, ref, mask, lo, hi, coef, reduction, w):
    mask = torch.ones_like(logp, dtype=torch.bool) if mask is None else mask.bool()
    d32 = logp - old                                                                 # the clip test is made on the fp32 difference
    A = A[:, None]
    over = mask & (A > 0) & (d32 > torch.tensor(math.log1p(hi), dtype=torch.float32))
    under = mask & (A < 0) & (d32 < torch.tensor(math.log1p(-lo), dtype=torch.float32))
    ratio = torch.exp(logp.double() - old.double())
    A = A.double()
    term = -A * torch.where(over, 1 + hi, torch.where(under, 1 - lo, ratio))
    grad = torch.where(over | under, 0.0, -A * ratio)
    kl = torch.zeros_like(term)
    if ref is not None:
        q = ref.double() - logp.double()
        kl = torch.expm1(q) - q
        term, grad = term + coef * kl, grad - coef * torch.expm1(q)
    count = mask.sum(1).double()
    c = {"sum": torch.ones_like(count), "row": 1 / count.clamp(min=1), "batch": (1 / count.sum().clamp(min=1)).expand_as(count)}[reduction]
    if w is not None:
        c = c * w.double()
    zero = lambda t: torch.where(mask, t, 0.0)
    return (zero(term).sum(1) * c, zero(kl).sum(1) / count.clamp(min=1), (over | under).sum(1).int(), zero(grad) * c[:, None],
            zero(term.abs()).sum(1) * c.abs(), zero(kl + 0 * term).sum(1) / count.clamp(min=1))


@pytest.mark.parametrize("n,width", [(1, 1), (2, 0), (3, 7), (300, 10), (5, 64), (70, 257), (2, 5000), (1100, 3)])
@pytest.mark.parametrize("reduction,masked,ref,weighted", [("sum", False, False, False), ("row", True, True, False), ("batch", True, True, True),
                                                           ("batch", False, False, True), ("row", False, True, True)])
def test_policy_loss(torch, sc, n, width, reduction, masked, ref, weighted):
    g = _gen(torch, n + width)
    randn = lambda: torch.randn((n, width), generator=g, device="cuda")
    logp = -torch.rand((n, width), generator=g, device="cuda") * 5 - 1
    old, rf = logp + 0.3 * randn(), logp + 0.5 * randn() if ref else None
    A = torch.randn(n, generator=g, device="cuda")
    if n > 2:
        A[2] = 0.0
    mask = torch.rand((n, width), generator=g, device="cuda") < 0.7 if masked else None
    w = torch.rand(n, generator=g, device="cuda") if weighted else None
    if masked and n > 1:
        mask[1] = False
        logp[mask == 0] = float("nan")
    got = sc.policy_loss(logp, old, A, ref_logp=rf, mask=mask, clip_low=0.2, clip_high=0.3, kl_coef=0.1 if ref else 0.0, reduction=reduction, weight=w)
    loss, kl, clipped, d, mag, _ = _policy_ref(torch, torch.nan_to_num(logp), old, A, rf, mask, 0.2, 0.3, 0.1 if ref else 0.0, reduction, w)
    assert torch.equal(got.clipped, clipped)
    # a difference of log-probabilities rounds by at most U * 8 here, exp and expm1 by 4 U: 16 U of a term, then one rounding each
    assert ((got.loss.double() - loss).abs() <= 24 * U * mag + 1e-30).all()
    c = d.abs() + 0.2 * (got.d_logp.double().abs() + d.abs())
    big = float(A.abs().max()) + 1
    unit = {"sum": 1.0, "row": 1.0, "batch": 1.0}[reduction]
    scale = (mag.clamp(min=0) * 0 + unit)[:, None] * (w.double()[:, None] if w is not None else 1.0)
    if reduction == "row":
        scale = scale / (mask.sum(1) if mask is not None else torch.full((n,), max(width, 1), device="cuda")).clamp(min=1).double()[:, None]
    elif reduction == "batch":
        scale = scale / max(1, int(mask.sum()) if mask is not None else n * width)
    assert ((got.d_logp.double() - d).abs() <= 24 * U * (c + 2 * big * scale) + 1e-30).all()
    if mask is not None:
        assert (got.d_logp[~mask] == 0).all()
    if ref:
        # kl = q^2 / 2 + ...: q rounds by at most 8 U of the log-probabilities' size where they are not within a factor of two
        assert ((got.kl.double() - kl).abs() <= 1e-5 * kl + 1e-9).all()
    else:
        assert got.kl is None


def test_policy_borders_and_differences(torch, sc):
    # exactly at the border is not clipped; a step beyond is
    hi, lo = np.float32(math.log1p(0.25)), np.float32(math.log1p(-0.25))
    d = torch.tensor([[hi, np.nextafter(hi, np.float32(1)), lo, np.nextafter(lo, np.float32(-1)), 0.0]], device="cuda")
    zero = torch.zeros_like(d)
    up = sc.policy_loss(d, zero, torch.ones(1, device="cuda"), clip_low=0.25, clip_high=0.25, reduction="sum")
    down = sc.policy_loss(d, zero, -torch.ones(1, device="cuda"), clip_low=0.25, clip_high=0.25, reduction="sum")
    assert up.clipped[0] == 1 and (up.d_logp[0] == 0).tolist() == [False, True, False, False, False]
    assert down.clipped[0] == 1 and (down.d_logp[0] == 0).tolist() == [False, False, False, True, False]
    # small KL terms do not cancel: exp(q) - q - 1 = q^2 / 2 (1 + q / 3 + ...)
    q = torch.tensor([[1e-3, -1e-3, 1e-4, 1e-5, 0.0, 0.4999, 0.5001, -3.0, 5.0]], device="cuda")
    for i in range(q.shape[1]):
        got = float(sc.policy_loss(torch.zeros((1, 1), device="cuda"), torch.zeros((1, 1), device="cuda"), torch.zeros(1, device="cuda"),
                                   ref_logp=q[:, i:i + 1], kl_coef=1.0).kl[0])
        x = float(q[0, i].double())
        want = x * x / 2 + x ** 3 / 6 + x ** 4 / 24 if abs(x) < 0.01 else math.expm1(x) - x
        assert abs(got - want) <= 8 * U * want + (2 * U * abs(x) if abs(x) >= 0.5 else 0)
    # differences
    g = _gen(torch, 4)
    logp = -torch.rand((20, 6), generator=g, device="cuda") * 4
    old, ref = logp + 0.3 * torch.randn((20, 6), generator=g, device="cuda"), logp + 0.3 * torch.randn((20, 6), generator=g, device="cuda")
    A, dirn = torch.randn(20, generator=g, device="cuda"), torch.randn((20, 6), generator=g, device="cuda").clamp(-1, 1)
    kw = dict(ref_logp=ref, kl_coef=0.2, clip_low=0.2, clip_high=0.2, reduction="row")
    p, h = sc.policy_loss(logp, old, A, **kw), 2.0 ** -7
    slope = (sc.policy_loss(logp + h * dirn, old, A, **kw).loss.double() - sc.policy_loss(logp - h * dirn, old, A, **kw).loss.double()) / (2 * h)
    d = (logp - old).double()
    far = (((d - math.log1p(0.2)).abs() > 2 * h) & ((d - math.log1p(-0.2)).abs() > 2 * h)).all(1)
    most = (A.abs().double() + 0.2) * torch.exp(torch.maximum(d.abs().amax(1), (ref - logp).abs().amax(1).double()) + h)
    assert far.sum() >= 3
    assert ((slope - (p.d_logp.double() * dirn).sum(1)).abs() <= most * (h * h / 6 + 32 * U / h))[far].all()
