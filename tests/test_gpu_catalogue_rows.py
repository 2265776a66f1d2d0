"""GPU tests of the catalogue operators row by row: users and items whose results are small beside their neighbours' or beside the parts
that they are the difference of.  Every tolerance is a worst-case bound of its own element, from a reference in 64 bits.

U = 2^-24 is half a step of fp32 relative to the value, B = 2^-8 of bf16."""
import math

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


class Exact:
    """Forward and gradient in float64, and for each element a bound of the kernels' error.  `score`: error of a score by the products of
    its operands, relative to sum |x v| + |b| (0 where operands and sums are exact); `part`: of a probability (times G) as an operand of
    the second product, relative to itself."""

    def __init__(self, torch, X, V, b, ids, dlogp, scale, score, part):
        x, v = X.double(), V.double()
        n, m = ids.shape
        items, k = V.shape
        s, room = x @ v.t(), x.abs() @ v.abs().t()
        if b is not None:
            s, room = s + b.double(), room + b.double().abs().nan_to_num(posinf=0.0)
        live = torch.ones_like(s, dtype=torch.bool) if b is None else (b != -math.inf).expand_as(s)
        z, room = scale * s, torch.where(live, scale * room, 0.0)
        self.lse = torch.logsumexp(z, 1)
        held, at = ids >= 0, ids.long().clamp(min=0)
        self.held = held
        self.logp = torch.where(held, z.gather(1, at) - self.lse[:, None], 0.0)
        P = torch.exp(z - self.lse[:, None])
        # a score: its operands, up to 3 k additions of fp32, the roundings of scale, base and log2(e); the exponent rounds |z| and |lse|
        # twice each; lse: v_exp_f32 (2^-22) and the sum of positive numbers, at most items / 2 + 64 additions
        e = (score + (3 * k + 4) * U * (score > 0)) * room
        Z = torch.where(live, z.abs(), 0.0) + self.lse.abs()[:, None] + 8
        self.e_lse = (torch.where(live, P * (e + 6 * Z * U), 0.0).sum(1) + 6 * U * (self.lse.abs() + 8) + 2.0 ** -21 + (items / 2 + 64) * U)
        self.e_logp = e.gather(1, at) + self.e_lse[:, None] + 6 * U * Z.gather(1, at)
        e_p = torch.where(live, e + self.e_lse[:, None] + 6 * Z * U + 2.0 ** -21, 0.0)            # relative, of a probability
        g = torch.where(held, dlogp.double(), 0.0)
        G, gabs = g.sum(1), g.abs().sum(1)
        hot = torch.zeros_like(z).scatter_add_(1, at, g)
        hot_abs = torch.zeros_like(z).scatter_add_(1, at, g.abs())
        dz = hot - G[:, None] * P
        self.dX, self.dV, self.db = scale * dz @ v, scale * dz.t() @ x, scale * dz.sum(0)
        low = U if X.dtype == torch.float32 else B
        # probabilities: their error, the part's and the operand's rounding (2^-21 covers a left-out product of low parts), m additions in G;
        # in the sums 3 a term; the named items' part: products and additions in fp32; the result's rounding
        mass = gabs[:, None] * P
        wx, wv = scale * mass * (e_p + part + 2.0 ** -21 + (m + 3 * items) * U), scale * mass * (e_p + part + 2.0 ** -21 + (m + 3 * n) * U)
        self.t_dX = wx @ v.abs() + (m + 4) * U * scale * hot_abs @ v.abs() + (low + 2 * U) * self.dX.abs() + 1e-35
        self.t_dV = wv.t() @ x.abs() + (n * m + 4) * U * scale * hot_abs.t() @ x.abs() + (low + 2 * U) * self.dV.abs() + 1e-35
        self.t_db = wv.sum(0) + (n * m + 4) * U * scale * hot_abs.sum(0) + 3 * U * self.db.abs() + 1e-35
        if X.dtype == torch.float32:
            # 32 neighbouring terms of one row's sum share the step of the largest, 2^-39 of it; so do the elements of an operand's row
            step = 32 * 2.0 ** -38 * scale
            self.t_dX = self.t_dX + step * (mass @ v.abs().amax(1))[:, None]
            self.t_dV = self.t_dV + step * (mass.t() @ x.abs().amax(1))[:, None]


def _within(got, want, tol):
    return ((got.double() - want).abs() <= tol)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("n,items,k", [(20, 150, 64), (130, 150, 64), (40, 141, 160)])
def test_gradient_of_confident_users(torch, sc, n, items, k, dtype):
    """Every user names its own item, which has nearly all of the probability: a row of the gradient is g (1 - P) times a difference of
    vectors, and what P loses before that difference is taken is lost to the row.  Operands are multiples of 1/8 of at most 2, so that
    scores are exact in fp32 and bf16 takes the operands as they are."""
    g = _gen(torch, n + k)
    V = (torch.randn((items, k), generator=g, device="cuda") * 0.4 * 8 * math.sqrt(64 / k)).round().clamp(-16, 16) / 8
    named = torch.randperm(items, generator=g, device="cuda")[:n]
    X, V = V[named].to(getattr(torch, dtype)), V.to(getattr(torch, dtype))
    ids = torch.stack([named, torch.full_like(named, -1)], 1).to(torch.int32)
    dlogp = torch.randn((n, 2), generator=g, device="cuda")
    scale = 1.2
    r = Exact(torch, X, V, None, ids, dlogp, scale, 0.0, 2.0 ** -16 if dtype == "bfloat16" else 2.0 ** -22)
    _, lse = sc.catalogue_logprob(X, V, ids, scale=scale)
    dX, dV, _ = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, scale=scale)
    assert float(r.logp[:, 0].exp().median()) > 0.99
    rows = named.long()
    for got, want, tol in ((dX, r.dX, r.t_dX), (dV[rows], r.dV[rows], r.t_dV[rows])):
        room = tol.norm(dim=1) / want.norm(dim=1)
        assert float(room.median()) < 0.2                       # the bound says something
        off = (got.double() - want).norm(dim=1) / want.norm(dim=1)
        assert (off <= room).all(), (float(off.max()), float((off / room).max()))
    assert _within(dX, r.dX, r.t_dX).all() and _within(dV, r.dV, r.t_dV).all()


@pytest.mark.parametrize("n,items,k", [(70, 300, 64), (33, 500, 200), (300, 200, 33)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_gradient_of_unlikely_items(torch, sc, n, items, k, dtype):
    """Items that nobody names and that have a probability of about 2^-87: their rows of dV keep the precision of the others'."""
    g = _gen(torch, n)
    dt = getattr(torch, dtype)
    X, V = (torch.randn((n, k), generator=g, device="cuda") * 0.3).to(dt), (torch.randn((items, k), generator=g, device="cuda") * 0.3).to(dt)
    b = torch.randn(items, generator=g, device="cuda")
    b[40:90] = -60.0
    ids = torch.randint(100, items, (n, 3), generator=g, device="cuda", dtype=torch.int32)
    dlogp = torch.randn((n, 3), generator=g, device="cuda")
    r = Exact(torch, X, V, b, ids, dlogp, 1.0, 3 * 2.0 ** -22, 2.0 ** -16 if dtype == "bfloat16" else 2.0 ** -21)
    _, lse = sc.catalogue_logprob(X, V, ids, ibase=b)
    dX, dV, db = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b)
    assert 0 < float(r.dV[40:90].abs().max()) < 1e-20
    assert float((r.t_dV[40:90].norm(dim=1) / r.dV[40:90].norm(dim=1)).median()) < 0.05
    assert _within(dX, r.dX, r.t_dX).all() and _within(dV, r.dV, r.t_dV).all() and _within(db, r.db, r.t_db).all()


@pytest.mark.parametrize("n,items,k", [(70, 300, 64), (40, 257, 200)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_gradient_beside_a_user_of_large_gradient(torch, sc, n, items, k, dtype):
    """One user's upstream gradient is 2^30 times the others', and all of its probability lies on one item: rows of dV of the other items,
    and the other users' rows of dX, are as precise as without it."""
    g = _gen(torch, n + 1)
    dt = getattr(torch, dtype)
    X, V = (torch.randn((n, k), generator=g, device="cuda") * 0.3), (torch.randn((items, k), generator=g, device="cuda") * 0.3).to(dt)
    X[3] = V[50].float() * (160 / float(V[50].float().norm() ** 2))
    X = X.to(dt)
    ids = torch.randint(60, items, (n, 3), generator=g, device="cuda", dtype=torch.int32)
    dlogp = torch.randn((n, 3), generator=g, device="cuda")
    ids[3], dlogp[3] = 50, dlogp[3] * 2.0 ** 30
    r = Exact(torch, X, V, None, ids, dlogp, 1.0, 3 * 2.0 ** -22, 2.0 ** -16 if dtype == "bfloat16" else 2.0 ** -21)
    _, lse = sc.catalogue_logprob(X, V, ids)
    dX, dV, _ = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp)
    others = torch.arange(items, device="cuda") != 50
    assert float((r.t_dV.norm(dim=1) / r.dV.norm(dim=1))[others].median()) < 0.05
    assert _within(dX, r.dX, r.t_dX).all() and _within(dV, r.dV, r.t_dV).all()


@pytest.mark.parametrize("n,items,k", [(90, 300, 50), (40, 310, 200), (130, 257, 128), (600, 90, 33)])
@pytest.mark.parametrize("large", [2.0 ** 24, 2.0 ** 40, 2.0 ** 60])
def test_large_rows_leave_their_neighbours_alone(torch, sc, n, items, k, large):
    """fp32: a user, an item that is taken out and a padding user whose rows are far larger than their neighbours', and an item that is large
    only where every user has a zero: the other users and items keep their precision."""
    g = _gen(torch, n + k)
    X, V = torch.randn((n, k), generator=g, device="cuda") * 0.3, torch.randn((items, k), generator=g, device="cuda") * 0.3
    b = torch.randn(items, generator=g, device="cuda")
    ids = torch.randint(12, items, (n, 3), generator=g, device="cuda", dtype=torch.int32)
    dlogp = torch.randn((n, 3), generator=g, device="cuda")
    X[7] *= large
    V[11] *= large
    b[11] = -math.inf
    X[20], ids[20] = large, -1
    X[:, k - 1] = 0
    with_item = V.clone()
    with_item[45] = 0
    with_item[45, k - 1] = large
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[7] = rest[20] = False
    for v in (V, with_item):
        r = Exact(torch, X, v, b, ids, dlogp, 1.0, 3 * 2.0 ** -22, 2.0 ** -21)
        logp, lse = sc.catalogue_logprob(X, v, ids, ibase=b)
        assert float(r.e_lse[rest].max()) < 2e-3
        assert _within(lse, r.lse, r.e_lse)[rest].all() and _within(logp, r.logp, r.e_logp)[rest].all()
    logp, lse = sc.catalogue_logprob(X, V, ids, ibase=b)
    r = Exact(torch, X, V, b, ids, dlogp, 1.0, 3 * 2.0 ** -22, 2.0 ** -21)
    dX, dV, db = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b)
    assert (dX[20] == 0).all() and _within(dX, r.dX, r.t_dX)[rest].all()
    # the large user's own part lies on the items that it names and on its likeliest ones
    clear = torch.ones(items, dtype=torch.bool, device="cuda")
    clear[ids[7].long()] = False
    clear[(X[7].double() @ V.double().t() + b.double()).topk(3).indices] = False
    assert float((r.t_dV.norm(dim=1) / r.dV.norm(dim=1).clamp(min=1e-12))[clear].median()) < 0.01
    assert _within(dV, r.dV, r.t_dV)[clear].all() and _within(db, r.db, r.t_db)[clear].all()


@pytest.mark.parametrize("n,items,k", [(90, 300, 50), (40, 200, 200)])
@pytest.mark.parametrize("spread", [1e-32, 1e-28, 1e-24, 1e28, 1e30])
def test_magnitudes_far_from_one(torch, sc, n, items, k, spread):
    """fp32 items far from 1 and users as far on the other side: ordinary scores, and every row with the precision of one near 1."""
    g = _gen(torch, n)
    X, V = torch.randn((n, k), generator=g, device="cuda") * 0.3 / spread, torch.randn((items, k), generator=g, device="cuda") * 0.3 * spread
    ids = torch.randint(0, items, (n, 3), generator=g, device="cuda", dtype=torch.int32)
    dlogp = torch.randn((n, 3), generator=g, device="cuda")
    r = Exact(torch, X, V, None, ids, dlogp, 1.0, 3 * 2.0 ** -22, 2.0 ** -21)
    logp, lse = sc.catalogue_logprob(X, V, ids)
    assert _within(lse, r.lse, r.e_lse).all() and _within(logp, r.logp, r.e_logp).all()
    dX, dV, _ = sc.catalogue_logprob_backward(X, V, ids, lse, dlogp)
    assert _within(dX, r.dX, r.t_dX).all() and _within(dV, r.dV, r.t_dV).all()
    assert float((r.t_dX.norm(dim=1) / r.dX.norm(dim=1)).median()) < 0.02 and float((r.t_dV.norm(dim=1) / r.dV.norm(dim=1)).median()) < 0.02
