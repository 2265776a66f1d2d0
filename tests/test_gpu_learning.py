"""GPU tests of what is built from the catalogue operators: log_prob, fit_preferences and fit_policy of the factor models against
plain 64-bit steps, the operators in a captured graph, on side streams, and the refusals of the C ABI."""
import ctypes

import numpy as np
import pytest

from recommenders_amd.models import BPR, EASE, MF, WMF

pytestmark = pytest.mark.gpu


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


def _model(kind, n_users=60, n_items=90, k=20, seed=0):
    rng = np.random.default_rng(seed)
    U, V = rng.normal(0, .4, (n_users, k)).astype(np.float32), rng.normal(0, .4, (n_items, k)).astype(np.float32)
    b = rng.normal(0, .3, n_items).astype(np.float32)
    if kind == "bpr":
        return BPR(k=k, init_params={"U": U, "V": V, "Bi": b}), U, V, b
    if kind == "mf":
        m = MF(k=k, init_params={"U": U, "V": V, "Bu": rng.normal(0, .1, n_users).astype(np.float32), "Bi": b, "mu": 3.0})
        return m, U, V, b
    return WMF(k=k, init_params={"U": U, "V": V}), U, V, None


def _slates(rng, n, places, n_items, empty=True):
    s = rng.integers(0, n_items, (n, places)).astype(np.int64)
    if empty:
        s[rng.random(s.shape) < 0.25] = -1
    return s


class Plain:
    """Parameters and one step in float64."""

    def __init__(self, U, V, b):
        self.U, self.V, self.b = U.astype(np.float64), V.astype(np.float64), None if b is None else b.astype(np.float64)

    def logp(self, users, ids, scale=1.0):
        z = scale * (self.U[users] @ self.V.T + (0 if self.b is None else self.b))
        top = z.max(1, keepdims=True)
        lse = top + np.log(np.exp(z - top).sum(1, keepdims=True))
        return np.where(ids >= 0, np.take_along_axis(z, np.maximum(ids, 0), 1) - lse, 0.0), np.exp(z - lse)

    def step(self, users, ids, P, d, lr, scale=1.0, reg=0.0):
        d = np.where(ids >= 0, d, 0.0)
        dz = -d.sum(1, keepdims=True) * P
        for r in range(len(ids)):
            for j in range(ids.shape[1]):
                if ids[r, j] >= 0:
                    dz[r, ids[r, j]] += d[r, j]
        X = self.U[users].copy()
        dX, dV = scale * dz @ self.V + reg * X, scale * dz.T @ X + reg * self.V
        np.add.at(self.U, users, -lr * dX)
        self.V -= lr * dV
        if self.b is not None:
            self.b -= lr * scale * dz.sum(0)

    def near(self, model, names, tol):
        for name, want in zip(names, (self.U, self.V, self.b)):
            if name is not None:
                got = np.asarray(getattr(model, name), np.float64)
                assert np.abs(got - want).max() <= tol, (name, np.abs(got - want).max())


# a step moves a parameter by lr times a gradient of at most a few units, computed to 2^-20 of its terms; the parameters themselves
# (below 4) are rounded to fp32 once a step: 1e-5 leaves room for five steps of both
TOL = 1e-5


@pytest.mark.parametrize("kind", ["bpr", "mf", "wmf"])
def test_log_prob_and_model_stay_apart(torch, kind):
    model, U, V, b = _model(kind)
    rng = np.random.default_rng(1)
    users, ids = rng.integers(0, 60, 33), _slates(rng, 33, 4, 90)
    want, _ = Plain(U, V, b).logp(users, ids, 1.5)
    got = model.log_prob(users, ids, scale=1.5)
    assert got.dtype == np.float32 and np.abs(got - want).max() < 1e-5
    four = model.log_prob(users, ids, scale=1.5, precision="mxfp4")
    assert np.abs(four - want).max() < 3.0 and np.abs(four - want).max() > 1e-3         # another model, 4 bits an element
    assert (four[ids < 0] == 0).all() and model.log_prob(users, ids[:, 0]).shape == (33, 1)
    assert model.log_prob(users[:0], ids[:0]).shape == (0, 4)


@pytest.mark.parametrize("kind,loss,average,reference,reg", [("bpr", "logistic", False, False, 0.0), ("mf", "hinge", True, True, 0.01),
                                                            ("wmf", "squared", True, True, 0.0), ("bpr", "logistic", True, True, 0.1)])
def test_fit_preferences_is_a_gradient_step(torch, kind, loss, average, reference, reg):
    model, U, V, b = _model(kind)
    names = model._hip_learned()
    before = [U.copy(), V.copy(), None if b is None else b.copy()]
    model.ranked_items[3] = np.arange(4)
    rng = np.random.default_rng(2)
    n = 50
    users = rng.integers(0, 60, n)                                        # some users twice
    chosen, rejected = _slates(rng, n, 3, 90), _slates(rng, n, 5, 90)
    chosen[4] = -1
    plain, frozen = Plain(U, V, b), Plain(U, V, b)
    beta, lr, seed, want = 0.7, 0.1, 5, []
    order_rng = np.random.default_rng(seed)
    ids = np.concatenate([chosen, rejected], 1)
    for epoch in range(2):
        order, total = order_rng.permutation(n), 0.0
        for at in (order[:32], order[32:]):
            lp, P = plain.logp(users[at], ids[at], 1.2)
            d = lp - (frozen.logp(users[at], ids[at], 1.2)[0] if reference else 0.0)
            mc, mr = ids[at][:, :3] >= 0, ids[at][:, 3:] >= 0
            nc, nr = (np.maximum(mc.sum(1), 1), np.maximum(mr.sum(1), 1)) if average else (np.ones(len(at)), np.ones(len(at)))
            h = beta * ((d[:, :3] * mc).sum(1) / nc - (d[:, 3:] * mr).sum(1) / nr)
            if loss == "logistic":
                value, slope = np.log1p(np.exp(-h)), -1 / (1 + np.exp(h))
            elif loss == "hinge":
                assert (np.abs(h - 1) > 1e-4).all()
                value, slope = np.maximum(1 - h, 0), -(h < 1).astype(float)
            else:
                value, slope = ((h - .5) / beta) ** 2, 2 * (h - .5) / beta ** 2
            g = slope * beta / len(at)
            total += value.sum()
            plain.step(users[at], ids[at], P, np.concatenate([mc * (g / nc)[:, None], mr * (-g / nr)[:, None]], 1), lr, 1.2, reg)
        want.append(total / n)
    got = model.fit_preferences(users, chosen, rejected, learning_rate=lr, epochs=2, batch_size=32, beta=beta, kind=loss, average=average,
                                reference=reference, scale=1.2, reg=reg, seed=seed)
    np.testing.assert_allclose(got, want, rtol=1e-5)
    plain.near(model, names, TOL)
    assert not model.ranked_items                                         # rankings of the old parameters are gone
    assert np.array_equal(before[0], U) and np.array_equal(before[1], V) and (b is None or np.array_equal(before[2], b))


def test_fit_policy_is_a_gradient_step(torch):
    model, U, V, b = _model("bpr")
    rng = np.random.default_rng(3)
    n = 40
    users, slates, A = rng.integers(0, 60, n), _slates(rng, n, 4, 90), rng.normal(size=n).astype(np.float32)
    slates[7] = -1
    plain, frozen = Plain(U, V, b), Plain(U, V, b)
    old = (frozen.logp(users, slates)[0] + rng.normal(0, .2, slates.shape)).astype(np.float32)
    order = np.random.default_rng(9).permutation(n)
    total, lo, hi, coef, lr = 0.0, 0.2, 0.3, 0.5, 0.1
    for at in (order[:25], order[25:]):
        ids = slates[at]
        lp, P = plain.logp(users[at], ids)
        mask, a = ids >= 0, A[at][:, None].astype(np.float64)
        d = lp - old[at]
        assert (np.abs(d - np.log1p(hi)) > 1e-5).all() and (np.abs(d - np.log1p(-lo)) > 1e-5).all()
        over, under = (a > 0) & (d > np.log1p(hi)), (a < 0) & (d < np.log1p(-lo))
        ratio = np.exp(d)
        q = frozen.logp(users[at], ids)[0] - lp
        c = 1.0 / np.maximum(mask.sum(1, keepdims=True), 1) / len(at)
        term = -a * np.where(over, 1 + hi, np.where(under, 1 - lo, ratio)) + coef * (np.exp(q) - q - 1)
        grad = np.where(over | under, 0.0, -a * ratio) - coef * np.expm1(q)
        total += (np.where(mask, term, 0) * c).sum() * len(at)
        plain.step(users[at], ids, P, np.where(mask, grad, 0) * c, lr)
    got = model.fit_policy(users, slates, A, old_log_prob=old, learning_rate=lr, batch_size=25, clip_low=lo, clip_high=hi, kl_coef=coef, seed=9)
    np.testing.assert_allclose(got, [total / n], rtol=1e-5, atol=1e-6)
    plain.near(model, model._hip_learned(), TOL)


def test_fit_policy_and_preferences_run_with_a_4bit_reference(torch):
    model, U, V, b = _model("bpr", k=37)
    rng = np.random.default_rng(4)
    users = rng.integers(0, 60, 30)
    s = _slates(rng, 30, 2, 90)
    assert len(model.fit_preferences(users, s, s[::-1].copy(), reference=True, reference_precision="mxfp4", epochs=3)) == 3
    assert len(model.fit_policy(users, s, rng.normal(size=30), kl_coef=0.1, reference_precision="mxfp4")) == 1
    assert np.isfinite(model.u_factors).all() and np.isfinite(model.i_factors).all() and np.isfinite(model.i_biases).all()
    a = model.fit_preferences(users, s, s[::-1].copy(), epochs=0)
    assert a == [] and model.u_factors.shape == U.shape


# ---------------------------------------------------------------- the operators together
def _step(sc, X, V, b, ids, ref, places):
    logp, lse = sc.catalogue_logprob(X, V, ids, ibase=b)
    p = sc.preference_loss(logp[:, :places], logp[:, places:], ref[:, :places], ref[:, places:], beta=0.5)
    import torch
    d = torch.cat([p.d_chosen, p.d_rejected], 1)
    return (logp, lse, p.loss, d) + sc.catalogue_logprob_backward(X, V, ids, lse, d, ibase=b)


@pytest.mark.parametrize("n,items,k,dtype", [(40, 300, 50, "float32"), (150, 1000, 128, "bfloat16"), (200, 40000, 64, "float32"), (70, 900, 200, "bfloat16")])
def test_a_captured_step_replays(torch, sc, n, items, k, dtype):
    """A graph of the whole step replayed on new inputs, with eager steps of the same operators between the replays."""
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    dt = getattr(torch, dtype)
    new = lambda: ((torch.randn((n, k), generator=g, device="cuda") * .3).to(dt), (torch.randn((items, k), generator=g, device="cuda") * .3).to(dt),
                   torch.randn(items, generator=g, device="cuda"), torch.randint(-1, items, (n, 7), generator=g, device="cuda", dtype=torch.int32),
                   -torch.rand((n, 7), generator=g, device="cuda"))
    held = [t.clone() for t in new()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(sc, *held, 3)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(sc, *held, 3)
    for _ in range(4):
        fresh = new()
        for t, f in zip(held, fresh):
            t.copy_(f)
        graph.replay()
        want = _step(sc, *fresh, 3)
        torch.cuda.synchronize()
        for a, w in zip(out, want):
            assert torch.equal(a, w)


def test_a_captured_policy_step_replays(torch, sc):
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    new = lambda: (-torch.rand((300, 33), generator=g, device="cuda"), -torch.rand((300, 33), generator=g, device="cuda"), torch.randn(300, generator=g, device="cuda"),
                   -torch.rand((300, 33), generator=g, device="cuda"), torch.rand((300, 33), generator=g, device="cuda") < .7)
    call = lambda logp, old, A, ref, mask: sc.policy_loss(logp, old, A, ref_logp=ref, mask=mask, kl_coef=.1, reduction="batch")
    held = [t.clone() for t in new()]
    call(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(*held)
        X = sc.quantize_mxfp4(held[0])
        scores = sc.score_mxfp4(X, X)
    for _ in range(4):
        fresh = new()
        for t, f in zip(held, fresh):
            t.copy_(f)
        graph.replay()
        want = call(*fresh)
        q = sc.quantize_mxfp4(fresh[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(out, want)) and torch.equal(scores, sc.score_mxfp4(q, q))


def test_calls_on_two_streams_at_once(torch, sc):
    """Two steps in flight on streams of their own: workspaces are each call's own."""
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    def inputs(n):
        return (torch.randn((n, 96), generator=g, device="cuda") * .3, torch.randn((3000, 96), generator=g, device="cuda") * .3,
                torch.randn(3000, generator=g, device="cuda"), torch.randint(0, 3000, (n, 6), generator=g, device="cuda", dtype=torch.int32),
                -torch.rand((n, 6), generator=g, device="cuda"))
    a, b = inputs(500), inputs(450)
    want = _step(sc, *a, 3), _step(sc, *b, 3)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        got = []
        for s, x in zip(streams, (a, b)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(_step(sc, *x, 3))
        torch.cuda.synchronize()
        for g1, w1 in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(g1, w1))


# ---------------------------------------------------------------- refusals of the C ABI
def test_c_refusals(torch, sc):
    from recommenders_amd import _lib
    from recommenders_amd.engine import IfrError
    lib, h = sc._lib, sc._h
    X, V = torch.zeros((4, 8), device="cuda"), torch.zeros((9, 8), device="cuda")
    ids = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    out = torch.zeros((4, 2), device="cuda")
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    args = lambda **kw: _lib.Catalogue(**{**dict(X=X.data_ptr(), V=V.data_ptr(), n=4, n_items=9, ldx=8, ldv=8, k=8, dtype=0, scale=1.0), **kw})

    def forward(c, w=ws.data_ptr(), size=1 << 20, m=2, ld=2, idp=ids.data_ptr()):
        return lib.ifr_catalogue_logprob(h, None if c is None else ctypes.byref(c), idp, m, ld, out.data_ptr(), 2, None, w, size, None)

    assert forward(args()) == 0
    bad = [forward(None), forward(args(X=None)), forward(args(V=None)), forward(args(k=0)), forward(args(k=257)), forward(args(n=-1)), forward(args(n_items=0)),
           forward(args(n=1 << 26)), forward(args(n_items=1 << 29)), forward(args(ldx=7)), forward(args(ldv=7)), forward(args(scale=0.0)),
           forward(args(scale=float("nan"))), forward(args(dtype=3)), forward(args(dtype=2)), forward(args(), w=None), forward(args(), size=64),
           forward(args(), w=ws.data_ptr() + 16), forward(args(), ld=1), forward(args(), m=-1), forward(args(), idp=None)]
    assert bad == [-1] * len(bad)
    with pytest.raises(IfrError, match="null ids"):
        sc._check(bad[-1])
    assert forward(args(n=0), w=None) == 0
    need = ctypes.c_int64(0)
    assert lib.ifr_catalogue_logprob_workspace(h, ctypes.byref(args()), None) == -1 and lib.ifr_catalogue_logprob_workspace(h, None, ctypes.byref(need)) == -1
    lse, d = torch.zeros(4, device="cuda"), torch.zeros((4, 2), device="cuda")
    backward = lambda c, lsep=lse.data_ptr(), dp=d.data_ptr(), ldx=8, w=ws.data_ptr(): lib.ifr_catalogue_logprob_backward(
        h, ctypes.byref(c), ids.data_ptr(), 2, 2, lsep, dp, 2, X.data_ptr(), ldx, None, 0, None, w, 1 << 20, None)
    bad = [backward(args(), lsep=None), backward(args(), dp=None), backward(args(), ldx=7), backward(args(), w=None),
           backward(args(dtype=2, x_scales=1, v_scales=1)), lib.ifr_catalogue_logprob_backward_workspace(h, ctypes.byref(args(dtype=2)), 2, 1, 1, 1, ctypes.byref(need)),
           lib.ifr_catalogue_logprob_backward_workspace(h, ctypes.byref(args()), -1, 1, 1, 1, ctypes.byref(need))]
    assert bad == [-1] * len(bad)
    u8 = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    p, o = u8.data_ptr(), out.data_ptr()
    bad = [lib.ifr_mxfp4_quantize(h, None, 0, 4, 8, 8, p, p, None), lib.ifr_mxfp4_quantize(h, o, 2, 4, 2, 2, p, p, None), lib.ifr_mxfp4_quantize(h, o, 0, 4, 2, 1, p, p, None),
           lib.ifr_mxfp4_quantize(h, o, 0, 4, 0, 2, p, p, None), lib.ifr_mxfp4_quantize(h, o, 0, 4, 2, 2, p + 4, p, None),
           lib.ifr_mxfp4_dequantize(h, p, None, 4, 2, o, 2, None), lib.ifr_mxfp4_dequantize(h, p, p, 4, 2, o, 1, None),
           lib.ifr_mxfp4_scores(h, p, p, 2, p, p, 2, 257, None, None, o, 0, 2, None), lib.ifr_mxfp4_scores(h, p, p, 2, p, p, 2, 8, None, None, o, 2, 2, None),
           lib.ifr_mxfp4_scores(h, p, p, 2, p, p, 2, 8, None, None, o, 0, 1, None), lib.ifr_mxfp4_scores(h, p + 8, p, 2, p, p, 2, 8, None, None, o, 0, 2, None)]
    assert bad == [-1] * len(bad)
    pref = lambda **kw: lib.ifr_preference_loss(h, ctypes.byref(_lib.Preference(**{**dict(n=4, len_chosen=1, len_rejected=1, chosen=o, rejected=o, ld_chosen=2,
                                                                                       ld_rejected=2, beta=1.0), **kw})), None)
    assert pref() == 0 and pref(n=0, chosen=None) == 0
    bad = [pref(chosen=None), pref(beta=0.0), pref(kind=3), pref(label_smoothing=0.5), pref(label_smoothing=0.1, kind=1), pref(n=-1), pref(ld_chosen=0),
           pref(ref_chosen=o, ld_ref_chosen=2), pref(d_chosen=o, ld_d_chosen=0), pref(mask_chosen=p, ld_mask_chosen=0), pref(margin=float("inf"))]
    assert bad == [-1] * len(bad)
    pol = lambda **kw: lib.ifr_policy_loss(h, ctypes.byref(_lib.Policy(**{**dict(n=4, len=2, logp=o, old_logp=o, advantages=lse.data_ptr(), ld_logp=2, ld_old=2), **kw})),
                                           None, 0, None)
    assert pol() == 0
    bad = [pol(logp=None), pol(advantages=None), pol(reduction=3), pol(clip_low=1.0), pol(clip_high=-1.0), pol(kl_coef=float("nan")), pol(ld_old=1),
           pol(mask=p, ld_mask=2, reduction=2), pol(d_logp=o, ld_d_logp=1), pol(n=-1)]
    assert bad == [-1] * len(bad)
    torch.cuda.synchronize()


def test_models_without_factors_do_not_learn(torch):
    assert not hasattr(EASE(trainable=False, B=np.zeros((3, 3))), "fit_preferences")


def test_a_model_that_learned_can_be_copied(torch):
    """hip_invalidate drops everything on the device, the learning engine too."""
    import copy
    m = _model("bpr")[0]
    m.fit_preferences([0, 1], [3, 4], [5, 6])
    before = m.log_prob([0], [[3]])
    m.hip_invalidate()
    assert np.array_equal(copy.deepcopy(m).log_prob([0], [[3]]), before)


def test_c_refusals_of_sizes_and_factors(torch, sc):
    from recommenders_amd import _lib
    x = torch.zeros(64, device="cuda")
    o, long = x.data_ptr(), (1 << 30) + 1
    pref = lambda **kw: sc._lib.ifr_preference_loss(sc._h, ctypes.byref(_lib.Preference(**{**dict(n=1, len_chosen=1, len_rejected=1, chosen=o, rejected=o, ld_chosen=1,
                                                                                             ld_rejected=1, beta=1.0), **kw})), None)
    pol = lambda **kw: sc._lib.ifr_policy_loss(sc._h, ctypes.byref(_lib.Policy(**{**dict(n=1, len=1, logp=o, old_logp=o, advantages=o, ld_logp=1, ld_old=1), **kw})),
                                               None, 0, None)
    c = lambda scale: ctypes.byref(_lib.Catalogue(X=o, V=o, n=1, n_items=1, ldx=8, ldv=8, k=8, dtype=0, scale=scale))
    need = ctypes.c_int64(0)
    size = lambda scale: sc._lib.ifr_catalogue_logprob_workspace(sc._h, c(scale), ctypes.byref(need))
    assert pref() == 0 and pol() == 0 and size(1e-30) == 0 and size(1e30) == 0
    bad = [pref(len_chosen=long, ld_chosen=long), pref(len_rejected=long, ld_rejected=long), pref(beta=1e-31), pol(len=long, ld_logp=long, ld_old=long),
           size(1e-31), size(1e31)]
    assert bad == [-1] * len(bad)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_captured_gradient_of_many_places_replays(torch, sc, dtype):
    """Batches whose places are dealt into buckets: one graph, batches of many and of no places in turn, every replay the eager call's bits."""
    n, items, k, m = 1100, 4096, 40, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    X, V = ((torch.randn((r, k), generator=g, device="cuda") * .3).to(getattr(torch, dtype)) for r in (n, items))

    def batch(lowest, highest):
        ids = torch.randint(lowest, highest, (n, m), generator=g, device="cuda", dtype=torch.int32)
        d = torch.randn((n, m), generator=g, device="cuda") / n
        return ids, d, sc.catalogue_logprob(X, V, ids)[1]

    held = [t.clone() for t in batch(-1, items)]
    call = lambda ids, d, lse: sc.catalogue_logprob_backward(X, V, ids, lse, d)[:2]
    call(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(*held)
    # every item; 128 of the last ones alone; empty places alone; half of them empty; behind the catalogue too
    for lowest, highest in ((0, items), (items - 128, items), (-1, 0), (-items, items), (0, 2 * items)):
        fresh = batch(lowest, highest)
        for t, f in zip(held, fresh):
            t.copy_(f)
        graph.replay()
        want = call(*fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(out, want))
        if highest == 0:
            assert not want[0].any() and not want[1].any()
