"""CPU tests of the catalogue operators' argument checks (recommenders_amd/catalogue.py): what is refused, before any library call."""
import pytest
import torch

from recommenders_amd import MxFp4Matrix
from recommenders_amd import catalogue as C


def _mx(n, k):
    kb = (k + 31) // 32
    return MxFp4Matrix(torch.zeros((n, 16 * kb), dtype=torch.uint8), torch.zeros((n, kb), dtype=torch.uint8), k)


def test_mxfp4_matrix():
    q = _mx(3, 50)
    assert q.shape == (3, 50) and q.device.type == "cpu"
    with pytest.raises(ValueError, match="takes codes"):
        MxFp4Matrix(torch.zeros((3, 16), dtype=torch.uint8), torch.zeros((3, 2), dtype=torch.uint8), 50)
    with pytest.raises(ValueError, match="takes codes"):
        MxFp4Matrix(torch.zeros((3, 32), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8), 50)
    with pytest.raises(ValueError, match="uint8"):
        MxFp4Matrix(torch.zeros((3, 32)), torch.zeros((3, 2), dtype=torch.uint8), 50)
    with pytest.raises(ValueError, match="at least 1"):
        MxFp4Matrix(torch.zeros((3, 0), dtype=torch.uint8), torch.zeros((3, 0), dtype=torch.uint8), 0)
    shifted = MxFp4Matrix(torch.zeros(97, dtype=torch.uint8)[1:].view(3, 32), torch.zeros((3, 2), dtype=torch.uint8), 64)
    assert shifted.codes.data_ptr() % 16 == 0


X, V, IDS = torch.zeros((4, 8)), torch.zeros((9, 8)), torch.zeros((4, 2), dtype=torch.int32)


@pytest.mark.parametrize("args,error,words", [
    ((X, V.bfloat16(), IDS, None, 1.0), TypeError, "V must be float32"),
    ((X.double(), V, IDS, None, 1.0), TypeError, "X must be float32 or bfloat16"),
    ((X.half(), V.half(), IDS, None, 1.0), TypeError, "X must be float32 or bfloat16"),
    ((X, V[:, :7], IDS, None, 1.0), ValueError, "V must be"),
    ((X[0], V, IDS, None, 1.0), ValueError, "matrix"),
    ((X, V, IDS.long(), None, 1.0), TypeError, "ids must be int32"),
    ((X, V, IDS[:3], None, 1.0), ValueError, "ids must be"),
    ((X, V, IDS[0], None, 1.0), ValueError, "matrix"),
    ((X, V[:0], IDS, None, 1.0), ValueError, "rows of V"),
    ((X, V, IDS, torch.zeros(8), 1.0), ValueError, "ibase must be"),
    ((X, V, IDS, torch.zeros(9).double(), 1.0), TypeError, "ibase must be float32"),
    ((X, V, IDS, None, 0.0), ValueError, "scale"),
    ((X, V, IDS, None, float("nan")), ValueError, "scale"),
    ((torch.zeros((4, 257)), torch.zeros((9, 257)), IDS, None, 1.0), ValueError, "k must be"),
    ((X.clone().requires_grad_(), V, IDS, None, 1.0), ValueError, "autograd"),
    ((X, V, IDS, torch.zeros(9, requires_grad=True), 1.0), ValueError, "gradient"),
    ((_mx(4, 8), V, IDS, None, 1.0), TypeError, "both"),
    ((_mx(4, 8), _mx(9, 9), IDS, None, 1.0), ValueError, "factors"),
    ((X.numpy(), V, IDS, None, 1.0), TypeError, "torch tensor"),
])
def test_catalogue_refusals(args, error, words):
    with pytest.raises(error, match=words):
        C.check_catalogue(*args)


def test_catalogue_device_and_no_grad():
    with pytest.raises(ValueError, match="the scorer on"):
        C.check_catalogue(X, V, IDS, None, 1.0, device=torch.device("cuda", 0))
    with torch.no_grad():
        C.check_catalogue(X.clone().requires_grad_(), V, IDS, None, 1.0)
    a = C.check_catalogue(X.t().contiguous().t(), V, IDS[:, :1].expand(4, 5), None, 1.0)
    assert a[0][0].stride() == (8, 1) and a[0][1] == 8 and a[2][0].is_contiguous() and a[2][1] == 5
    assert C.check_catalogue(torch.zeros((4, 20))[:, 3:11], V, IDS, None, 1.0)[0][1] == 20 and C.check_catalogue(X[:1].expand(4, 8), V, IDS, None, 1.0)[0][1] == 8
    assert C.check_catalogue(torch.zeros((9, 20))[2:3, 3:11], V, IDS[:1], None, 1.0)[0][1] == 8


L, R = torch.zeros((4, 3)), torch.zeros((4, 5))


def _pref(**kw):
    a = dict(chosen=L, rejected=R, ref_chosen=None, ref_rejected=None, mask_chosen=None, mask_rejected=None, weight=None, beta=0.1, kind="logistic",
             label_smoothing=0.0, margin=0.0)
    a.update(kw)
    return C.check_preference(**a)


@pytest.mark.parametrize("kw,error,words", [
    (dict(rejected=R[:3]), ValueError, "rejected must be"),
    (dict(chosen=L.bfloat16()), TypeError, "chosen must be float32"),
    (dict(ref_chosen=L), ValueError, "both"),
    (dict(ref_chosen=L, ref_rejected=L), ValueError, "ref_rejected must be"),
    (dict(mask_chosen=torch.ones((4, 2), dtype=torch.bool)), ValueError, "mask_chosen must be"),
    (dict(mask_rejected=R), TypeError, "mask_rejected must be bool"),
    (dict(weight=torch.ones(3)), ValueError, "weight must be"),
    (dict(beta=0.0), ValueError, "beta"),
    (dict(beta=float("nan")), ValueError, "beta"),
    (dict(kind="other"), ValueError, "kind"),
    (dict(label_smoothing=0.5), ValueError, "label_smoothing"),
    (dict(label_smoothing=0.1, kind="hinge"), ValueError, "logistic"),
    (dict(margin=float("inf")), ValueError, "margin"),
    (dict(chosen=L.clone().requires_grad_()), ValueError, "autograd"),
])
def test_preference_refusals(kw, error, words):
    with pytest.raises(error, match=words):
        _pref(**kw)
    _pref()


def _pol(**kw):
    a = dict(logp=L, old_logp=L, advantages=torch.zeros(4), ref_logp=None, mask=None, weight=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, reduction="row")
    a.update(kw)
    return C.check_policy(**a)


@pytest.mark.parametrize("kw,error,words", [
    (dict(old_logp=R), ValueError, "old_logp must be"),
    (dict(advantages=None), TypeError, "advantages"),
    (dict(advantages=torch.zeros((4, 3))), ValueError, "advantages must be"),
    (dict(ref_logp=R), ValueError, "ref_logp must be"),
    (dict(mask=L), TypeError, "mask must be bool"),
    (dict(clip_low=1.0), ValueError, "clip_low"),
    (dict(clip_high=-0.1), ValueError, "clip_high"),
    (dict(kl_coef=0.1), ValueError, "kl_coef needs"),
    (dict(kl_coef=float("nan"), ref_logp=L), ValueError, "finite"),
    (dict(reduction="mean"), ValueError, "reduction"),
    (dict(weight=torch.zeros(5)), ValueError, "weight must be"),
])
def test_policy_refusals(kw, error, words):
    with pytest.raises(error, match=words):
        _pol(**kw)
    _pol()


# ---------------------------------------------------------------- the factor models' checks
def test_learning_refusals():
    import numpy as np

    from recommenders_amd.models import BPR
    m = BPR(k=3, init_params={"U": np.zeros((4, 3), np.float32), "V": np.zeros((5, 3), np.float32), "Bi": np.zeros(5, np.float32)})
    assert m._hip_users([0, 3, 3]).tolist() == [0, 3, 3] and m._hip_slates([1, -1], 2, "x").shape == (2, 1)
    for users in ([4], [-1, 0]):
        with pytest.raises(IndexError, match="user index"):
            m._hip_users(users)
    for users in ([[0]], [0.5]):
        with pytest.raises(ValueError, match="users"):
            m._hip_users(users)
    for items in ([[5]], [[-2]]):
        with pytest.raises(IndexError, match="item index"):
            m._hip_slates(items, 1, "chosen")
    with pytest.raises(ValueError, match="chosen"):
        m._hip_slates([[1], [2]], 1, "chosen")
    for bad in (dict(batch_size=0), dict(learning_rate=0.0), dict(reg=-1.0), dict(epochs=-1)):
        with pytest.raises(ValueError, match="batch_size"):
            list(m._hip_schedule(3, **{**dict(batch_size=2, epochs=1, learning_rate=.1, reg=0.0, seed=0), **bad}))
    assert sorted(np.concatenate([b for _, b in m._hip_schedule(5, 2, 1, .1, 0.0, 0)]).tolist()) == list(range(5))


def test_sizes_and_factors_out_of_range():
    """Rows that the kernels' 32-bit places do not hold, and factors whose reciprocal fp32 does not hold."""
    wide = torch.empty((1, C.MAX_LENGTH + 1), device="meta")
    one = torch.empty((1, 1), device="meta")
    args = (None, None, None, None, None, 0.1, "logistic", 0.0, 0.0)
    with pytest.raises(ValueError, match="places"):
        C.check_preference(wide, one, *args)
    with pytest.raises(ValueError, match="places"):
        C.check_preference(one, wide, *args)
    with pytest.raises(ValueError, match="places"):
        C.check_policy(wide, wide, torch.empty(1, device="meta"), None, None, None, 0.2, 0.2, 0.0, "row")
    for scale in (1e-31, 1e31, float("nan")):
        with pytest.raises(ValueError, match="scale must be positive"):
            C.check_catalogue(X, V, IDS, None, scale)
    with pytest.raises(ValueError, match="beta must be positive"):
        C.check_preference(torch.zeros((2, 3)), torch.zeros((2, 3)), None, None, None, None, None, 1e-31, "logistic", 0.0, 0.0)
