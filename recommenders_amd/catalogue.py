"""Catalogue operators of `HipScorer`: a 4-bit microscaled model and its score rows, log-probabilities of items under the
softmax over the whole catalogue with their gradient, and the preference and policy losses (contracts: include/ifr.h).

Operands are torch tensors on the scorer's GPU; a tensor whose last dimension is not contiguous is copied, any row stride is
taken as it is.  Every call runs on the GPU's current stream, allocates its outputs and its workspace there with torch's
allocator (so it can be captured into a graph) and does not synchronise.  Gradients are results of their own, not of autograd:
tensors that require one are refused while autograd records, those with a tangent always (torch.no_grad does not stop
forward-mode differentiation)."""
import ctypes
from collections import namedtuple

from . import _lib

F32, BF16, MXFP4 = 0, 1, 2
MAX_FACTORS = 256            # IFR_MAX_FACTORS
MAX_ROWS, MAX_CATALOGUE, MAX_LENGTH = 1 << 23, 1 << 28, 1 << 30

_KINDS = {"logistic": 0, "hinge": 1, "squared": 2}
_REDUCTIONS = {"sum": 0, "row": 1, "batch": 2}

PreferenceLoss = namedtuple("PreferenceLoss", "loss h d_chosen d_rejected")
PolicyLoss = namedtuple("PolicyLoss", "loss kl clipped d_logp")


class MxFp4Matrix:
    """A matrix [n, k] in 4-bit microscaled floating point (OCP MX: E2M1 elements, a power of two per 32 columns): `codes` uint8
    [n, 16 * ceil(k / 32)], element 2j of a row in the low half of byte j, and `scales` uint8 [n, ceil(k / 32)], exponent + 127
    (255: the block stands for NaN).  17/32 byte an element."""

    __slots__ = ("codes", "scales", "k")

    def __init__(self, codes, scales, k):
        import torch
        k = int(k)
        kb = (k + 31) // 32
        if k < 1 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2 or scales.dim() != 2:
            raise ValueError("MxFp4Matrix: codes and scales must be uint8 matrices, k at least 1")
        if codes.shape[1] != 16 * kb or tuple(scales.shape) != (codes.shape[0], kb):
            raise ValueError(f"MxFp4Matrix: k = {k} takes codes [n, {16 * kb}] and scales [n, {kb}]")
        if codes.device != scales.device:
            raise ValueError("MxFp4Matrix: codes and scales must be on one device")
        self.codes, self.scales, self.k = codes.contiguous(), scales.contiguous(), k
        if self.codes.data_ptr() % 16:
            self.codes = self.codes.clone()

    @classmethod
    def _of(cls, codes, scales, k):
        q = cls.__new__(cls)                     # fresh from quantize_mxfp4: nothing to check
        q.codes, q.scales, q.k = codes, scales, k
        return q

    @property
    def shape(self):
        return (self.codes.shape[0], self.k)

    @property
    def device(self):
        return self.codes.device


def _ptr(t):
    return None if t is None else t.data_ptr()


def _name(dtype):
    return str(dtype).replace("torch.", "")


def _refuse(t, name, dtypes, shape, device):
    """The refusal of a tensor that `_matrix` or `_vector` does not take."""
    import torch
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(_name(d) for d in dtypes)}, not {_name(t.dtype)}")
    if t.dim() != len(shape) and len(shape) == 2:
        raise ValueError(f"{name} must be a matrix, not {t.dim()}-dimensional")
    if t.dim() != len(shape) or any(w is not None and w != h for w, h in zip(shape, t.shape)):
        raise ValueError(f"{name} must be [{', '.join('any' if w is None else str(w) for w in shape)}], not {list(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the scorer on {device}")
    raise ValueError(f"{name} requires a gradient: autograd does not see this call, pass {name}.detach() and use the gradients it returns")


def _recorded():
    import torch
    return torch.is_grad_enabled()


def _refuse_tangents(**tensors):
    """ValueError if one of them carries a tangent of forward-mode differentiation."""
    import torch
    ad = torch.autograd.forward_ad
    if ad._current_level < 0:                    # no level is open
        return
    for name, t in tensors.items():
        if isinstance(t, torch.Tensor) and ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name} carries a tangent: forward-mode differentiation does not see this call, pass the primal of unpack_dual({name})")


def _matrix(t, name, dtypes, cols=None, rows=None, device=None):
    """(`t`, elements from one row to the next): a matrix with contiguous rows at least its width apart -- a single row reaches as far as it
    is wide; ValueError / TypeError where it is not what `name` is."""
    try:
        n, w = t.shape
        fine = t.dtype in dtypes and (rows is None or n == rows) and (cols is None or w == cols) and (device is None or t.device == device)
    except (AttributeError, TypeError, ValueError):
        fine = False
    if not fine or t.requires_grad and _recorded():
        _refuse(t, name, dtypes, (rows, cols), device)
    down, across = t.stride()
    if across == 1 and down >= w and n > 1:
        return t, down
    if (across == 1 or w <= 1) and n <= 1:
        return t, w
    return t.contiguous(), w


def _vector(t, name, n, device=None):
    """None, or `t` as a contiguous vector of n fp32 values."""
    if t is None:
        return None
    import torch
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.float32 or t.shape != (n,) or (device is not None and t.device != device) or t.requires_grad and _recorded():
        _refuse(t, name, (torch.float32,), (n,), device)
    return t.contiguous()


NONE = (None, 0)


def _optional(t, *args):
    return NONE if t is None else _matrix(t, *args)


def check_catalogue(X, V, ids, ibase, scale, device=None, extra=()):
    """What the log-probability calls take, ready for the library -- (X, row stride), (V, row stride), (ids, row stride), ibase -- or the refusal."""
    import torch
    _refuse_tangents(X=X, V=V, ibase=ibase)
    if isinstance(X, MxFp4Matrix) != isinstance(V, MxFp4Matrix):
        raise TypeError("X and V must both be tensors or both be MxFp4Matrix")
    if isinstance(X, MxFp4Matrix):
        if X.k != V.k:
            raise ValueError(f"X has {X.k} factors, V {V.k}")
        for name, q in (("X", X), ("V", V)):
            if device is not None and q.device != device:
                raise ValueError(f"{name} is on {q.device}, the scorer on {device}")
        ldx = ldv = 0
    else:
        X, ldx = _matrix(X, "X", (torch.float32, torch.bfloat16), device=device)
        V, ldv = _matrix(V, "V", (X.dtype,), cols=X.shape[1], device=device)
    n, k = X.shape
    n_items = V.shape[0]
    if not 1 <= k <= MAX_FACTORS:
        raise ValueError(f"k must be in [1, {MAX_FACTORS}], not {k}")
    if n > MAX_ROWS or not 1 <= n_items <= MAX_CATALOGUE:
        raise ValueError(f"at most {MAX_ROWS} rows of X and 1 ... {MAX_CATALOGUE} rows of V")
    scale = float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError("scale must be positive, in [1e-30, 1e30]")
    return (X, ldx), (V, ldv), _matrix(ids, "ids", (torch.int32,), rows=n, device=device), _vector(ibase, "ibase", n_items, device)


def check_preference(chosen, rejected, ref_chosen, ref_rejected, mask_chosen, mask_rejected, weight, beta, kind, label_smoothing, margin, device=None):
    """What `preference_loss` takes, ready for the library -- six (matrix, row stride), weight -- or the refusal."""
    import torch
    _refuse_tangents(chosen=chosen, rejected=rejected, ref_chosen=ref_chosen, ref_rejected=ref_rejected, weight=weight)
    f32, masks = (torch.float32,), (torch.bool, torch.uint8)
    c = _matrix(chosen, "chosen", f32, None, None, device)
    n, wc = c[0].shape
    r = _matrix(rejected, "rejected", f32, None, n, device)
    wr = r[0].shape[1]
    if wc > MAX_LENGTH or wr > MAX_LENGTH:
        raise ValueError(f"a slate has at most {MAX_LENGTH} places")
    if (ref_chosen is None) != (ref_rejected is None):
        raise ValueError("a reference needs both ref_chosen and ref_rejected")
    matrices = (c, r, _optional(ref_chosen, "ref_chosen", f32, wc, n, device), _optional(ref_rejected, "ref_rejected", f32, wr, n, device),
                _optional(mask_chosen, "mask_chosen", masks, wc, n, device), _optional(mask_rejected, "mask_rejected", masks, wr, n, device))
    if kind not in _KINDS:
        raise ValueError("kind must be 'logistic', 'hinge' or 'squared'")
    if not 1e-30 <= float(beta) <= 1e30:
        raise ValueError("beta must be positive, in [1e-30, 1e30]")
    if not 0.0 <= float(label_smoothing) < 0.5:
        raise ValueError("label_smoothing must be in [0, 1/2)")
    if label_smoothing and kind != "logistic":
        raise ValueError("label_smoothing needs kind='logistic'")
    if not abs(float(margin)) < 1e30:
        raise ValueError("margin must be finite")
    return matrices, _vector(weight, "weight", n, device)


def check_policy(logp, old_logp, advantages, ref_logp, mask, weight, clip_low, clip_high, kl_coef, reduction, device=None):
    """What `policy_loss` takes, ready for the library -- four (matrix, row stride), advantages, weight -- or the refusal."""
    import torch
    _refuse_tangents(logp=logp, old_logp=old_logp, advantages=advantages, ref_logp=ref_logp, weight=weight)
    f32 = (torch.float32,)
    x = _matrix(logp, "logp", f32, None, None, device)
    n, width = x[0].shape
    if width > MAX_LENGTH:
        raise ValueError(f"a row has at most {MAX_LENGTH} places")
    matrices = (x, _matrix(old_logp, "old_logp", f32, width, n, device), _optional(ref_logp, "ref_logp", f32, width, n, device),
                _optional(mask, "mask", (torch.bool, torch.uint8), width, n, device))
    if advantages is None:
        raise TypeError("advantages must be a torch tensor")
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be 'sum', 'row' or 'batch'")
    if not 0.0 <= float(clip_low) < 1.0 or not 0.0 <= float(clip_high) < 1e30:
        raise ValueError("clip_low must be in [0, 1) and clip_high at least 0")
    if not abs(float(kl_coef)) < 1e30:
        raise ValueError("kl_coef must be finite")
    if kl_coef and ref_logp is None:
        raise ValueError("kl_coef needs ref_logp")
    return matrices, _vector(advantages, "advantages", n, device), _vector(weight, "weight", n, device)


def _refuse_out(out):
    """TypeError / ValueError where `out` is not a tensor, or one whose history would not know of what is written."""
    import torch
    if not isinstance(out, torch.Tensor):
        raise TypeError("out must be a torch tensor")
    if out.requires_grad and _recorded():
        raise ValueError("out requires a gradient: autograd does not see this call")
    _refuse_tangents(out=out)


class CatalogueOps:
    """The catalogue operators of `HipScorer` (engine.py), which supplies `_lib`, `_h`, `device` and `_check`."""

    def _workspace(self, like, fn, key, *args):
        """(workspace where `like` lies, bytes) of a call; `key`: the sizes its length depends on, remembered."""
        import torch
        known = self.__dict__.setdefault("_workspace_bytes", {})
        need = known.get(key)
        if need is None:
            value = ctypes.c_int64(0)
            self._check(fn(self._h, *args, ctypes.byref(value)))
            need = value.value
            if len(known) >= 256:
                known.clear()
            known[key] = need
        return like.new_empty(max(1, need), dtype=torch.uint8), need

    def _stream_of(self):
        """The current stream's handle (the call behind torch.cuda.current_stream, without the object around it)."""
        import torch
        return torch._C._cuda_getCurrentRawStream(self.device.index)

    # ------------------------------------------------------------------ 4-bit model
    def quantize_mxfp4(self, X):
        """`X` [n, k] (fp32 or bf16) as an MxFp4Matrix: per block of 32 columns the exponent floor(log2 max|v|) - 2 (at least -127)
        and elements rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 times it, ties to the even code, at most 6."""
        import torch
        _refuse_tangents(X=X)
        X, ld = _matrix(X, "X", (torch.float32, torch.bfloat16), None, None, self.device)
        n, k = X.shape
        if k < 1:
            raise ValueError("X must have at least one column")
        kb = (k + 31) // 32
        codes = X.new_empty((n, 16 * kb), dtype=torch.uint8)
        scales = X.new_empty((n, kb), dtype=torch.uint8)
        self._check(self._lib.ifr_mxfp4_quantize(self._h, _ptr(X), F32 if X.dtype == torch.float32 else BF16, n, k, ld,
                                                 _ptr(codes), _ptr(scales), self._stream_of()))
        return MxFp4Matrix._of(codes, scales, k)

    def dequantize_mxfp4(self, q, out=None):
        """The fp32 values [n, k] that an MxFp4Matrix stands for."""
        import torch
        if not isinstance(q, MxFp4Matrix) or q.device != self.device:
            raise ValueError(f"dequantize_mxfp4 takes an MxFp4Matrix on {self.device}")
        out, ld = self._out(out, q.shape, torch.float32, q.codes)
        self._check(self._lib.ifr_mxfp4_dequantize(self._h, _ptr(q.codes), _ptr(q.scales), q.shape[0], q.k, _ptr(out), ld,
                                                   self._stream_of()))
        return out

    def _out(self, out, shape, dtype, like):
        """(output, row stride)"""
        if out is None:
            return like.new_empty(shape, dtype=dtype), shape[1]
        _refuse_out(out)
        if tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != self.device or (out.numel() and (
                out.stride(1) != 1 and out.shape[1] > 1 or out.shape[0] > 1 and out.stride(0) < out.shape[1])):
            raise ValueError(f"out must be {_name(dtype)} {list(shape)} on {self.device} with contiguous rows")
        return out, out.stride(0) if shape[0] > 1 else shape[1]

    def score_mxfp4(self, X, V, ubase=None, ibase=None, out=None, dtype=None):
        """Score rows [n, n_items] of a 4-bit model, beside `score_dense`: (ibase + ubase) + <X[u], V[i]>, fp32 sums rounded once to
        `dtype` (float32, the default, or bfloat16)."""
        import torch
        if not isinstance(X, MxFp4Matrix) or not isinstance(V, MxFp4Matrix):
            raise TypeError("score_mxfp4 takes two MxFp4Matrix (quantize_mxfp4)")
        if X.k != V.k:
            raise ValueError(f"X has {X.k} factors, V {V.k}")
        if X.k > MAX_FACTORS or X.shape[0] > MAX_ROWS or not 1 <= V.shape[0] <= MAX_CATALOGUE:
            raise ValueError(f"score_mxfp4: at most {MAX_FACTORS} factors, {MAX_ROWS} rows of X, 1 ... {MAX_CATALOGUE} rows of V")
        if X.device != self.device or V.device != self.device:
            raise ValueError(f"X and V must be on {self.device}")
        _refuse_tangents(ubase=ubase, ibase=ibase)
        if out is not None:
            _refuse_out(out)
        dtype = torch.float32 if dtype is None and out is None else out.dtype if dtype is None else dtype
        if dtype not in (torch.float32, torch.bfloat16):
            raise TypeError("score_mxfp4 writes float32 or bfloat16")
        n, n_items = X.shape[0], V.shape[0]
        ubase, ibase = _vector(ubase, "ubase", n, self.device), _vector(ibase, "ibase", n_items, self.device)
        out, ld = self._out(out, (n, n_items), dtype, V.codes)
        self._check(self._lib.ifr_mxfp4_scores(self._h, _ptr(X.codes), _ptr(X.scales), n, _ptr(V.codes), _ptr(V.scales), n_items, X.k, _ptr(ubase),
                                               _ptr(ibase), _ptr(out), F32 if dtype == torch.float32 else BF16, ld, self._stream_of()))
        return out

    # ------------------------------------------------------------------ log-probabilities
    def _catalogue(self, X, ldx, V, ldv, ibase, scale):
        import torch
        n, k = X.shape
        if isinstance(X, MxFp4Matrix):
            return _lib.Catalogue(X.codes.data_ptr(), V.codes.data_ptr(), X.scales.data_ptr(), V.scales.data_ptr(), _ptr(ibase), n, V.shape[0], 0, 0, k, MXFP4,
                                  float(scale))
        return _lib.Catalogue(X.data_ptr(), V.data_ptr(), None, None, _ptr(ibase), n, V.shape[0], ldx, ldv, k, F32 if X.dtype is torch.float32 else BF16, float(scale))

    def catalogue_logprob(self, X, V, ids, ibase=None, scale=1.0):
        """(logp [n, m], lse [n]), fp32: logp[u, j] = z[u, ids[u, j]] - lse[u] with z[u, i] = scale * (<X[u], V[i]> + ibase[i]) and
        lse[u] = log sum_i exp z[u, i] over the whole catalogue.  X [n, k] and V [n_items, k]: both fp32, both bf16, or both
        MxFp4Matrix (a frozen model); ids int32 [n, m], negative = an empty place (logp 0; an id past the catalogue gives NaN);
        an ibase of -inf takes an item out.  The n x n_items scores are not stored."""
        import torch
        (X, ldx), (V, ldv), (ids, ld_ids), ibase = check_catalogue(X, V, ids, ibase, scale, self.device)
        n, m = ids.shape
        c = self._catalogue(X, ldx, V, ldv, ibase, scale)
        logp, lse = ids.new_empty((n, m), dtype=torch.float32), ids.new_empty(n, dtype=torch.float32)
        ws, need = self._workspace(ids, self._lib.ifr_catalogue_logprob_workspace, (c.n, c.n_items, c.k, c.dtype), ctypes.byref(c))
        self._check(self._lib.ifr_catalogue_logprob(self._h, ctypes.byref(c), _ptr(ids), m, ld_ids, _ptr(logp), max(m, 1), _ptr(lse),
                                                    _ptr(ws), need, self._stream_of()))
        return logp, lse

    def catalogue_logprob_backward(self, X, V, ids, lse, dlogp, ibase=None, scale=1.0, want=("X", "V", "ibase")):
        """(dX, dV, dibase) for the upstream gradient dlogp [n, m] of `catalogue_logprob`'s logp, with its lse: dX and dV in the
        operands' type, dibase fp32 (None where there is no ibase, or where `want` leaves one out).  The same call gives the
        same bits."""
        import torch
        if isinstance(X, MxFp4Matrix) or isinstance(V, MxFp4Matrix):
            raise TypeError("a 4-bit model has no gradient")
        if set(want) - {"X", "V", "ibase"}:
            raise ValueError("want holds 'X', 'V' and 'ibase'")
        (X, ldx), (V, ldv), (ids, ld_ids), ibase = check_catalogue(X, V, ids, ibase, scale, self.device)
        n, m = ids.shape
        _refuse_tangents(lse=lse, dlogp=dlogp)
        dlogp, ld_dlogp = _matrix(dlogp, "dlogp", (torch.float32,), m, n, self.device)
        if lse is None:
            raise TypeError("lse must be a torch tensor")
        lse = _vector(lse, "lse", n, self.device)
        dX = X.new_empty(X.shape) if "X" in want else None
        dV = (V.new_empty if n else V.new_zeros)(V.shape) if "V" in want else None
        db = (ibase.new_empty if n else ibase.new_zeros)(V.shape[0]) if "ibase" in want and ibase is not None else None
        c = self._catalogue(X, ldx, V, ldv, ibase, scale)
        ws, need = self._workspace(ids, self._lib.ifr_catalogue_logprob_backward_workspace, (c.n, c.n_items, c.k, c.dtype, m, dX is None, dV is None, db is None),
                                   ctypes.byref(c), m, int(dX is not None), int(dV is not None), int(db is not None))
        k = X.shape[1]
        self._check(self._lib.ifr_catalogue_logprob_backward(self._h, ctypes.byref(c), _ptr(ids), m, ld_ids, _ptr(lse), _ptr(dlogp), ld_dlogp, _ptr(dX), k,
                                                             _ptr(dV), k, _ptr(db), _ptr(ws), need, self._stream_of()))
        return dX, dV, db

    # ------------------------------------------------------------------ losses
    def preference_loss(self, chosen, rejected, ref_chosen=None, ref_rejected=None, mask_chosen=None, mask_rejected=None, beta=0.1, kind="logistic",
                        label_smoothing=0.0, margin=0.0, average=False, weight=None):
        """PreferenceLoss(loss [n], h [n], d_chosen, d_rejected) of n pairs of slates from the log-probabilities of their items
        [n, places]: h = beta ((C - R) - (Cr - Rr)) - margin with C, R the sums (`average`: means) over the masks of the chosen and
        the rejected slate and Cr, Rr those of a frozen reference.  kind "logistic": log(1 + exp(-h)), smoothed towards the other
        order by label_smoothing; "hinge": max(0, 1 - h); "squared": ((h - 1/2) / beta)^2.  d_chosen and d_rejected are the
        gradients of sum(weight * loss), weight 1 unless given.  Slates of one item with beta = 1 and no reference are BPR's criterion."""
        (c, r, rc, rr, mc, mr), weight = check_preference(chosen, rejected, ref_chosen, ref_rejected, mask_chosen, mask_rejected, weight, beta, kind,
                                                          label_smoothing, margin, self.device)
        n, wc = c[0].shape
        wr = r[0].shape[1]
        loss, h, d_chosen, d_rejected = c[0].new_empty(n), c[0].new_empty(n), c[0].new_empty((n, wc)), c[0].new_empty((n, wr))
        p = _lib.Preference(n, wc, wr, _KINDS[kind], 1 if average else 0, c[0].data_ptr(), r[0].data_ptr(), _ptr(rc[0]), _ptr(rr[0]), _ptr(mc[0]), _ptr(mr[0]),
                            _ptr(weight), loss.data_ptr(), h.data_ptr(), d_chosen.data_ptr(), d_rejected.data_ptr(), c[1], r[1], rc[1], rr[1], mc[1], mr[1],
                            wc, wr, float(beta), float(margin), float(label_smoothing))
        self._check(self._lib.ifr_preference_loss(self._h, ctypes.byref(p), self._stream_of()))
        return PreferenceLoss(loss, h, d_chosen, d_rejected)

    def policy_loss(self, logp, old_logp, advantages, ref_logp=None, mask=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, reduction="row", weight=None):
        """PolicyLoss(loss [n], kl [n], clipped int32 [n], d_logp [n, places]) of n rows of choices sampled from an older policy: per
        place of the mask -A r, r = exp(logp - old_logp) clipped to [1 - clip_low, 1 + clip_high] where that raises the loss, plus
        kl_coef (exp(q) - q - 1), q = ref_logp - logp.  loss[row] = c * the sum over its places with c = weight (1 unless given) times
        1 ("sum"), 1 / places of the row ("row") or 1 / places of the batch ("batch"); d_logp is the gradient of sum(loss).  kl is the row's
        mean (None without ref_logp), clipped its number of clipped places."""
        import torch
        (x, old, ref, m), advantages, weight = check_policy(logp, old_logp, advantages, ref_logp, mask, weight, clip_low, clip_high, kl_coef, reduction, self.device)
        n, width = x[0].shape
        loss, kl, d_logp = x[0].new_empty(n), None if ref_logp is None else x[0].new_empty(n), x[0].new_empty((n, width))
        clipped = x[0].new_empty(n, dtype=torch.int32)
        p = _lib.Policy(n, width, _REDUCTIONS[reduction], x[0].data_ptr(), old[0].data_ptr(), _ptr(ref[0]), advantages.data_ptr(), _ptr(weight), _ptr(m[0]),
                        loss.data_ptr(), _ptr(kl), clipped.data_ptr(), d_logp.data_ptr(), x[1], old[1], ref[1], m[1], width, float(clip_low), float(clip_high),
                        float(kl_coef))
        ws, need = (None, 0) if mask is None or reduction != "batch" else self._workspace(clipped, self._lib.ifr_policy_loss_workspace, ("policy", not p.mask), ctypes.byref(p))
        self._check(self._lib.ifr_policy_loss(self._h, ctypes.byref(p), _ptr(ws), need, self._stream_of()))
        return PolicyLoss(loss, kl, clipped, d_logp)
