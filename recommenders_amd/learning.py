"""Learning a factor model from preferences and from rewards, on the device.

The reference trains BPR with a pairwise criterion on sampled item pairs (cornac/models/bpr/recom_bpr.pyx:208-269) and has no
counterpart of what follows.  Here the model is a policy: user u picks item i with probability softmax_i(scale * score(u, i)) over
the whole catalogue (a user's own bias shifts all of them and drops out).  `fit_preferences` learns from pairs of slates of which
one was preferred, `fit_policy` from slates that were shown and what they earned; both take plain gradient steps on the user
factors, the item factors and the item biases, every part of a step one call of the engine: log-probabilities, loss with its gradient,
gradient of the log-probabilities.  A frozen reference model keeps the learned one near: its two factor matrices stay on the device
in fp32, or in 4 bits (`reference_precision="mxfp4"`, an eighth of the memory)."""
import numpy as np


class CatalogueLearningMixin:
    """`log_prob`, `fit_preferences` and `fit_policy` for a dot-product model.  A concrete class supplies `_hip_learned`: the names of
    its user factors, item factors and item biases (None: the model has none)."""

    def _hip_learned(self):
        raise NotImplementedError

    # ------------------------------------------------------------------ device state
    def _hip_ops(self):
        ops = getattr(self, "_hip_ops_engine", None)
        if ops is None:
            from .engine import HipScorer
            ops = self._hip_ops_engine = HipScorer(self.hip_device)
        return ops

    def hip_invalidate(self):
        super().hip_invalidate()
        ops, self._hip_ops_engine = getattr(self, "_hip_ops_engine", None), None
        if ops is not None:
            ops.close()

    def _hip_parameters(self):
        """(U, V, item biases or None) as new fp32 tensors on the model's GPU."""
        import torch
        dev = self._hip_ops().device
        out = []
        for name in self._hip_learned():
            a = None if name is None else getattr(self, name)
            out.append(None if a is None else torch.tensor(np.asarray(a, np.float32), device=dev))
        return out

    def _hip_frozen(self, parameters, precision):
        """A copy that stays as it is: (users, items, item biases), the factors in fp32 or in 4 bits."""
        if precision not in ("f32", "mxfp4"):
            raise ValueError("the precision of a frozen model must be 'f32' or 'mxfp4'")
        U, V, b = parameters
        if precision == "mxfp4":
            ops = self._hip_ops()
            return ops.quantize_mxfp4(U), ops.quantize_mxfp4(V), None if b is None else b.clone()
        return U.clone(), V.clone(), None if b is None else b.clone()

    @staticmethod
    def _hip_rows(U, rows):
        from .catalogue import MxFp4Matrix
        return MxFp4Matrix(U.codes[rows], U.scales[rows], U.k) if isinstance(U, MxFp4Matrix) else U[rows]

    def _hip_store(self, parameters):
        """Learned parameters back into the model: its device copies and cached rankings are of the old ones."""
        for name, t in zip(self._hip_learned(), parameters):
            if name is not None and t is not None:
                setattr(self, name, t.cpu().numpy())
        self.hip_invalidate()
        self.ranked_items, self.item_scores, self.item_scores_mapped_indices = {}, {}, {}

    # ------------------------------------------------------------------ checks
    def _hip_users(self, users):
        if any(getattr(self, name) is None for name in self._hip_learned()[:2]):
            raise RuntimeError(f"{self.name} has no factors: pass init_params")
        u = np.asarray(users)
        n = len(getattr(self, self._hip_learned()[0]))
        if u.ndim != 1 or u.dtype.kind not in "iu":
            raise ValueError("users must be a vector of user indices")
        if u.size and (u.min() < 0 or u.max() >= n):
            raise IndexError(f"user index {int(u.min()) if u.min() < 0 else int(u.max())} is out of bounds for {n} users")
        return u.astype(np.int64)

    def _hip_slates(self, items, n, name):
        s = np.asarray(items)
        n_items = len(getattr(self, self._hip_learned()[1]))
        s = s.reshape(-1, 1) if s.ndim == 1 else s
        if s.ndim != 2 or len(s) != n or (s.size and s.dtype.kind not in "iu"):
            raise ValueError(f"{name} must be [{n}, places] item indices, -1 for an empty place")
        if s.size and (s.min() < -1 or s.max() >= n_items):
            raise IndexError(f"{name}: item index {int(s.min()) if s.min() < -1 else int(s.max())} is out of bounds for {n_items} items")
        return s.astype(np.int32)

    @staticmethod
    def _hip_schedule(n, batch_size, epochs, learning_rate, reg, seed):
        if int(batch_size) < 1 or int(epochs) < 0 or not learning_rate > 0 or reg < 0:
            raise ValueError("batch_size must be at least 1, epochs at least 0, learning_rate positive, reg at least 0")
        rng = np.random.default_rng(seed)
        for epoch in range(int(epochs)):
            order = rng.permutation(n)
            for b in range(0, n, int(batch_size)):
                yield epoch, order[b:b + int(batch_size)]

    def _hip_step(self, parameters, rows, ids, lse, dlogp, scale, learning_rate, reg):
        """One gradient step: the users of the batch, all items, all biases."""
        U, V, b = parameters
        X = U[rows]
        dX, dV, db = self._hip_ops().catalogue_logprob_backward(X, V, ids, lse, dlogp, ibase=b, scale=scale)
        if reg:
            dX += reg * X
            dV += reg * V
        U.index_put_((rows,), -learning_rate * dX, accumulate=True)       # a user may stand in a batch more than once
        V.sub_(dV, alpha=learning_rate)
        if b is not None:
            b.sub_(db, alpha=learning_rate)

    # ------------------------------------------------------------------ public
    def log_prob(self, user_indices, items, scale=1.0, precision="f32"):
        """log p(item | user) [n, places], fp32, for `items` [n, places] (-1: an empty place, 0) under the softmax of scale * score
        over the whole catalogue.  precision="mxfp4": of the model with its factors in 4 bits."""
        import torch
        users = self._hip_users(user_indices)
        ids = self._hip_slates(items, len(users), "items")
        ops = self._hip_ops()
        U, V, b = self._hip_frozen(self._hip_parameters(), precision)
        rows = torch.as_tensor(users, device=ops.device)
        logp, _ = ops.catalogue_logprob(self._hip_rows(U, rows), V, torch.as_tensor(ids, device=ops.device), ibase=b, scale=scale)
        return logp.cpu().numpy()

    def fit_preferences(self, users, chosen, rejected, learning_rate=0.05, epochs=1, batch_size=4096, beta=1.0, kind="logistic", label_smoothing=0.0,
                        margin=0.0, average=False, reference=False, reference_precision="f32", scale=1.0, reg=0.0, seed=None):
        """Learns from pairs: `users` [n], `chosen` [n, places] and `rejected` [n, places'] item indices (-1: an empty place) -- the slate the
        user preferred and the one passed over.  The loss is `HipScorer.preference_loss` of their log-probabilities, averaged over a batch;
        reference=True takes log ratios against the model as it is now.  One-item slates with beta = 1 are BPR's criterion.  Returns the
        mean loss of every epoch; the learned parameters replace the model's arrays (the caller's init_params stay as they are)."""
        import torch
        users = self._hip_users(users)
        n = len(users)
        chosen, rejected = self._hip_slates(chosen, n, "chosen"), self._hip_slates(rejected, n, "rejected")
        ops, places = self._hip_ops(), chosen.shape[1]
        parameters = self._hip_parameters()
        frozen = self._hip_frozen(parameters, reference_precision) if reference else None
        ids = torch.as_tensor(np.concatenate([chosen, rejected], 1), device=ops.device)
        rows = torch.as_tensor(users, device=ops.device)
        totals = [torch.zeros((), dtype=torch.float64, device=ops.device) for _ in range(int(epochs))]
        for epoch, batch in self._hip_schedule(n, batch_size, epochs, learning_rate, reg, seed):
            at = torch.as_tensor(batch, device=ops.device)
            r, i = rows[at], ids[at]
            logp, lse = ops.catalogue_logprob(parameters[0][r], parameters[1], i, ibase=parameters[2], scale=scale)
            ref = None
            if frozen is not None:
                ref, _ = ops.catalogue_logprob(self._hip_rows(frozen[0], r), frozen[1], i, ibase=frozen[2], scale=scale)
            mask = i >= 0
            weight = torch.full((len(batch),), 1.0 / len(batch), device=ops.device)
            loss = ops.preference_loss(logp[:, :places], logp[:, places:], None if ref is None else ref[:, :places], None if ref is None else ref[:, places:],
                                       mask[:, :places], mask[:, places:], beta=beta, kind=kind, label_smoothing=label_smoothing, margin=margin,
                                       average=average, weight=weight)
            self._hip_step(parameters, r, i, lse, torch.cat([loss.d_chosen, loss.d_rejected], 1), scale, learning_rate, reg)
            totals[epoch] += loss.loss.double().sum()
        self._hip_store(parameters)
        return [float(t) / max(n, 1) for t in totals]

    def fit_policy(self, users, slates, advantages, old_log_prob=None, learning_rate=0.05, epochs=1, batch_size=4096, clip_low=0.2, clip_high=0.2, kl_coef=0.0,
                   reference_precision="f32", scale=1.0, reg=0.0, seed=None):
        """Learns from shown slates: `users` [n], `slates` [n, places] (-1: an empty place), `advantages` [n] -- what each earned above
        expectation -- and `old_log_prob` [n, places], the log-probabilities under the policy that drew them (the model as it is now, if
        left out).  The loss is `HipScorer.policy_loss`, averaged over the places of a slate and the slates of a batch, with kl_coef
        times the divergence from the model as it is now.  Returns the mean loss of every epoch."""
        import torch
        users = self._hip_users(users)
        n = len(users)
        slates = self._hip_slates(slates, n, "slates")
        A = np.asarray(advantages, np.float32)
        if A.shape != (n,):
            raise ValueError(f"advantages must be [{n}]")
        ops = self._hip_ops()
        parameters = self._hip_parameters()
        frozen = self._hip_frozen(parameters, reference_precision) if kl_coef else None
        if old_log_prob is None:
            old_log_prob = self.log_prob(users, slates, scale=scale)
        old = np.asarray(old_log_prob, np.float32)
        if old.shape != slates.shape:
            raise ValueError(f"old_log_prob must be {list(slates.shape)}")
        dev = lambda a: torch.as_tensor(a, device=ops.device)
        rows, ids, A, old = dev(users), dev(slates), dev(A), dev(old)
        totals = [torch.zeros((), dtype=torch.float64, device=ops.device) for _ in range(int(epochs))]
        for epoch, batch in self._hip_schedule(n, batch_size, epochs, learning_rate, reg, seed):
            at = dev(batch)
            r, i = rows[at], ids[at]
            logp, lse = ops.catalogue_logprob(parameters[0][r], parameters[1], i, ibase=parameters[2], scale=scale)
            ref = None
            if frozen is not None:
                ref, _ = ops.catalogue_logprob(self._hip_rows(frozen[0], r), frozen[1], i, ibase=frozen[2], scale=scale)
            weight = torch.full((len(batch),), 1.0 / len(batch), device=ops.device)
            loss = ops.policy_loss(logp, old[at], A[at], ref_logp=ref, mask=i >= 0, clip_low=clip_low, clip_high=clip_high, kl_coef=kl_coef, reduction="row",
                                   weight=weight)
            self._hip_step(parameters, r, i, lse, loss.d_logp, scale, learning_rate, reg)
            totals[epoch] += loss.loss.double().sum() * len(batch)
        self._hip_store(parameters)
        return [float(t) / max(n, 1) for t in totals]
