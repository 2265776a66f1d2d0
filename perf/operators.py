"""The catalogue operators as a user's program meets them: cases, inputs, plain forms and exact values.

Five operators: 4-bit microscaled quantisation, score rows from a 4-bit catalogue, log-probabilities over the catalogue
(forward, and with gradients), the preference loss on paired log ratios and the clipped policy loss with a KL term.
`own` chooses between elementary torch operations and the calls of this package."""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # the factors of one small model, and of a catalogue of a million items, brought into 4 bits
        {"name": "quantize model", "op": "quantize", "n": 1682, "k": 50, "dtype": "f32"},
        {"name": "quantize catalogue", "op": "quantize", "n": 1000000, "k": 128, "dtype": "f32"},
        # one user's scores over a film catalogue (a serving request), and a batch over a million items
        {"name": "scores of one user", "op": "scores", "n": 1, "items": 26744, "k": 128, "dtype": "f32", "out": "f32", "bias": True},
        {"name": "scores of a batch", "op": "scores", "n": 1000, "items": 1000000, "k": 128, "dtype": "f32", "out": "bf16", "bias": False},
        # the probability of one user's slate out of a million items
        {"name": "logprob of one slate", "op": "logprob", "n": 1, "items": 1000000, "k": 128, "m": 10, "dtype": "f32", "bias": True, "grad": False},
        # a frozen reference model kept in 4 bits
        {"name": "logprob of a reference", "op": "logprob", "n": 2048, "items": 125000, "k": 128, "m": 10, "dtype": "mxfp4", "bias": True, "grad": False},
        # a training step over a film catalogue, and the largest: a million items in bfloat16
        {"name": "logprob step", "op": "logprob", "n": 2048, "items": 26744, "k": 200, "m": 20, "dtype": "f32", "bias": True, "grad": True},
        {"name": "logprob step, large", "op": "logprob", "n": 2048, "items": 1000000, "k": 128, "m": 2, "dtype": "bf16", "bias": False, "grad": True},
        # pairs of recommended slates of ten, and of long candidate pools
        {"name": "preference of slates", "op": "preference", "n": 64, "chosen": 10, "rejected": 10, "kind": "logistic", "average": False, "ref": True},
        {"name": "preference of pools", "op": "preference", "n": 16384, "chosen": 500, "rejected": 1000, "kind": "logistic", "average": True, "ref": True},
        # slates sampled from a policy, and long sequences of choices
        {"name": "policy of slates", "op": "policy", "n": 256, "len": 10, "reduction": "row", "kl": 0.05},
        {"name": "policy of sequences", "op": "policy", "n": 4096, "len": 8191, "reduction": "batch", "kl": 0.05},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "scores", "logprob", "logprob", "preference", "policy"])
    if op == "quantize":
        return {"op": op, "n": _log(rng, 1, 1000000), "k": rng.randint(1, 128), "dtype": rng.choice(["f32", "bf16"])}
    if op == "scores":
        items = _log(rng, 100, 1000000)
        return {"op": op, "n": _log(rng, 1, min(4096, 1000000000 // items)), "items": items, "k": rng.randint(1, 128),
                "dtype": rng.choice(["f32", "bf16"]), "out": rng.choice(["f32", "bf16"]), "bias": rng.random() < 0.5}
    if op == "logprob":
        items, k = _log(rng, 100, 1000000), rng.choice([rng.randint(1, 128), rng.randint(129, 256)])
        most = 2048 * 1000000 * 128 // (items * max(k, 128))
        dtype = rng.choice(["f32", "bf16", "mxfp4"])
        n = _log(rng, 1, min(8192, most // 3 if dtype == "f32" else most))
        return {"op": op, "n": n, "items": items, "k": k, "m": _log(rng, 1, 64), "dtype": dtype,
                "bias": rng.random() < 0.5, "grad": dtype != "mxfp4" and rng.random() < 0.7}
    if op == "preference":
        n = _log(rng, 1, 65536)
        most = min(8192, 16384 * 500 // n)
        return {"op": op, "n": n, "chosen": _log(rng, 1, most), "rejected": _log(rng, 1, most), "kind": rng.choice(["logistic", "hinge", "squared"]),
                "average": rng.random() < 0.5, "ref": rng.random() < 0.7}
    n = _log(rng, 1, 65536)
    return {"op": op, "n": n, "len": _log(rng, 1, min(8192, 4096 * 8191 // n)), "reduction": rng.choice(["sum", "row", "batch"]),
            "kl": rng.choice([0.0, 0.05])}


# ------------------------------------------------------------------ inputs

def _padded_ids(g, n, m, items):
    """Slates of 1 ... m items by popularity (a skewed law, spread over the catalogue), -1 behind a slate's end."""
    r = torch.rand((n, m), generator=g, device=DEV, dtype=torch.float64)
    rank = (items * r ** 3).long().clamp_(max=items - 1)
    step = 7919
    while math.gcd(step, items) != 1:
        step += 2
    ids = (rank * step) % items
    length = torch.randint(1, m + 1, (n, 1), generator=g, device=DEV)
    return torch.where(torch.arange(m, device=DEV)[None, :] < length, ids, -1).to(torch.int32)


def _ragged_mask(g, n, width):
    length = torch.randint(0 if n > 1 else 1, width + 1, (n, 1), generator=g, device=DEV)
    return torch.arange(width, device=DEV)[None, :] < length


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op, n = case["op"], case["n"]
    normal = lambda *shape, s=1.0: torch.randn(shape, generator=g, device=DEV) * s
    st = {"case": case}
    if op == "quantize":
        st["X"] = normal(n, case["k"], s=0.1).to(DTYPES[case["dtype"]])
    elif op == "scores":
        st["X"] = normal(n, case["k"], s=0.1).to(DTYPES[case["dtype"]])
        st["V"] = _pack(normal(case["items"], case["k"], s=0.1))                   # the catalogue is laid out once
        st["ibase"] = normal(case["items"], s=0.01) if case["bias"] else None
    elif op == "logprob":
        X, V = normal(n, case["k"], s=0.4), normal(case["items"], case["k"], s=0.4)
        if case["dtype"] == "mxfp4":
            st["X"], st["V"] = _pack(X), _pack(V)
        else:
            st["X"], st["V"] = X.to(DTYPES[case["dtype"]]), V.to(DTYPES[case["dtype"]])
        st["ibase"] = normal(case["items"], s=0.5) if case["bias"] else None
        st["ids"] = _padded_ids(g, n, case["m"], case["items"])
        if case["grad"]:
            st["dlogp"] = normal(n, case["m"], s=1.0 / n)
    elif op == "preference":
        w = case["chosen"] + case["rejected"]
        logp = -normal(n, w).abs() * 2 - 4                                         # one tensor holds both slates of a pair
        st["logp"] = logp
        st["ref"] = logp + normal(n, w, s=0.3) if case["ref"] else None
        st["mask"] = torch.cat([_ragged_mask(g, n, case["chosen"]), _ragged_mask(g, n, case["rejected"])], 1)
        st["weight"] = torch.full((n,), 1.0 / n, device=DEV)
    else:
        st["logp"] = -normal(n, case["len"]).abs() * 2 - 4
        st["old"] = st["logp"] + normal(n, case["len"], s=0.15)
        st["ref"] = st["logp"] + normal(n, case["len"], s=0.3) if case["kl"] else None
        st["mask"] = _ragged_mask(g, n, case["len"])
        st["adv"] = normal(n)
    return st


# ------------------------------------------------------------------ 4 bits, plain

def _blocks(X):
    """[n, k] as [n, blocks, 32] in 64 bits, zeros behind the last column."""
    n, k = X.shape
    kb = (k + 31) // 32
    Y = torch.zeros((n, kb * 32), dtype=torch.float64, device=X.device)
    Y[:, :k] = X
    return Y.view(n, kb, 32)


def _codes(X):
    """Index into 0, .5, 1, 1.5, 2, 3, 4, 6 (plus 8 for a negative element) and the exponent of every block of 32."""
    Y = _blocks(X)
    top = Y.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top)[1] - 3, torch.full_like(top, -127).int()).clamp(-127, 127)
    y = torch.ldexp(Y.abs(), -e[..., None].int())                                  # 64 bits: a value next to a border stays there
    low, mid = y < 2, y < 4
    code = torch.where(low, torch.round(y * 2), torch.where(mid, torch.round(y) + 2, torch.round(y / 2) + 4)).clamp(max=7)
    return (code + 8 * torch.signbit(Y)).to(torch.uint8), e


def _pack(X):
    """(codes [n, 16 * blocks], element 2j in the low half of byte j; scales [n, blocks], exponent + 127; k)."""
    code, e = _codes(X)
    n = X.shape[0]
    pairs = code.view(n, -1, 2)
    return (pairs[..., 0] | (pairs[..., 1] << 4)).contiguous(), (e + 127).to(torch.uint8), X.shape[1]


def _grid(device, dtype):
    return torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=device, dtype=dtype)


def _values(code, e, k, dtype=torch.float32):
    v = torch.ldexp(_grid(code.device, dtype)[code.long()], e[..., None].int())
    return v.view(code.shape[0], -1)[:, :k]


def _unpack(q, dtype=torch.float32):
    codes, scales, k = q
    n = codes.shape[0]
    code = torch.stack([codes & 15, codes >> 4], -1).view(n, -1, 32)
    return _values(code, scales.int() - 127, k, dtype)


# ------------------------------------------------------------------ plain forms

def _plain_logprob(st):
    c = st["case"]
    if c["dtype"] == "mxfp4":
        X, V = _unpack(st["X"]), _unpack(st["V"])
    else:
        X, V = st["X"].float(), st["V"].float()
    z = X @ V.t()
    if st["ibase"] is not None:
        z += st["ibase"]
    top = z.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    ids = st["ids"].long()
    held = ids >= 0
    at = ids.clamp(min=0)
    out = {"logp": torch.where(held, z.gather(1, at) - lse, 0.0), "lse": lse[:, 0]}
    if c["grad"]:
        grad = torch.where(held, st["dlogp"], 0.0)
        dz = torch.exp(z - lse) * -grad.sum(1, keepdim=True)
        dz.scatter_add_(1, at, grad)
        out["dX"] = (dz @ V).to(st["X"].dtype)
        out["dV"] = (dz.t() @ X).to(st["V"].dtype)
        if st["ibase"] is not None:
            out["dibase"] = dz.sum(0)
    return out


def _plain_preference(st):
    c, w, beta = st["case"], st["weight"], 0.1
    lc = c["chosen"]
    mask = st["mask"]
    diff = st["logp"] if st["ref"] is None else st["logp"] - st["ref"]
    diff = torch.where(mask, diff, 0.0).double()                                    # long sums
    count = torch.stack([mask[:, :lc].sum(1), mask[:, lc:].sum(1)], 1).clamp(min=1) if c["average"] else torch.ones((c["n"], 2), device=DEV)
    h = (beta * (diff[:, :lc].sum(1) / count[:, 0] - diff[:, lc:].sum(1) / count[:, 1])).float()
    if c["kind"] == "logistic":
        loss = torch.log1p(torch.exp(-h.abs())) + torch.clamp(-h, min=0)
        slope = -torch.exp(torch.clamp(-h, max=0)) / (1 + torch.exp(-h.abs()))      # sigmoid(h) - 1
    elif c["kind"] == "hinge":
        loss, slope = torch.clamp(1 - h, min=0), torch.where(h < 1, -1.0, 0.0)
    else:
        loss, slope = ((h - 0.5) / beta) ** 2, 2 * (h - 0.5) / beta ** 2
    part = (w * slope * beta)[:, None] / count
    return {"loss": loss, "h": h, "dchosen": mask[:, :lc] * part[:, :1], "drejected": mask[:, lc:] * -part[:, 1:]}


LOW, HIGH = 0.2, 0.28


def _plain_policy(st):
    c, mask, A = st["case"], st["mask"], st["adv"][:, None]
    count = mask.sum(1, keepdim=True)
    scale = {"sum": torch.ones_like(A), "row": 1.0 / count.clamp(min=1), "batch": (1.0 / count.sum().clamp(min=1)).expand_as(A)}[c["reduction"]]
    d = st["logp"] - st["old"]
    ratio = torch.exp(d)
    over, under = (A > 0) & (d > math.log1p(HIGH)), (A < 0) & (d < math.log1p(-LOW))
    clipped = (over | under) & mask
    term = -A * torch.where(over, 1 + HIGH, torch.where(under, 1 - LOW, ratio))
    grad = torch.where(clipped, 0.0, -A * ratio)
    out = {"clipped": clipped.sum(1).int()}
    if c["kl"]:
        q = st["ref"].double() - st["logp"].double()                                # small differences: 32 bits cancel
        more = torch.expm1(q)
        kl = (more - q).float()
        term = term + c["kl"] * kl
        grad = grad - c["kl"] * more.float()
        out["kl"] = (torch.where(mask, kl, 0.0).sum(1, keepdim=True) / count.clamp(min=1))[:, 0]
    out["loss"] = (torch.where(mask, term, 0.0).double().sum(1, keepdim=True) * scale)[:, 0].float()
    out["dlogp"] = torch.where(mask, grad * scale, 0.0)
    return out


def _plain(st):
    c = st["case"]
    if c["op"] == "quantize":
        return {"values": _values(*_codes(st["X"]), c["k"])}
    if c["op"] == "scores":
        s = _values(*_codes(st["X"]), c["k"]) @ _unpack(st["V"]).t()
        if st["ibase"] is not None:
            s += st["ibase"]
        return {"scores": s.to(DTYPES[c["out"]])}
    return {"logprob": _plain_logprob, "preference": _plain_preference, "policy": _plain_policy}[c["op"]](st)


# ------------------------------------------------------------------ this package

_scorer = None


def _engine():
    global _scorer
    if _scorer is None:
        from recommenders_amd import HipScorer
        _scorer = HipScorer(0)
    return _scorer


def _package(st):
    from recommenders_amd import MxFp4Matrix
    c, sc = st["case"], _engine()
    if c["op"] == "quantize":
        return {"values": sc.dequantize_mxfp4(sc.quantize_mxfp4(st["X"]))}
    if c["op"] == "scores":
        return {"scores": sc.score_mxfp4(sc.quantize_mxfp4(st["X"]), MxFp4Matrix(*st["V"]), ibase=st["ibase"], dtype=DTYPES[c["out"]])}
    if c["op"] == "logprob":
        X, V = (MxFp4Matrix(*st["X"]), MxFp4Matrix(*st["V"])) if c["dtype"] == "mxfp4" else (st["X"], st["V"])
        logp, lse = sc.catalogue_logprob(X, V, st["ids"], ibase=st["ibase"])
        out = {"logp": logp, "lse": lse}
        if c["grad"]:
            dX, dV, db = sc.catalogue_logprob_backward(X, V, st["ids"], lse, st["dlogp"], ibase=st["ibase"])
            out |= {"dX": dX, "dV": dV}
            if db is not None:
                out["dibase"] = db
        return out
    if c["op"] == "preference":
        lc, logp, ref, mask = c["chosen"], st["logp"], st["ref"], st["mask"]
        r = sc.preference_loss(logp[:, :lc], logp[:, lc:], None if ref is None else ref[:, :lc], None if ref is None else ref[:, lc:],
                               mask[:, :lc], mask[:, lc:], beta=0.1, kind=c["kind"], average=c["average"], weight=st["weight"])
        return {"loss": r.loss, "h": r.h, "dchosen": r.d_chosen, "drejected": r.d_rejected}
    r = sc.policy_loss(st["logp"], st["old"], st["adv"], ref_logp=st["ref"], mask=st["mask"], clip_low=LOW, clip_high=HIGH,
                       kl_coef=c["kl"], reduction=c["reduction"])
    out = {"loss": r.loss, "dlogp": r.d_logp, "clipped": r.clipped}
    if c["kl"]:
        out["kl"] = r.kl
    return out


def run(st):
    return _package(st) if own else _plain(st)


def work(case):
    op, n = case["op"], case["n"]
    size = {"f32": 4.0, "bf16": 2.0, "mxfp4": 0.5 + 1 / 32}
    if op == "quantize":
        return {"bytes": n * case["k"] * (size[case["dtype"]] + 4), "flops": 0}
    if op == "scores":
        i, k = case["items"], case["k"]
        return {"bytes": n * k * size[case["dtype"]] + i * k * size["mxfp4"] + 4 * i * case["bias"] + n * i * size[case["out"]], "flops": 2.0 * n * i * k}
    if op == "logprob":
        i, k, s = case["items"], case["k"], size[case["dtype"]]
        once = (n + i) * k * s + 4 * i * case["bias"]
        out = n * case["m"] * 4 + 4 * n
        grad = once + n * case["m"] * 4 if case["grad"] else 0
        return {"bytes": once + out + n * case["m"] * 4 + grad, "flops": (6.0 if case["grad"] else 2.0) * n * i * k}
    if op == "preference":
        return {"bytes": n * (case["chosen"] + case["rejected"]) * (9 + 4 * case["ref"]) + 12 * n, "flops": 0}
    return {"bytes": n * case["len"] * (13 + 4 * bool(case["kl"])) + 16 * n, "flops": 0}


# ------------------------------------------------------------------ exact values, in 64 bits

def _exact_values(X):
    """The nearest of the sixteen values times the block's power of two, by the distance to every one of them; of two equally
    near ones the one with the even index."""
    x = X.double()
    n, k = x.shape
    out = torch.empty_like(x)
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    for c in range(0, k, 32):
        blk = x[:, c:c + 32]
        top = blk.abs().max(1, keepdim=True).values
        unit = torch.exp2((torch.floor(torch.log2(top.clamp(min=2.0 ** -300))) - 2).clamp(-127, 127))
        unit = torch.where(top >= unit * 8, unit * 2, torch.where((top < unit * 4) & (unit > 2.0 ** -127), unit / 2, unit))   # log2 next to a power
        y = blk.abs() / unit
        best, near = torch.zeros_like(y), (y - 0.0).abs()
        for j in (2, 4, 6, 1, 3, 5, 7):                                             # even ones first: they keep a tie
            d = (y - grid[j]).abs()
            best = torch.where(d < near, torch.full_like(y, grid[j]), best)
            near = torch.minimum(d, near)
        out[:, c:c + 32] = torch.where(blk < 0, -best, best) * unit
    return out


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "quantize":
        return {"values": _exact_values(st["X"])}
    if op == "scores":
        a, b = _exact_values(st["X"]), _unpack(st["V"], torch.float64)
        s = torch.empty((a.shape[0], b.shape[0]), dtype=torch.float64, device=DEV)
        torch.mm(a, b.t(), out=s)
        return {"scores": s if st["ibase"] is None else s.add_(st["ibase"])}
    if op == "logprob":
        mx = case["dtype"] == "mxfp4"
        A, B = (_unpack(st["X"], torch.float64), _unpack(st["V"], torch.float64)) if mx else (st["X"].double(), st["V"].double())
        bias = None if st["ibase"] is None else st["ibase"].double()
        logp, lse = torch.zeros(st["ids"].shape, dtype=torch.float64, device=DEV), torch.zeros(case["n"], dtype=torch.float64, device=DEV)
        dA, dB, db = torch.zeros_like(A), torch.zeros_like(B), torch.zeros(B.shape[0], dtype=torch.float64, device=DEV)
        step = max(1, int(2.5e8 // B.shape[0]))
        for r in range(0, case["n"], step):                                         # a few rows of logits at a time
            s = A[r:r + step] @ B.t()
            if bias is not None:
                s += bias
            lse[r:r + step] = torch.logsumexp(s, 1)
            ids = st["ids"][r:r + step].long()
            row, col = torch.nonzero(ids >= 0, as_tuple=True)
            item = ids[row, col]
            logp[r + row, col] = s[row, item] - lse[r + row]
            if case["grad"]:
                w = st["dlogp"][r:r + step].double()
                total = torch.zeros(s.shape[0], dtype=torch.float64, device=DEV).index_add_(0, row, w[row, col])
                s = s.sub_(lse[r:r + step, None]).exp_().mul_(-total[:, None])
                s.index_put_((row, item), w[row, col], accumulate=True)
                dA[r:r + step] = s @ B
                dB += s.t() @ A[r:r + step]
                db += s.sum(0)
        out = {"logp": logp, "lse": lse}
        if case["grad"]:
            out |= {"dX": dA, "dV": dB}
            if bias is not None:
                out["dibase"] = db
        return out
    m = st["mask"]
    if op == "preference":
        lc = case["chosen"]
        x = st["logp"].double() - (0 if st["ref"] is None else st["ref"].double())
        nc, nr = (m[:, :lc].sum(1).clamp(min=1), m[:, lc:].sum(1).clamp(min=1)) if case["average"] else (1, 1)
        h = 0.1 * ((x[:, :lc] * m[:, :lc]).sum(1) / nc - (x[:, lc:] * m[:, lc:]).sum(1) / nr)
        if case["kind"] == "logistic":
            loss, slope = torch.nn.functional.softplus(-h), -torch.sigmoid(-h)
        elif case["kind"] == "hinge":
            loss, slope = (1 - h).clamp(min=0), -(h < 1).double()
        else:
            loss, slope = (h / 0.1 - 5) ** 2, 20 * (h / 0.1 - 5)
        g = 0.1 * slope * st["weight"].double()
        return {"loss": loss, "h": h, "dchosen": (g / nc)[:, None] * m[:, :lc], "drejected": -(g / nr)[:, None] * m[:, lc:]}
    logp, old, A = st["logp"].double(), st["old"].double(), st["adv"].double()[:, None]
    count = m.sum(1)
    c = {"sum": torch.ones_like(count).double(), "row": 1 / count.clamp(min=1).double(), "batch": (1 / count.sum().clamp(min=1).double()).expand(case["n"])}[case["reduction"]]
    r = (logp - old).exp()
    inner = torch.minimum(r * A, r.clamp(1 - LOW, 1 + HIGH) * A)
    free = r * A <= r.clamp(1 - LOW, 1 + HIGH) * A
    loss, grad = -inner, -(r * A) * free
    out = {"clipped": None}
    if case["kl"]:
        q = st["ref"].double() - logp
        kl = q.exp() - q - 1
        loss, grad = loss + case["kl"] * kl, grad + case["kl"] * (1 - q.exp())
        out["kl"] = (kl * m).sum(1) / count.clamp(min=1)
    return out | {"loss": c * (loss * m).sum(1), "dlogp": c[:, None] * grad * m}
