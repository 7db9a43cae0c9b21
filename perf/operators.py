"""Cases, plain forms and exact values of the operators at the two ends of a model with a vocabulary: the scaled table
lookup with its gradient by sorted indices (``pointnet2_utils.embedding_operation``), the softmax cross entropy of a linear
head without its logits (``losses.LinearCrossEntropy``) and the distance to a teacher's top logits
(``losses.TopLogitsDistill``).

``own = False`` computes them with elementary torch operations in float32; ``own = True`` calls the framework."""
import math

import torch

own = False

DEV = "cuda"
IGNORE = -100
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a batch of 32 instances, the 512-wide pooled feature, six object categories: the smallest call, latency counts
        dict(name="ce_category_f32", op="ce", n=32, d=512, v=6, dtype="f32", bias=True, ignored=0.0, reduction="mean",
             train=True),
        # 32 clouds of 1024 points, the 128-wide point feature, a coordinate axis cut into 64 bins, a third of the points
        # unlabelled: many rows, few classes
        dict(name="ce_point_bins_f32", op="ce", n=32768, d=128, v=64, dtype="f32", bias=True, ignored=0.3,
             reduction="mean", train=True),
        # the joint cells of a 32 x 32 x 32 grid as classes, rows weighted by the caller: single precision, no reduction
        dict(name="ce_grid_cells_f32", op="ce", n=1024, d=512, v=32768, dtype="f32", bias=False, ignored=0.0,
             reduction="none", train=True),
        # nothing is a multiple of anything, padded sequences
        dict(name="ce_ragged_f16", op="ce", n=2047, d=387, v=40001, dtype="f16", bias=True, ignored=0.25,
             reduction="sum", train=True),
        # the largest: a training step over a large vocabulary
        dict(name="ce_large_bf16", op="ce", n=8192, d=1024, v=65536, dtype="bf16", bias=False, ignored=0.1,
             reduction="mean", train=True),
        # scoring one token: the table is read once
        dict(name="ce_score_one_bf16", op="ce", n=1, d=1024, v=65536, dtype="bf16", bias=False, ignored=0.0,
             reduction="none", train=False),
        # a small batch against a thousand classes
        dict(name="distill_small_f32", op="distill", n=64, v=1000, k=8, pad=0, dtype="f32", temperature=1.0,
             reduction="mean", empty=0.0, index="int64"),
        # rows cut out of a padded buffer, slots and whole rows without a teacher, rows weighted by the caller
        dict(name="distill_ragged_f16", op="distill", n=1501, v=40001, k=33, pad=63, dtype="f16", temperature=2.0,
             reduction="none", empty=0.2, index="int32"),
        # a training step over a large vocabulary
        dict(name="distill_large_bf16", op="distill", n=8192, v=65536, k=64, pad=0, dtype="bf16", temperature=1.5,
             reduction="mean", empty=0.05, index="int32"),
        # the category of each of 32 x 1024 points: six rows, very long sums
        dict(name="embed_category_f32", op="embed", n=32768, v=6, d=64, dtype="f32", scale=1.0, padding=-1, index="int32"),
        # a short odd batch with a padding row
        dict(name="embed_short_f16", op="embed", n=77, v=1000, d=99, dtype="f16", scale=math.sqrt(99.0), padding=0,
             index="int64"),
        # a training step's tokens over a large table, a few of them very frequent
        dict(name="embed_large_bf16", op="embed", n=32768, v=65536, d=1024, dtype="bf16", scale=32.0, padding=-1,
             index="int64"),
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]; every other one is odd on purpose."""
    x = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        x |= 1
    return max(lo, min(hi, x))


def draw(rng):
    op = rng.choice(["ce", "distill", "embed"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "ce":
        n, d, v = _log_int(rng, 1, 8192), _log_int(rng, 32, 1024), _log_int(rng, 2, 65536)
        return dict(op=op, n=n, d=d, v=v, dtype=dtype, bias=rng.random() < 0.5, ignored=rng.choice([0.0, 0.1, 0.4]),
                    reduction=rng.choice(["mean", "sum", "none"]), train=rng.random() < 0.8)
    if op == "distill":
        v = _log_int(rng, 2, 65536)
        return dict(op=op, n=_log_int(rng, 1, 8192), v=v, k=_log_int(rng, 1, min(64, v)), pad=rng.choice([0, 0, 1, 63]),
                    dtype=dtype, temperature=rng.choice([0.5, 1.0, 2.0, 4.0]),
                    reduction=rng.choice(["mean", "sum", "none"]), empty=rng.choice([0.0, 0.3]),
                    index=rng.choice(["int32", "int64"]))
    d = _log_int(rng, 16, 1024)
    return dict(op=op, n=_log_int(rng, 1, 32768), v=_log_int(rng, 2, 65536), d=d, dtype=dtype,
                scale=rng.choice([1.0, math.sqrt(d)]), padding=rng.choice([-1, 0]), index=rng.choice(["int32", "int64"]))


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _skewed(g, n, v):
    """n indices in [0, v), the small ones frequent (the density falls like 1 / index)."""
    u = torch.rand(n, device=DEV, generator=g, dtype=torch.float64)
    return (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)


def prepare(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, device=DEV, generator=g)
    rand = lambda *s: torch.rand(*s, device=DEV, generator=g)
    s = {"case": case}
    if case["op"] == "ce":
        n, d, v = case["n"], case["d"], case["v"]
        w = randn(v, d).div_(math.sqrt(d))
        t = _skewed(g, n, v)
        # features that lean towards the row of their class, some hardly, some almost sure of it
        x = randn(n, d) + w[t] * rand(n, 1) * (4.0 + 2.0 * math.log(v))
        if case["ignored"]:
            t = torch.where(rand(n) < case["ignored"], torch.full_like(t, IGNORE), t)
        s["x"], s["w"] = x.to(dt).requires_grad_(case["train"]), w.to(dt).requires_grad_(case["train"])
        s["b"] = (0.5 * randn(v)).to(dt).requires_grad_(case["train"]) if case["bias"] else None
        s["t"] = t
        # the gradient of what a program does with the loss(es): one for a scalar, weights for rows
        s["g"] = 0.5 + rand(n) if case["reduction"] == "none" else torch.ones((), device=DEV)
        return s
    if case["op"] == "distill":
        n, v, k = case["n"], case["v"], case["k"]
        z = torch.empty(n, v + case["pad"], device=DEV, dtype=dt)
        for a in range(0, n, 1024):
            z[a:a + 1024] = (1.5 * randn(min(1024, n - a), v + case["pad"])).to(dt)
        # k different classes a row, the student's own opinion of them raised and falling from the first to the last
        start = (rand(n, 1) * v).long()
        idx = (start + torch.arange(k, device=DEV) * max(1, v // k)) % v
        fall = 9.0 * torch.exp(-0.15 * torch.arange(k, device=DEV, dtype=torch.float32))
        z.scatter_(1, idx, (fall + randn(n, k)).to(dt))
        s["z"] = z[:, :v].requires_grad_(True)
        s["top"] = (fall + 0.7 * randn(n, k)).to(dt)
        if case["empty"]:
            # a teacher that kept fewer entries for some rows, and none for others
            kept = torch.where(rand(n, 1) < case["empty"], torch.zeros(n, 1, device=DEV),
                               torch.where(rand(n, 1) < 0.5, torch.ceil(rand(n, 1) * k), torch.full((n, 1), float(k), device=DEV)))
            idx = torch.where(torch.arange(k, device=DEV) < kept, idx, torch.full_like(idx, -1))
        s["idx"] = idx.to(torch.int32 if case["index"] == "int32" else torch.int64)
        s["g"] = 0.5 + rand(n) if case["reduction"] == "none" else torch.ones((), device=DEV)
        return s
    n, v, d = case["n"], case["v"], case["d"]
    ids = _skewed(g, n, v)
    s["ids"] = ids.to(torch.int32 if case["index"] == "int32" else torch.int64)
    s["w"] = (randn(v, d) / math.sqrt(d)).to(dt).requires_grad_(True)
    s["g"] = randn(n, d).to(dt)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _reduce(rows, keep, reduction):
    """Loss and the factor of every row's gradient."""
    if reduction == "none":
        return rows.float(), keep.float()
    if reduction == "sum":
        return rows.double().sum().float(), keep.float()
    n = keep.sum()
    return (rows.double().sum() / n).float(), keep.float() / n


def _ce_plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    x, w, t = s["x"].detach().float(), s["w"].detach().float(), s["t"]
    keep = t != IGNORE
    pick = torch.where(keep, t, torch.zeros_like(t)).unsqueeze(1)
    z = x @ w.t()
    if s["b"] is not None:
        z += s["b"].detach().float()
    m = z.amax(1, keepdim=True)
    zt = z.gather(1, pick) - m
    e = torch.exp(z - m)
    tot = e.sum(1, keepdim=True)
    rows = torch.where(keep, (torch.log(tot) - zt).squeeze(1), torch.zeros_like(m).squeeze(1))
    loss, factor = _reduce(rows, keep, case["reduction"])
    if not case["train"]:
        return {"loss": loss}
    e /= tot
    e.scatter_add_(1, pick, -torch.ones_like(zt))
    e *= (factor * s["g"]).unsqueeze(1)
    out = {"loss": loss, "dx": (e @ w).to(dt), "dw": (e.t() @ x).to(dt)}
    if s["b"] is not None:
        out["db"] = e.sum(0, dtype=torch.float64).to(dt)
    return out


def _distill_plain(s):
    case = s["case"]
    dt, temp = DTYPES[case["dtype"]], case["temperature"]
    idx = s["idx"].long()
    used = idx >= 0
    keep = used.any(1)
    pick = torch.where(used, idx, torch.zeros_like(idx))
    t = torch.where(used, s["top"].float() / temp, torch.full((), -math.inf, device=DEV))
    t = t - torch.where(keep, t.amax(1), torch.zeros((), device=DEV)).unsqueeze(1)
    et = torch.exp(t)
    et_sum = torch.where(keep, et.sum(1), torch.ones((), device=DEV)).unsqueeze(1)
    q = et / et_sum
    log_q = torch.where(used, t - torch.log(et_sum), torch.zeros((), device=DEV))
    z = s["z"].detach().float() / temp
    m = z.amax(1, keepdim=True)
    z -= m
    zk = z.gather(1, pick)
    z.exp_()
    tot = z.sum(1, keepdim=True)
    log_p = zk - torch.log(tot)
    rows = temp * temp * (q * (log_q - log_p)).sum(1)
    loss, factor = _reduce(rows, keep, case["reduction"])
    z /= tot
    z.scatter_add_(1, pick, -q)
    z *= (temp * factor * s["g"]).unsqueeze(1)
    return {"loss": loss, "dz": z.to(dt)}


def _embed_plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    ids = s["ids"].long()
    out = (s["w"].detach()[ids].float() * case["scale"]).to(dt)
    grad = s["g"].float()
    if case["padding"] >= 0:
        grad = grad * (ids != case["padding"]).unsqueeze(1)
    dw = torch.zeros(case["v"], case["d"], device=DEV)
    dw.index_add_(0, ids, grad)
    return {"out": out, "dw": (dw * case["scale"]).to(dt)}


# ---- the framework's calls ---------------------------------------------------------------------------------------------

def _ce_own(s):
    from istnet_amd import losses
    case = s["case"]
    loss = losses.LinearCrossEntropy(s["x"], s["w"], s["t"], bias=s["b"], ignore_index=IGNORE, reduction=case["reduction"])
    if not case["train"]:
        return {"loss": loss}
    if s["b"] is None:
        dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]), s["g"])
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    dx, dw, db = torch.autograd.grad(loss, (s["x"], s["w"], s["b"]), s["g"])
    return {"loss": loss.detach(), "dx": dx, "dw": dw, "db": db}


def _distill_own(s):
    from istnet_amd import losses
    case = s["case"]
    loss = losses.TopLogitsDistill(s["z"], s["top"], s["idx"], temperature=case["temperature"], reduction=case["reduction"])
    (dz,) = torch.autograd.grad(loss, (s["z"],), s["g"])
    return {"loss": loss.detach(), "dz": dz}


def _embed_own(s):
    from istnet_amd.pointnet2 import pointnet2_utils
    case = s["case"]
    out = pointnet2_utils.embedding_operation(s["w"], s["ids"], case["scale"],
                                              case["padding"] if case["padding"] >= 0 else None)
    (dw,) = torch.autograd.grad(out, (s["w"],), s["g"])
    return {"out": out.detach(), "dw": dw}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"ce": _ce_own, "distill": _distill_own, "embed": _embed_own}[op](state)
    with torch.no_grad():
        return {"ce": _ce_plain, "distill": _distill_plain, "embed": _embed_plain}[op](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "ce":
        n, d, v = case["n"], case["d"], case["v"]
        rows = max(1.0, n * (1.0 - case["ignored"]))
        inputs = e * (rows * d + v * d + (v if case["bias"] else 0)) + 8 * n
        loss = 4 * n if case["reduction"] == "none" else 4
        if not case["train"]:
            return {"bytes": inputs + loss, "flops": 2.0 * rows * v * d}
        grads = e * (n * d + v * d + (v if case["bias"] else 0))
        return {"bytes": inputs + loss + grads, "flops": 6.0 * rows * v * d}
    if case["op"] == "distill":
        n, v, k = case["n"], case["v"], case["k"]
        rows = max(1.0, n * (1.0 - case["empty"]))
        ie = 4 if case["index"] == "int32" else 8
        return {"bytes": e * (rows * v + n * v) + n * k * (e + ie) + (8 * n if case["reduction"] == "none" else 4),
                "flops": 8.0 * rows * v}
    n, v, d = case["n"], case["v"], case["d"]
    ie = 4 if case["index"] == "int32" else 8
    touched = min(n, v)
    return {"bytes": e * (touched * d + n * d + n * d + v * d) + ie * n, "flops": 2.0 * n * d}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def _rows_to_loss(per_row, counted, reduction):
    if reduction == "none":
        return per_row
    return per_row.sum() if reduction == "sum" else per_row.sum() / counted


def _exact_ce(case, s):
    """-log softmax of the class, row by row, and its derivative; rows in blocks of 512."""
    X, W = s["x"].detach().to(torch.float64), s["w"].detach().to(torch.float64)
    B = s["b"].detach().to(torch.float64) if s["b"] is not None else torch.zeros(case["v"], device=DEV, dtype=torch.float64)
    labelled = (s["t"] != IGNORE).nonzero().squeeze(1)
    per_row = torch.zeros(case["n"], device=DEV, dtype=torch.float64)
    dX, dW, dB = torch.zeros_like(X), torch.zeros_like(W), torch.zeros_like(B)
    weight = s["g"].to(torch.float64).expand(case["n"])
    if case["reduction"] == "mean":
        weight = weight / labelled.numel()
    for a in range(0, labelled.numel(), 512):
        r = labelled[a:a + 512]
        logits = torch.addmm(B, X[r], W.t())
        log_soft = logits - torch.logsumexp(logits, 1, keepdim=True)
        del logits
        here = torch.arange(r.numel(), device=DEV)
        per_row[r] = -log_soft[here, s["t"][r]]
        if case["train"]:
            dlogits = log_soft.exp_()
            dlogits[here, s["t"][r]] -= 1.0
            dlogits *= weight[r].unsqueeze(1)
            dX[r] = dlogits @ W
            dW.addmm_(dlogits.t(), X[r])
            dB += dlogits.sum(0)
    out = {"loss": _rows_to_loss(per_row, labelled.numel(), case["reduction"])}
    if case["train"]:
        out["dx"], out["dw"] = dX, dW
        if s["b"] is not None:
            out["db"] = dB
    return out


def _exact_distill(case, s):
    """T^2 KL(teacher over its kept entries || student over all classes), row by row; rows in blocks of 512."""
    n, temp = case["n"], case["temperature"]
    per_row = torch.zeros(n, device=DEV, dtype=torch.float64)
    dZ = torch.zeros(n, case["v"], device=DEV, dtype=torch.float64)
    used = s["idx"] >= 0
    rows = used.any(1).nonzero().squeeze(1)
    weight = s["g"].to(torch.float64).expand(n)
    if case["reduction"] == "mean":
        weight = weight / rows.numel()
    for a in range(0, rows.numel(), 512):
        r = rows[a:a + 512]
        u, k = used[r], s["idx"][r].long().clamp(min=0)
        teacher = (s["top"][r].to(torch.float64) / temp).masked_fill(~u, -math.inf)
        log_t = teacher - torch.logsumexp(teacher, 1, keepdim=True)
        prob_t = log_t.exp()
        student = s["z"].detach()[r].to(torch.float64) / temp
        log_s = student - torch.logsumexp(student, 1, keepdim=True)
        gap = (log_t - log_s.gather(1, k)).masked_fill(~u, 0.0)
        per_row[r] = temp * temp * (prob_t * gap).sum(1)
        d = log_s.exp_()
        d.scatter_add_(1, k, -prob_t)
        dZ[r] = d * (temp * weight[r]).unsqueeze(1)
    return {"loss": _rows_to_loss(per_row, rows.numel(), case["reduction"]), "dz": dZ}


def _exact_embed(case, s):
    """The lookup, and the table's gradient as sums over the sorted indices."""
    ids = s["ids"].long()
    out = s["w"].detach().to(torch.float64).index_select(0, ids) * case["scale"]
    order = torch.argsort(ids, stable=True)
    present, count = torch.unique_consecutive(ids[order], return_counts=True)
    dW = torch.zeros(case["v"], case["d"], device=DEV, dtype=torch.float64)
    end = torch.cumsum(count, 0)
    for c in range(0, case["d"], 128):            # running sums over the sorted tokens, a block of columns at a time
        run_sum = torch.cumsum(s["g"][order, c:c + 128].to(torch.float64), 0)
        upto = run_sum[end - 1]
        dW[present, c:c + 128] = torch.diff(upto, dim=0, prepend=torch.zeros_like(upto[:1]))
    if case["padding"] >= 0:
        dW[case["padding"]] = 0.0
    return {"out": out, "dw": dW * case["scale"]}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"ce": _exact_ce, "distill": _exact_distill, "embed": _exact_embed}[case["op"]](case, s)
