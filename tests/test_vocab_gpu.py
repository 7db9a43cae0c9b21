"""Vocabulary operators on the GPU against their definitions in float64.

Tolerances.  u(t) = finfo(t).eps / 2 is the largest relative error of one rounding to t, U = 2^-24 that of float32.  A float32 sum of
n terms is off by at most n U times the sum of their magnitudes, whatever its order.  Results below the smallest normal number of
their type are off by half their spacing.  Every bound below is put together from these."""
import math

import pytest
import torch

from istnet_amd import losses
from istnet_amd.pointnet2 import pointnet2_utils

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24
NAN, INF = float("nan"), float("inf")


def _round(t):
    return torch.finfo(t).eps / 2


def _tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _within(got, want, bound, what):
    """got is as finite as want, and off by no more than bound where it is finite."""
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, what
    assert torch.equal(got.isnan(), want.isnan()), what
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), what
    ok = want.isfinite()
    off = ((got - want).abs() - bound.expand_as(want) if torch.is_tensor(bound) else (got - want).abs() - bound)[ok]
    assert off.numel() == 0 or float(off.max()) <= 0.0, f"{what}: off by {float((got - want).abs()[ok].max())}, over by {float(off.max())}"


# ---- lookup ------------------------------------------------------------------------------------------------------------

def _lookup_reference(w, ids, scale, padding, grad):
    v = w.shape[0]
    scale = float(torch.tensor(scale, dtype=F32))
    flat = ids.reshape(-1).long()
    ok = (flat >= 0) & (flat < v)
    out = torch.where(ok.unsqueeze(1), w.detach().double()[flat.clamp(0, v - 1)] * scale, NAN).reshape(*ids.shape, -1)
    part = ok if padding is None else ok & (flat != padding)
    g = grad.reshape(flat.numel(), -1).double()[part]
    dw = torch.zeros_like(w, dtype=torch.float64).index_add_(0, flat[part], g) * scale
    mass = torch.zeros_like(w, dtype=torch.float64).index_add_(0, flat[part], g.abs()) * abs(scale)
    count = torch.bincount(flat[part], minlength=v).double().unsqueeze(1)
    return out, dw, mass * (count + 2) * U


def _check_lookup(w, ids, scale, padding, grad=None, call=None):
    w = w.detach().requires_grad_()
    out = (call or pointnet2_utils.embedding_operation)(w, ids, scale, padding)
    t = w.dtype
    if grad is None:
        grad = torch.randn(out.shape, device=DEV, generator=_gen(7)).to(t)
    (dw,) = torch.autograd.grad(out, w, grad)
    want, dwant, slack = _lookup_reference(w, ids, scale, padding, grad)
    assert out.dtype == t and dw.dtype == t
    _within(out, want, want.abs().nan_to_num() * (_round(t) + 2 * U) + _tiny(t), "out")
    _within(dw, dwant, dwant.abs() * (_round(t) + 2 * U) + slack + _tiny(t), "dw")
    return out, dw


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 5, 3), (63, 6, 64), (64, 7, 8), (129, 6, 100), (1000, 1000, 257), (8192, 33, 16),
                                   (8193, 33, 16), (20000, 70000, 40), (5, 300000, 7), (40000, 2, 130), (300000, 515, 9),
                                   (17, 9, 2500)])
def test_lookup(n, v, d, dtype):
    g = _gen(n + v + d)
    w = torch.randn(v, d, device=DEV, generator=g).to(dtype)
    ids = (torch.rand(n, device=DEV, generator=g) ** 3 * v).long().clamp(max=v - 1)
    _check_lookup(w, ids, 1.0, None)
    _check_lookup(w, ids.int(), math.sqrt(d), 0)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_lookup_shapes_strides_and_bad_indices(index):
    g = _gen(3)
    table = torch.randn(50, 40, device=DEV, generator=g)
    ids = torch.randint(0, 50, (3, 4, 5), device=DEV, generator=g).to(index)
    _check_lookup(table[:, :33], ids, 2.0, 7)                              # a slice with a row stride
    _check_lookup(table.t(), ids % 40, 2.0, 7)                             # columns as rows: copied
    _check_lookup(table[:, 3:4], ids, 2.0, None)                           # one column
    _check_lookup(table[5:6], ids * 0, 2.0, None)                          # one row
    _check_lookup(table[:, 1:34], ids.permute(2, 0, 1), 2.0, None)         # an odd first element, permuted indices
    flat = ids.reshape(-1).clone()
    flat[::7], flat[3], flat[11] = -1, 50, -2 ** 31
    if index == torch.int64:
        flat[13], flat[17] = 2 ** 40 + 1, -2 ** 40
    out, _ = _check_lookup(table, flat, 1.5, 3)
    assert out[0].isnan().all() and out[1].isfinite().all()
    _check_lookup(table, torch.full_like(flat, 60), 1.5, 3)                # no index points anywhere
    grad = torch.randn(1, 40, device=DEV, generator=g).expand(60, 40)      # an expanded gradient
    _check_lookup(table, flat, 1.5, 3, grad)
    wide = torch.randn(60, 80, device=DEV, generator=g)[:, ::2]            # a gradient with a stride
    _check_lookup(table, flat, 1.5, 3, wide)


def test_lookup_without_indices_and_infinite_values():
    w = torch.randn(5, 4, device=DEV).requires_grad_()
    out = pointnet2_utils.embedding_operation(w, torch.zeros(2, 0, dtype=torch.int64, device=DEV))
    assert out.shape == (2, 0, 4)
    out.sum().backward()
    assert (w.grad == 0).all()
    w2 = torch.tensor([[INF, -INF, NAN], [1.0, 2.0, 3.0]], device=DEV)
    ids = torch.tensor([0, 1, 1], device=DEV)
    grad = torch.tensor([[1.0, 1.0, 1.0], [INF, NAN, 1.0], [1.0, 1.0, -INF]], device=DEV)
    _check_lookup(w2, ids, 2.0, None, grad)


@pytest.mark.parametrize("n", [500, 9000, 70000])
def test_lookup_gradient_is_the_same_bits_every_time(n):
    g = _gen(n)
    ids = torch.randint(0, 5, (n,), device=DEV, generator=g)
    w = torch.randn(5, 65, device=DEV, generator=g).requires_grad_()
    grad = torch.randn(n, 65, device=DEV, generator=g)
    first = torch.autograd.grad(pointnet2_utils.embedding_operation(w, ids), w, grad)[0]
    for _ in range(3):
        assert torch.equal(first, torch.autograd.grad(pointnet2_utils.embedding_operation(w, ids), w, grad)[0])


def test_lookup_refusals():
    w, ids = torch.randn(5, 4, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    call = pointnet2_utils.embedding_operation
    with pytest.raises(TypeError, match="weight"):
        call(w.double(), ids)
    with pytest.raises(TypeError, match="idx"):
        call(w, ids.float())
    with pytest.raises(RuntimeError, match="idx must be a CUDA"):
        call(w, ids.cpu())
    with pytest.raises(ValueError, match="non-empty"):
        call(w[:0], ids)
    with pytest.raises(ValueError, match="non-empty"):
        call(w[0], ids)
    with pytest.raises(ValueError, match="padding_idx"):
        call(w, ids, 1.0, 5)
    w.requires_grad_()
    (dw,) = torch.autograd.grad(call(w, ids).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        dw.sum().backward()


def test_scaled_embedding_module():
    torch.manual_seed(0)
    m = pointnet2_utils.ScaledEmbedding(400, 64, padding_idx=2).to(DEV)
    assert (m.weight[2] == 0).all() and abs(float(m(torch.arange(400, device=DEV)).std()) - 1.0) < 0.05
    ids = torch.randint(0, 400, (4, 100), device=DEV)
    m(ids).square().sum().backward()
    assert (m.weight.grad[2] == 0).all() and m.weight.grad.isfinite().all()


# ---- distance to a teacher's top logits --------------------------------------------------------------------------------

def _distill_inputs(n, v, k, dtype, seed, pad=0, index=torch.int64):
    g = _gen(seed)
    z = (2.0 * torch.randn(n, v + pad, device=DEV, generator=g)).to(dtype)[:, :v]
    idx = torch.stack([torch.randperm(v, device=DEV, generator=g)[:k] for _ in range(min(n, 64))]).repeat((n + 63) // 64, 1)[:n]
    top = (3.0 * torch.randn(n, k, device=DEV, generator=g)).to(dtype)
    return z, top, idx.to(index)


def _distill_reference(z, top, idx, temp, reduction, gout):
    """float64 loss and gradient, and the bounds of a float32 evaluation of each."""
    v, t = z.shape[1], z.dtype
    x = z.detach().double().cpu().requires_grad_()
    # the CPU composition in float64 (checked against the definition, slot by slot, without a GPU)
    loss = losses.TopLogitsDistill(x, top.double().cpu(), idx.cpu(), temp, reduction)
    (dx,) = torch.autograd.grad(loss, x, gout.double().cpu())
    loss, dx = loss.detach().to(DEV), dx.to(DEV)
    rows = losses.TopLogitsDistill(x.detach(), top.double().cpu(), idx.cpu(), temp, "none").to(DEV)
    used = idx != -1
    counted = used.any(1)
    zf = z.detach().double().masked_fill(~counted.unsqueeze(1), 0.0)
    fin = zf.masked_fill(~zf.isfinite(), 0.0)
    reach = (fin.amax(1) - fin.amin(1)) / temp                    # largest |z - m| / T
    tf = top.double().masked_fill(~used | ~top.isfinite(), 0.0)
    treach = (tf.amax(1) - tf.amin(1)) / temp
    # an exponential of (z - m) / T: the difference, the product with log2(e) / T (itself rounded) and exp2 itself, 1.5 ulp;
    # the sum of v of them; the same for the teacher's k
    rel_p = U * (4 * reach + 4 + v + 2)
    rel_q = U * (4 * treach + 4 + top.shape[1] + 2)
    # loss row = T^2 sum q (log q - log p): every log is off by the relative error of its sum plus its own rounding, and q by rel_q
    size = reach + treach + math.log(max(v, 2)) + math.log(top.shape[1] + 1) + 2
    row_bound = temp ** 2 * (rel_p + rel_q + size * (rel_q + 8 * U)) * counted
    count = counted.sum().double()
    if reduction == "none":
        loss_bound = row_bound
        factor = gout.double()
    else:
        share = 1.0 / count if reduction == "mean" else 1.0
        loss_bound = (row_bound.sum() + rows.nan_to_num(0, 0, 0).abs().sum() * 2 * U) * share
        factor = gout.double() * share * torch.ones_like(count).expand(z.shape[0])
    q = torch.where(used, top.double() / temp, -INF)
    q = torch.softmax(torch.where(counted.unsqueeze(1), q, 0.0), 1).masked_fill(~used, 0.0).nan_to_num()
    p = torch.softmax(zf / temp, 1).nan_to_num()
    merged = torch.zeros_like(p).scatter_add_(1, idx.long().clamp(0, v - 1), q)
    grad_bound = temp * factor.abs().unsqueeze(1) * ((rel_p + 4 * U).unsqueeze(1) * p + (rel_q + 4 * U).unsqueeze(1) * merged) \
        + dx.nan_to_num().abs() * _round(t) + _tiny(t)
    # float32 results below its smallest normal number may be flushed
    return loss, dx, loss_bound + 2.0 ** -126, (grad_bound + temp * factor.abs().unsqueeze(1) * 2.0 ** -120).nan_to_num(INF)


def _check_distill(z, top, idx, temp, reduction):
    z = z.detach().requires_grad_()
    loss = losses.TopLogitsDistill(z, top, idx, temp, reduction)
    gout = 0.5 + torch.rand(loss.shape, device=DEV, generator=_gen(11))
    (dz,) = torch.autograd.grad(loss, z, gout)
    assert loss.dtype == F32 and dz.dtype == z.dtype
    want, dwant, lb, gb = _distill_reference(z, top, idx, temp, reduction, gout)
    _within(loss, want, lb, "loss")
    _within(dz, dwant, gb, "dz")
    return loss, dz


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (1, 2, 2), (3, 64, 1), (7, 1000, 8), (64, 1025, 64), (1, 5000, 16), (2, 40001, 33),
                                   (2100, 37, 5), (2049, 4099, 64), (5, 300, 256)])
def test_distill(n, v, k, dtype):
    for i, (temp, reduction) in enumerate([(1.0, "mean"), (2.0, "none"), (0.5, "sum")]):
        z, top, idx = _distill_inputs(n, v, k, dtype, n + v + k + i, pad=(0, 1, 63)[i], index=(torch.int32, torch.int64)[i % 2])
        _check_distill(z, top, idx, temp, reduction)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("n,v", [(9, 50), (9, 9000)])
def test_distill_masks_and_repeats(n, v, reduction):
    """Rows without a teacher (their NaN logits are not looked at), slots without one, repeated classes, weights of zero, classes the
    student excludes."""
    z, top, idx = _distill_inputs(n, v, 6, F32, v)
    idx[0], z[0] = -1, NAN
    idx[1, 2:], top[1, 2:] = -1, NAN
    idx[2, 1] = idx[2, 3] = idx[2, 5]
    idx[3, :] = idx[3, 0]
    top[4, 1:] = -INF
    free = [i for i in range(v) if i not in idx[5].tolist()]
    z[5, free[0]] = -INF
    z[6] += 3000.0
    z[7] = -60000.0
    _check_distill(z, top, idx, 1.5, reduction)


@pytest.mark.parametrize("v", [50, 9000])
def test_distill_rows_that_cannot_be_right_are_nan(v):
    z, top, idx = _distill_inputs(6, v, 4, F32, v)
    idx[0, 2], idx[1, 0], top[2, 1], z[3, 7], z[4, 8] = v, -2, NAN, NAN, INF
    loss, dz = _check_distill(z, top, idx, 1.0, "none")
    assert loss[:5].isnan().all() and loss[5].isfinite()
    assert dz[:5].isnan().all() and dz[5].isfinite().all()


def test_distill_mean_over_no_row():
    z, top, idx = _distill_inputs(5, 40, 3, F32, 1)
    z = z.detach().requires_grad_()
    loss = losses.TopLogitsDistill(z, top, torch.full_like(idx, -1))
    loss.backward()
    assert loss.isnan() and (z.grad == 0).all()
    z0 = torch.zeros(0, 5, device=DEV, requires_grad=True)
    assert losses.TopLogitsDistill(z0, torch.zeros(0, 2, device=DEV), torch.zeros(0, 2, dtype=torch.int32, device=DEV)).isnan()


def test_distill_leading_shape_teacher_type_and_strides():
    z, top, idx = _distill_inputs(12, 100, 4, BF16, 5)
    want, dwant = _check_distill(z, top.float(), idx, 1.0, "none")
    z3 = z.detach().reshape(3, 4, 100).requires_grad_()
    loss = losses.TopLogitsDistill(z3, top.float().reshape(3, 4, 4), idx.reshape(3, 4, 4), 1.0, "none")
    assert loss.shape == (3, 4) and torch.equal(loss.reshape(-1), want)
    cols = z.detach().float().t().contiguous().t()                 # column-major logits
    _check_distill(cols, top, idx, 1.0, "mean")
    _check_distill(z.float()[::2, ::3], top[::2, :], idx[::2] % 34, 1.0, "mean")


def test_distill_gradient_against_differences():
    """Central differences of the float32 loss: off by h^2 / 6 times the third derivative (at most T^-1) plus 2 U |loss| / h."""
    z, top, idx = _distill_inputs(1, 9, 3, F32, 2)
    z = z.detach().requires_grad_()
    loss = losses.TopLogitsDistill(z, top, idx, 1.0, "sum")
    (dz,) = torch.autograd.grad(loss, z)
    h = 2.0 ** -6
    for c in range(9):
        step = torch.zeros_like(z)
        step[0, c] = h
        with torch.no_grad():
            hi, lo = (float(losses.TopLogitsDistill(z + s, top, idx, 1.0, "sum")) for s in (step, -step))
        assert abs((hi - lo) / (2 * h) - float(dz[0, c])) < h * h / 6 + 64 * U * (1 + abs(hi)) / h


def test_distill_refusals():
    z, top, idx = _distill_inputs(4, 10, 3, F32, 1)
    with pytest.raises(TypeError, match="logits"):
        losses.TopLogitsDistill(z.double(), top, idx)
    with pytest.raises(TypeError, match="top_logits"):
        losses.TopLogitsDistill(z, top.double(), idx)
    with pytest.raises(RuntimeError, match="same device"):
        losses.TopLogitsDistill(z, top.cpu(), idx)
    z.requires_grad_()
    (dz,) = torch.autograd.grad(losses.TopLogitsDistill(z, top, idx), z, create_graph=True)
    with pytest.raises(RuntimeError):
        dz.sum().backward()
