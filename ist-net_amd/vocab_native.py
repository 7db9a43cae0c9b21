"""Native operators at the two ends of a model with discrete classes (csrc/vocab/, include/istnet_vocab.h): the scaled table
lookup with its gradient by sorted indices (``pointnet2_utils.embedding_operation``), the distance to a teacher's top logits
(``losses.TopLogitsDistill``), and the cross entropy of a linear head without its logits (``losses.LinearCrossEntropy``).

CUDA tensors of float32, bfloat16 or float16 run the kernels or raise; there is no fallback on the GPU.  CPU tensors (host-logic
tests) take the literal torch composition in the callers.  Nothing synchronises and nothing is kept between calls: every call
takes its scratch memory from torch's allocator on the current stream, so calls on several streams and captured graphs do not
share any.
"""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _native

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def require(cond, msg, kind=RuntimeError):
    if not cond:
        raise kind(msg)


def require_float(t, name):
    require(t.dtype in DTYPES, f"{name} must be a float32, bfloat16 or float16 tensor, got {t.dtype}", TypeError)


def require_index(t, name):
    require(t.dtype in (torch.int32, torch.int64), f"{name} must be an int32 or int64 tensor, got {t.dtype}", TypeError)


def require_device(lead, name, **others):
    for other, t in others.items():
        require(t.device == lead.device, f"{other} must be on the same device as {name}")


def _launch(dev, what, fn, *args):
    """fn(*args, current stream of dev) with dev as the current device, which it nearly always is already."""
    if torch.cuda.current_device() == dev.index:
        _native.check(fn(*args, torch._C._cuda_getCurrentRawStream(dev.index)), what)
    else:
        with torch.cuda.device(dev):
            _native.check(fn(*args, torch._C._cuda_getCurrentRawStream(dev.index)), what)


def _rows(t):
    """(tensor, leading dimension) of a 2-D operand with contiguous rows that do not overlap; anything else is copied."""
    if t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return t, t.stride(0)
    if t.shape[1] == 1 and t.stride(0) >= 1:
        return t, t.stride(0)
    if t.shape[0] == 1 and t.stride(1) == 1:
        return t, t.shape[1]
    t = t.contiguous()
    return t, t.shape[1]


def _scratch(kib, dev):
    return torch.empty(max(kib, 1) * 1024, dtype=torch.uint8, device=dev)


class EmbeddingFunction(Function):
    """weight (V, D), idx (...) -> scale * weight[idx] (..., D); gradient for weight."""

    @staticmethod
    def forward(ctx, weight, idx, scale, padding):
        dev, (v, d), n = weight.device, weight.shape, idx.numel()
        out = torch.empty((*idx.shape, d), dtype=weight.dtype, device=dev)
        ids = idx.contiguous()
        if n:
            w, ldw = _rows(weight)
            _launch(dev, "embed_forward", _native.lib().istnet_embed_forward, n, v, d, DTYPES[weight.dtype],
                    ids.dtype == torch.int64, w.data_ptr(), ldw, ids.data_ptr(), scale, out.data_ptr())
        ctx.save_for_backward(ids)
        ctx.args = (v, d, scale, padding, weight.dtype)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        (ids,) = ctx.saved_tensors
        v, d, scale, padding, dtype = ctx.args
        dev, n = ids.device, ids.numel()
        if n == 0:
            return torch.zeros((v, d), dtype=dtype, device=dev), None, None, None
        g, ldg = _rows(grad_out.reshape(n, d))
        dw = torch.empty((v, d), dtype=dtype, device=dev)
        lib = _native.lib()
        ws = _scratch(lib.istnet_embed_scratch_kib(n, v, d), dev)
        _launch(dev, "embed_backward", lib.istnet_embed_backward, n, v, d, DTYPES[dtype], ids.dtype == torch.int64, g.data_ptr(),
                ldg, ids.data_ptr(), -1 if padding is None else padding, scale, ws.data_ptr(), dw.data_ptr())
        return dw, None, None, None


class DistillFunction(Function):
    """logits (N, V), top (N, K), idx (N, K) -> loss (N,) or scalar, float32; gradient for logits."""

    @staticmethod
    def forward(ctx, logits, top, idx, temperature, reduction):
        dev, (n, v), k = logits.device, logits.shape, idx.shape[1]
        lib = _native.lib()
        z, ldz = _rows(logits)
        top, ids = top.contiguous(), idx.contiguous()
        loss = torch.empty((n,) if reduction == 0 else (), dtype=torch.float32, device=dev)
        keep = torch.empty(n * (2 + k) + 1, dtype=torch.float32, device=dev)      # stats (n, 2), q (n, k), count
        ws = _scratch(lib.istnet_distill_scratch_kib(n, v, k), dev)
        at = keep.data_ptr()
        _launch(dev, "distill_forward", lib.istnet_distill_forward, n, v, k, DTYPES[z.dtype], DTYPES[top.dtype],
                ids.dtype == torch.int64, z.data_ptr(), ldz, top.data_ptr(), ids.data_ptr(), temperature, reduction,
                loss.data_ptr(), at, at + 8 * n, at + 4 * n * (2 + k), ws.data_ptr())
        ctx.save_for_backward(logits, ids, keep)
        ctx.args = (temperature, reduction)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        logits, ids, keep = ctx.saved_tensors
        temperature, reduction = ctx.args
        dev, (n, v), k = logits.device, logits.shape, ids.shape[1]
        z, ldz = _rows(logits)
        gout = gout.contiguous()
        dz = torch.empty((n, v), dtype=logits.dtype, device=dev)
        at = keep.data_ptr()
        _launch(dev, "distill_backward", _native.lib().istnet_distill_backward, n, v, k, DTYPES[z.dtype],
                ids.dtype == torch.int64, z.data_ptr(), ldz, ids.data_ptr(), temperature, reduction, gout.data_ptr(), at,
                at + 8 * n, at + 4 * n * (2 + k), dz.data_ptr())
        return dz, None, None, None, None


class LinearCEFunction(Function):
    """x (N, D), weight (V, D), bias (V) or None, target (N) -> loss (N,) or scalar, float32; gradients for x, weight, bias.
    ``train``: a backward may follow."""

    @staticmethod
    def forward(ctx, x, weight, bias, target, ignore, reduction, train):
        dev, (n, d), v, dtype = x.device, x.shape, weight.shape[0], DTYPES[x.dtype]
        lib = _native.lib()
        xr, ldx = _rows(x)
        w, ldw = _rows(weight)
        b, t = (None if bias is None else bias.contiguous()), target.contiguous()
        loss = torch.empty((n,) if reduction == 0 else (), dtype=torch.float32, device=dev)
        keep = _scratch(lib.istnet_linear_ce_keep_kib(n, d, v, dtype, train, w.data_ptr(), ldw), dev)
        ws = _scratch(lib.istnet_linear_ce_scratch_kib(n, d, v, dtype, reduction, 0), dev)
        _launch(dev, "linear_ce_forward", lib.istnet_linear_ce_forward, n, d, v, dtype, t.dtype == torch.int64, train, xr.data_ptr(),
                ldx, w.data_ptr(), ldw, None if b is None else b.data_ptr(), t.data_ptr(), ignore, reduction, loss.data_ptr(),
                keep.data_ptr(), ws.data_ptr())
        if train:
            ctx.save_for_backward(x, weight, keep)
            ctx.args = (reduction, None if bias is None else bias.dtype)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        x, weight, keep = ctx.saved_tensors
        reduction, bias_type = ctx.args
        dev, (n, d), v, dtype = x.device, x.shape, weight.shape[0], DTYPES[x.dtype]
        lib = _native.lib()
        xr, ldx = _rows(x)
        w, ldw = _rows(weight)
        gout = gout.contiguous()
        need = ctx.needs_input_grad
        dx = torch.empty((n, d), dtype=x.dtype, device=dev) if need[0] else None
        dw = torch.empty((v, d), dtype=x.dtype, device=dev) if need[1] else None
        db = torch.empty((v,), dtype=bias_type, device=dev) if need[2] else None
        ws = _scratch(lib.istnet_linear_ce_scratch_kib(n, d, v, dtype, reduction, 1), dev)
        _launch(dev, "linear_ce_backward", lib.istnet_linear_ce_backward, n, d, v, dtype, xr.data_ptr(), ldx, w.data_ptr(), ldw,
                bias_type is not None, reduction, gout.data_ptr(), keep.data_ptr(), ws.data_ptr(),
                *(None if t is None else t.data_ptr() for t in (dx, dw, db)))
        return dx, dw, db, None, None, None, None
