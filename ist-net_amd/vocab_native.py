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
INDEX = {torch.int32: 0, torch.int64: 1}
REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}

# The host's work is what a small call costs, so that checks build their messages only when they fail, tensors are taken from the
# allocator at once, and the device and stream are asked for without the wrappers of torch.cuda.


def _once(fn):
    """once_differentiable at no cost where no graph of the backward is asked for."""
    graph = once_differentiable(fn)

    def backward(ctx, *grads):
        return graph(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)
    return staticmethod(backward)


def check_float(t, name):
    if t.dtype not in DTYPES:
        raise TypeError(f"{name} must be a float32, bfloat16 or float16 tensor, got {t.dtype}")


def check_index(t, name):
    if t.dtype not in INDEX:
        raise TypeError(f"{name} must be an int32 or int64 tensor, got {t.dtype}")


def check_device(lead, name, t, other):
    if t.device != lead.device:
        raise RuntimeError(f"{other} must be on the same device as {name}")


def check_reduction(reduction):
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(REDUCTIONS)}, got {reduction!r}")


def _launch(dev, what, fn, *args):
    """fn(*args, current stream of dev) with dev as the current device, which it nearly always is already."""
    if torch._C._cuda_getDevice() == dev.index:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if status:
        _native.check(status, what)


def _rows(t):
    """(tensor, leading dimension) of a 2-D operand with contiguous rows that do not overlap; anything else is copied."""
    if t.is_contiguous():
        return t, t.shape[1]
    n, d = t.shape
    ld, step = t.stride()
    if (step == 1 and ld >= d) or (d == 1 and ld >= 1):
        return t, ld
    return t.contiguous(), d


def _scratch(kib, dev):
    """The tensor (to be kept until the call that uses it was made) and its address."""
    if kib == 0:
        return None, None
    t = torch.empty(kib * 1024, dtype=torch.uint8, device=dev)
    return t, t.data_ptr()


class EmbeddingFunction(Function):
    """weight (V, D), idx (...) -> scale * weight[idx] (..., D); gradient for weight."""

    @staticmethod
    def forward(ctx, weight, idx, scale, padding):
        dev, (v, d), n = weight.device, weight.shape, idx.numel()
        out = weight.new_empty((*idx.shape, d))
        ids = idx if idx.is_contiguous() else idx.contiguous()
        if n:
            w, ldw = _rows(weight)
            _launch(dev, "embed_forward", _native.lib().istnet_embed_forward, n, v, d, DTYPES[weight.dtype],
                    INDEX[ids.dtype], w.data_ptr(), ldw, ids.data_ptr(), scale, out.data_ptr())
        ctx.save_for_backward(ids)
        ctx.args = (v, d, scale, padding, weight.dtype)
        return out

    @_once
    def backward(ctx, grad_out):
        (ids,) = ctx.saved_tensors
        v, d, scale, padding, dtype = ctx.args
        dev, n = ids.device, ids.numel()
        if n == 0:
            return torch.zeros((v, d), dtype=dtype, device=dev), None, None, None
        g, ldg = _rows(grad_out if grad_out.dim() == 2 else grad_out.reshape(n, d))
        dw = g.new_empty((v, d))
        lib = _native.lib()
        ws, at = _scratch(lib.istnet_embed_scratch_kib(n, v, d), dev)
        _launch(dev, "embed_backward", lib.istnet_embed_backward, n, v, d, DTYPES[dtype], INDEX[ids.dtype], g.data_ptr(),
                ldg, ids.data_ptr(), -1 if padding is None else padding, scale, at, dw.data_ptr())
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
        ws, at_ws = _scratch(lib.istnet_distill_scratch_kib(n, v, k), dev)
        at = keep.data_ptr()
        _launch(dev, "distill_forward", lib.istnet_distill_forward, n, v, k, DTYPES[z.dtype], DTYPES[top.dtype],
                INDEX[ids.dtype], z.data_ptr(), ldz, top.data_ptr(), ids.data_ptr(), temperature, reduction,
                loss.data_ptr(), at, at + 8 * n, at + 4 * n * (2 + k), at_ws)
        ctx.save_for_backward(logits, ids, keep)
        ctx.args = (temperature, reduction)
        return loss

    @_once
    def backward(ctx, gout):
        logits, ids, keep = ctx.saved_tensors
        temperature, reduction = ctx.args
        dev, (n, v), k = logits.device, logits.shape, ids.shape[1]
        z, ldz = _rows(logits)
        gout = gout.contiguous()
        dz = torch.empty((n, v), dtype=logits.dtype, device=dev)
        at = keep.data_ptr()
        _launch(dev, "distill_backward", _native.lib().istnet_distill_backward, n, v, k, DTYPES[z.dtype],
                INDEX[ids.dtype], z.data_ptr(), ldz, ids.data_ptr(), temperature, reduction, gout.data_ptr(), at,
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
        b, t = (None if bias is None else bias.contiguous()), target if target.is_contiguous() else target.contiguous()
        loss = torch.empty((n,) if reduction == 0 else (), dtype=torch.float32, device=dev)
        keep, at = _scratch(lib.istnet_linear_ce_keep_kib(n, d, v, dtype, train, w.data_ptr(), ldw), dev)
        ws, at_ws = _scratch(lib.istnet_linear_ce_scratch_kib(n, d, v, dtype, reduction, 0), dev)
        _launch(dev, "linear_ce_forward", lib.istnet_linear_ce_forward, n, d, v, dtype, INDEX[t.dtype], train, xr.data_ptr(),
                ldx, w.data_ptr(), ldw, None if b is None else b.data_ptr(), t.data_ptr(), ignore, reduction, loss.data_ptr(),
                at, at_ws)
        if train:
            ctx.save_for_backward(x, weight, keep)
            ctx.args = (reduction, bias is not None)
        return loss

    @_once
    def backward(ctx, gout):
        x, weight, keep = ctx.saved_tensors
        reduction, biased = ctx.args
        dev, (n, d), v, dtype = x.device, x.shape, weight.shape[0], DTYPES[x.dtype]
        lib = _native.lib()
        xr, ldx = _rows(x)
        w, ldw = _rows(weight)
        gout = gout if gout.is_contiguous() else gout.contiguous()
        need = ctx.needs_input_grad
        dx = x.new_empty((n, d)) if need[0] else None
        dw = x.new_empty((v, d)) if need[1] else None
        db = x.new_empty((v,)) if need[2] else None
        ws, at_ws = _scratch(lib.istnet_linear_ce_scratch_kib(n, d, v, dtype, reduction, 1), dev)
        _launch(dev, "linear_ce_backward", lib.istnet_linear_ce_backward, n, d, v, dtype, xr.data_ptr(), ldx, w.data_ptr(), ldw,
                biased, reduction, gout.data_ptr(), keep.data_ptr(), at_ws, None if dx is None else dx.data_ptr(),
                None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr())
        return dx, dw, db, None, None, None, None
