"""Autograd Functions over csrc/xq_drop.hip and csrc/xq_embed.hip: the operators of a token model that reads the tokenizer's codes (dropout with a
counter-based generator, embedding with a sorted gradient).  The public entry points are nn_ops.dropout / nn_ops.embedding; everything here takes
tensors that live on an MI355X.  Every call enqueues on the current stream of its tensors' device and allocates its outputs and workspace there."""
import torch

from . import _lib
from ._lib import XqError, check

_TYPES = (torch.bfloat16, torch.float32)
_raw_stream = torch._C._cuda_getCurrentRawStream       # the handle alone: torch.cuda.current_stream builds an object, 4 us of a 5 us call
_current_device = torch._C._cuda_getDevice


def _launch(name, device, *args):
    """one C entry point on the current stream of `device`, which is made the current device only where it is not"""
    fn = getattr(_lib.lib(), name)
    i = device.index
    if _current_device() == i:
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _raw_stream(i))
    if rc:
        check(rc, name)


def _at(t):
    return None if t is None else t.data_ptr()


def _same_device(name, first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise XqError(f"{name}: all tensors have to live on one device (got {first.device} and {t.device})")


# ---- dropout -------------------------------------------------------------------------------------------------------------------------------

def _dense(t):
    """whether the elements of t fill its memory without holes or overlaps, in whatever order (contiguous, channels-last, transposed, ...)"""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((st, sz) for sz, st in zip(t.shape, t.stride()) if sz != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _like(t, ref):
    """t with the memory order of the dense tensor `ref`"""
    if t.stride() == ref.stride():
        return t
    out = torch.empty_like(ref, dtype=t.dtype)
    out.copy_(t)
    return out


def _dropout(x, residual, p, key, out_dtype):
    y = torch.empty_like(x, dtype=out_dtype)          # keeps the strides of a dense x
    _launch("xq_dropout", x.device, x.data_ptr(), x.dtype == torch.bfloat16, _at(residual), x.numel(), p, key.data_ptr(), y.data_ptr(),
            out_dtype == torch.bfloat16)
    return y


class DropoutFn(torch.autograd.Function):
    """y = dropout(x) [+ residual]; keeps the 16-byte key for the backward pass, no mask.  xq_dropout in both directions."""

    @staticmethod
    def forward(ctx, x, residual, p, key):
        xd = x.detach()
        if not _dense(xd):
            xd = xd.contiguous()
        rd = None if residual is None else _like(residual.detach(), xd)
        ctx.save_for_backward(key)
        ctx.cfg = (p, xd.dtype, xd.stride())
        return _dropout(xd, rd, p, key, xd.dtype if rd is None else rd.dtype)

    @staticmethod
    def backward(ctx, g):
        (key,) = ctx.saved_tensors
        p, dtype, stride = ctx.cfg
        dx = None
        if ctx.needs_input_grad[0]:
            gd = g.detach()
            if gd.stride() != stride:                  # the mask belongs to places in memory: the gradient has to lie as x did
                gd = torch.empty_strided(g.shape, stride, dtype=g.dtype, device=g.device).copy_(gd)
            dx = _dropout(gd, None, p, key, dtype)
        return dx, (g if ctx.needs_input_grad[1] else None), None, None


def dropout(x, p, key=None, residual=None):
    if x.dtype not in _TYPES:
        raise XqError(f"dropout: x of type {x.dtype} (bf16 / fp32)")
    if not 0.0 <= p <= 1.0:
        raise XqError(f"dropout: p = {p} does not lie in [0, 1]")
    if residual is not None:
        if residual.shape != x.shape:
            raise XqError(f"dropout: residual of shape {tuple(residual.shape)} for x of shape {tuple(x.shape)}")
        if residual.dtype != x.dtype and residual.dtype != torch.float32:
            raise XqError(f"dropout: residual of type {residual.dtype} for x of type {x.dtype} (x's own type or fp32)")
    if key is None:
        # from the device's default generator: follows torch.manual_seed, and a captured graph draws anew at every replay
        key = torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), dtype=torch.int64, device=x.device)
    elif key.dtype != torch.int64 or tuple(key.shape) != (2,) or not key.is_contiguous():
        raise XqError(f"dropout: key is an int64 tensor of two values (got {key.dtype}, shape {tuple(key.shape)})")
    _same_device("dropout", x, residual, key)
    return DropoutFn.apply(x, residual, float(p), key)


# ---- embedding -----------------------------------------------------------------------------------------------------------------------------

class EmbeddingFn(torch.autograd.Function):
    """y = scale * weight[idx] (xq_embedding_forward); the gradient of the table from the tokens sorted by row (xq_embedding_backward)."""

    @staticmethod
    def forward(ctx, idx, weight, scale, skip, dtype):
        ic, w = idx.contiguous(), weight.detach().contiguous()
        V, D = w.shape
        y = torch.empty(*idx.shape, D, dtype=dtype, device=w.device)
        _launch("xq_embedding_forward", w.device, ic.data_ptr(), ic.dtype == torch.int64, w.data_ptr(), w.dtype == torch.bfloat16, ic.numel(), V, D, scale,
                y.data_ptr(), dtype == torch.bfloat16)
        if ctx.needs_input_grad[1]:
            ctx.save_for_backward(ic)
            ctx.cfg = (V, D, scale, skip, w.dtype)
        return y

    @staticmethod
    def backward(ctx, g):
        (ic,) = ctx.saved_tensors
        V, D, scale, skip, wdtype = ctx.cfg
        gc = g.detach().contiguous()
        dw = torch.empty(V, D, dtype=wdtype, device=g.device)
        N = ic.numel()
        nbytes = _lib.lib().xq_embedding_backward_workspace_bytes(N, V, D)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=g.device) if nbytes else None
        _launch("xq_embedding_backward", gc.device, ic.data_ptr(), ic.dtype == torch.int64, gc.data_ptr(), gc.dtype == torch.bfloat16, N, V, D, scale, skip,
                dw.data_ptr(), wdtype == torch.bfloat16, _at(ws), nbytes)
        return None, dw, None, None, None


def embedding(idx, weight, scale=1.0, padding_idx=None, dtype=None):
    dtype = weight.dtype if dtype is None else dtype
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise XqError(f"embedding: the table is (rows, width) (got shape {tuple(weight.shape)})")
    if weight.dtype not in _TYPES or dtype not in _TYPES:
        raise XqError(f"embedding: table of type {weight.dtype}, result of type {dtype} (bf16 / fp32)")
    if idx.dtype not in (torch.int64, torch.int32):
        raise XqError(f"embedding: indices of type {idx.dtype} (int64 / int32)")
    skip = -1
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise XqError(f"embedding: padding_idx = {padding_idx} outside the table of {weight.shape[0]} rows")
        skip = padding_idx % weight.shape[0]
    _same_device("embedding", weight, idx)
    return EmbeddingFn.apply(idx, weight, float(scale), skip, dtype)
