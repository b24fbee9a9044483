"""Autograd Functions over csrc/xq_drop.hip, csrc/xq_embed.hip and csrc/xq_xattn.hip: the operators of a token model that reads the tokenizer's codes
(dropout with a counter-based generator, embedding with a sorted gradient, attention to another sequence).  The public entry points are nn_ops.dropout,
nn_ops.embedding and nn_ops.cross_attention; everything here takes tensors that live on an MI355X.  Every call enqueues on the current stream of its
tensors' device and allocates its outputs and workspace there."""
import ctypes
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import XqError, check

_TYPES = (torch.bfloat16, torch.float32)
_raw_stream = torch._C._cuda_getCurrentRawStream       # the handle alone: torch.cuda.current_stream builds an object, 4 us of a 5 us call
_current_device = torch._C._cuda_getDevice
is_tracing = torch._C._is_tracing                        # (torch.jit.is_tracing asks this and more, for half a microsecond)


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


def _wants_node(*tensors):
    """whether autograd has to see the call (an autograd node costs a small call as much as its kernel): a gradient is wanted, tangents may be on their way (a dual
    tensor requires no gradient; the node refuses it, the bare kernel would drop its tangent), or a trace records the call (it sees the node, not the kernel)"""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return forward_ad._current_level >= 0 or is_tracing()


def transformed():
    """whether something other than plain autograd looks on (a compiler's tracing, an open forward-mode level, torch.func's transforms): where a kernel stands for a library
    operator that has formulas for those, the operator runs"""
    return torch.compiler.is_compiling() or forward_ad._current_level >= 0 or torch._C._are_functorch_transforms_active()


def _same_device(name, first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise XqError(f"{name}: all tensors have to live on one device (got {first.device} and {t.device})")


def _first_order(backward):
    """a backward pass through a kernel has no graph of its own: differentiating through it is an error, not a zero (the check for it only where a graph is asked for)"""
    checked = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return (checked if torch.is_grad_enabled() else backward)(ctx, *grads)
    return run


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
        xd = x if _dense(x) else x.contiguous()
        rd = None if residual is None else _like(residual, xd)
        ctx.save_for_backward(key)
        ctx.cfg = (p, xd.dtype, xd.stride())
        return _dropout(xd, rd, p, key, xd.dtype if rd is None else rd.dtype)

    @staticmethod
    @_first_order
    def backward(ctx, g):
        (key,) = ctx.saved_tensors
        p, dtype, stride = ctx.cfg
        dx = None
        if ctx.needs_input_grad[0]:
            gd = g
            if gd.stride() != stride:                  # the mask belongs to places in memory: the gradient has to lie as x did
                gd = torch.empty_strided(g.shape, stride, dtype=g.dtype, device=g.device).copy_(g)
            dx = _dropout(gd, None, p, key, dtype)
        return dx, (g if ctx.needs_input_grad[1] else None), None, None


def check_dropout(x, p, residual):
    """what holds on whatever device, training or not"""
    if not 0.0 <= p <= 1.0:
        raise XqError(f"dropout: p = {p} does not lie in [0, 1]")
    if residual is not None:
        if residual.shape != x.shape:
            raise XqError(f"dropout: residual of shape {tuple(residual.shape)} for x of shape {tuple(x.shape)}")
        if residual.dtype != x.dtype and residual.dtype != torch.float32:
            raise XqError(f"dropout: residual of type {residual.dtype} for x of type {x.dtype} (x's own type or fp32)")


def dropout(x, p, key=None, residual=None):
    if x.dtype not in _TYPES:
        raise XqError(f"dropout: x of type {x.dtype} (bf16 / fp32)")
    check_dropout(x, p, residual)
    if key is None:
        # from the device's default generator: follows torch.manual_seed, and a captured graph draws anew at every replay
        key = torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), dtype=torch.int64, device=x.device)
    elif key.dtype != torch.int64 or tuple(key.shape) != (2,) or not key.is_contiguous():
        raise XqError(f"dropout: key is an int64 tensor of two values (got {key.dtype}, shape {tuple(key.shape)})")
    _same_device("dropout", x, residual, key)
    if not _wants_node(x, residual):
        xd = x if _dense(x) else x.contiguous()
        rd = None if residual is None else _like(residual, xd)
        return _dropout(xd, rd, float(p), key, x.dtype if rd is None else rd.dtype)
    return DropoutFn.apply(x, residual, float(p), key)


# ---- embedding -----------------------------------------------------------------------------------------------------------------------------

MAX_ROWS = 1 << 20                                     # of a table, csrc/xq_embed.hip


def _embedding(ic, w, scale, dtype):
    V, D = w.shape
    y = w.new_empty((*ic.shape, D), dtype=dtype)
    _launch("xq_embedding_forward", w.device, ic.data_ptr(), ic.dtype == torch.int64, w.data_ptr(), w.dtype == torch.bfloat16, ic.numel(), V, D, scale,
            y.data_ptr(), dtype == torch.bfloat16)
    return y


@functools.lru_cache(maxsize=4096)
def _embedding_workspace(N, V, D):
    return _lib.lib().xq_embedding_backward_workspace_bytes(N, V, D)


def _embedding_gradient(ic, g, V, D, scale, skip, wdtype):
    gc = g.contiguous()
    dw = gc.new_empty((V, D), dtype=wdtype)
    N = ic.numel()
    nbytes = _embedding_workspace(N, V, D)
    ws = gc.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch("xq_embedding_backward", gc.device, ic.data_ptr(), ic.dtype == torch.int64, gc.data_ptr(), gc.dtype == torch.bfloat16, N, V, D, scale, skip,
            dw.data_ptr(), wdtype == torch.bfloat16, _at(ws), nbytes)
    return dw


class EmbeddingFn(torch.autograd.Function):
    """y = scale * weight[idx] (xq_embedding_forward); the gradient of the table from the tokens sorted by row (xq_embedding_backward)."""

    @staticmethod
    def forward(ctx, idx, weight, scale, skip, dtype):
        ic, w = idx.contiguous(), weight.contiguous()
        ctx.save_for_backward(ic)
        ctx.cfg = (*w.shape, scale, skip, w.dtype)
        return _embedding(ic, w, scale, dtype)

    @staticmethod
    @_first_order
    def backward(ctx, g):
        return None, _embedding_gradient(*ctx.saved_tensors, g, *ctx.cfg), None, None, None


class EmbeddingAgainFn(EmbeddingFn):
    """the lookup of an nn.Embedding, whose gradient can be differentiated again as the module's can"""

    @staticmethod
    def backward(ctx, g):
        f = EmbeddingGradientFn.apply if torch.is_grad_enabled() else _embedding_gradient
        return None, f(*ctx.saved_tensors, g, *ctx.cfg), None, None, None


class EmbeddingGradientFn(torch.autograd.Function):
    """the gradient of the table is linear in g: its own gradient is the lookup of what comes back, zeros where g added nothing"""

    @staticmethod
    def forward(ctx, ic, g, V, D, scale, skip, wdtype):
        ctx.save_for_backward(ic)
        ctx.cfg = (V, scale, skip, g.dtype)
        return _embedding_gradient(ic, g, V, D, scale, skip, wdtype)

    @staticmethod
    def backward(ctx, gg):
        (ic,) = ctx.saved_tensors
        V, scale, skip, dtype = ctx.cfg
        dg = embedding(ic, gg, scale, None, dtype, again=True)
        return None, torch.where(((ic >= 0) & (ic < V) & (ic != skip)).unsqueeze(-1), dg, torch.zeros_like(dg)), None, None, None, None, None


def embedding(idx, weight, scale=1.0, padding_idx=None, dtype=None, again=False):
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
    if not _wants_node(weight):
        return _embedding(idx.contiguous(), weight.contiguous(), float(scale), dtype)
    return (EmbeddingAgainFn if again else EmbeddingFn).apply(idx, weight, float(scale), skip, dtype)


# ---- attention to another sequence ---------------------------------------------------------------------------------------------------------

_NINE = ctypes.c_int64 * 9


def _rows(t, group=1):
    """t (B, N, heads, D) as the kernels read it: elements of a row side by side, rows 16-byte aligned, 64 tokens and the `group` heads that share a kv head within
    2^30 elements; a copy where it is not"""
    s = t.stride()
    if (s[3] == 1 or t.shape[3] == 1) and not (s[0] | s[1] | s[2]) & 7 and not t.data_ptr() & 15 and s[1] <= 1 << 23 and s[2] <= 1 << 22 and (
            64 * s[1] + group * s[2] <= 1 << 30):
        return t
    if t.is_contiguous() and not t.data_ptr() & 15:
        return t                                       # (strides of dimensions of one element may be anything: _nine leaves them out)
    return t.clone(memory_format=torch.contiguous_format)


def _nine(shapes, strides):
    return _NINE(*[0 if n == 1 else st for shape, stride in zip(shapes, strides) for n, st in zip(shape[:3], stride[:3])])


@functools.lru_cache(maxsize=4096)
def _xattn_plan(q, k, sq, sk, sv, sdq, sdk, sdv):
    """by shapes and strides alone: the sizes and stride arrays of the C calls, and their workspaces' bytes"""
    sizes = (q[0], q[1], k[1], q[2], k[2], q[3])
    l = _lib.lib()
    return (sizes, _nine((q, k, k), (sq, sk, sv)), l.xq_xattn_forward_workspace_bytes(*sizes),
            l.xq_xattn_backward_workspace_bytes(*sizes) if sdq else 0, _nine((q, k, k), (sdq, sdk, sdv)) if sdq else None)


def _xattn_forward(q, k, v, lens, mask, scale, want_lse):
    sizes, strides, nbytes, _, _ = _xattn_plan(q.shape, k.shape, q.stride(), k.stride(), v.stride(), None, None, None)
    out = q.new_empty(q.shape)
    lse = q.new_empty((sizes[0], sizes[4], sizes[1] * (sizes[3] // sizes[4])), dtype=torch.float32) if want_lse else None
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch("xq_xattn_forward", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), *sizes, strides, _at(lens), lens is not None and lens.dtype == torch.int64,
            _at(mask), scale, out.data_ptr(), _at(lse), _at(ws), nbytes)
    return out, lse


def _xattn_backward(q, k, v, out, g, lse, lens, mask, scale, dq, dk, dv):
    if not g.is_contiguous() or g.data_ptr() & 15:
        g = g.clone(memory_format=torch.contiguous_format)
    sizes, strides, _, nbytes, grad_strides = _xattn_plan(q.shape, k.shape, q.stride(), k.stride(), v.stride(), dq.stride(), dk.stride(), dv.stride())
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch("xq_xattn_backward", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), g.data_ptr(), lse.data_ptr(), *sizes, strides, _at(lens),
            lens is not None and lens.dtype == torch.int64, _at(mask), scale, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), grad_strides, _at(ws), nbytes)


class CrossAttentionFn(torch.autograd.Function):
    """softmax(scale q k^T over valid keys) v: xq_xattn_forward / xq_xattn_backward"""

    @staticmethod
    def forward(ctx, q, k, v, lens, mask, scale):
        q, k, v = _rows(q, q.shape[2] // k.shape[2]), _rows(k), _rows(v)
        out, lse = _xattn_forward(q, k, v, lens, mask, scale, True)
        ctx.save_for_backward(q, k, v, out, lse, lens, mask)
        ctx.scale = scale
        return out

    @staticmethod
    @_first_order
    def backward(ctx, g):
        q, k, v, out, lse, lens, mask = ctx.saved_tensors
        dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        _xattn_backward(q, k, v, out, g, lse, lens, mask, ctx.scale, dq, dk, dv)
        return dq, dk, dv, None, None, None


def _packed_forward(x, num_heads, want_lse):
    B, N, C3 = x.shape
    x = x.contiguous()
    if x.data_ptr() & 15:
        x = x.clone()
    q, k, v = x.view(B, N, 3, num_heads, C3 // (3 * num_heads)).unbind(2)
    scale = float(q.shape[3]) ** -0.5
    out, lse = _xattn_forward(q, k, v, None, None, scale, want_lse)
    return x, out, lse, scale


class PackedAttentionFn(torch.autograd.Function):
    """self-attention on the packed (B, N, 3, H, D) projection through the same kernels, for the head widths that csrc/xq_attn.hip (64) does not take"""

    @staticmethod
    def forward(ctx, qkv, num_heads):
        x, out, lse, ctx.scale = _packed_forward(qkv.detach(), num_heads, True)
        ctx.save_for_backward(x, out, lse)
        return out.flatten(2)

    @staticmethod
    @_first_order
    def backward(ctx, g):
        x, out, lse = ctx.saved_tensors
        B, N, H, D = out.shape
        dx = torch.empty_like(x)
        _xattn_backward(*x.view(B, N, 3, H, D).unbind(2), out, g.detach().to(x.dtype).reshape(B, N, H, D), lse, None, None, ctx.scale,
                        *dx.view(B, N, 3, H, D).unbind(2))
        return dx, None


def packed_attention(qkv, num_heads):
    if _wants_node(qkv):
        return PackedAttentionFn.apply(qkv, num_heads)
    return _packed_forward(qkv, num_heads, False)[1].flatten(2)


def packed_attention_supported(qkv, num_heads):
    if not (qkv.is_cuda and qkv.dtype == torch.bfloat16 and qkv.dim() == 3) or transformed():
        return False
    B, N, C3 = qkv.shape
    D = C3 // (3 * num_heads)
    if C3 != 3 * num_heads * D or D % 8 or not 8 <= D <= 128:
        return False
    # xq_xattn_forward's limits on one call (blocks of a launch; 64 tokens of the packed projection within 32 bits of bytes)
    return B * num_heads * ((N + 127) // 128 + 8) <= 1 << 22 and B * num_heads * N <= 0x3fffffff and C3 <= 1 << 23


@functools.lru_cache(maxsize=4096)
def _check_shapes(q, k, v, lens, mask, scale):
    """by shapes and types alone (lens, mask: (shape, type) or None) -> the scale"""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if len(t) != 4:
            raise XqError(f"cross_attention: {name} is (batch, tokens, heads, head dim) (got shape {tuple(t)})")
    B, Nq, H, D = q
    Nk, Hk = k[1], k[2]
    if k != v or k[0] != B or k[3] != D:
        raise XqError(f"cross_attention: q {tuple(q)}, k {tuple(k)} and v {tuple(v)} do not go together")
    if H < 1 or Hk < 1 or H % Hk:
        raise XqError(f"cross_attention: {H} query heads do not share {Hk} key / value heads evenly")
    if D < 1:
        raise XqError("cross_attention: a head dim of 0")
    if lens is not None and (tuple(lens[0]) != (B,) or lens[1] not in (torch.int32, torch.int64)):
        raise XqError(f"cross_attention: kv_lens is an int32 or int64 tensor of {B} lengths (got {lens[1]}, shape {tuple(lens[0])})")
    if mask is not None and (tuple(mask[0]) != (B, Nk) or mask[1] != torch.bool):
        raise XqError(f"cross_attention: key_mask is a bool tensor of shape {(B, Nk)} (got {mask[1]}, shape {tuple(mask[0])})")
    scale = float(D) ** -0.5 if scale is None else scale
    if not 2.0 ** -64 <= scale <= 2.0 ** 64:
        raise XqError(f"cross_attention: scale = {scale} is not positive, 2^-64 .. 2^64")
    return scale


def check_cross_attention(q, k, v, kv_lens, key_mask, scale):
    """shapes and types, on whatever device -> the scale"""
    return _check_shapes(q.shape, k.shape, v.shape, None if kv_lens is None else (kv_lens.shape, kv_lens.dtype),
                         None if key_mask is None else (key_mask.shape, key_mask.dtype), None if scale is None else float(scale))


def cross_attention(q, k, v, kv_lens=None, key_mask=None, scale=None):
    scale = check_cross_attention(q, k, v, kv_lens, key_mask, scale)
    if q.dtype != torch.bfloat16 or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise XqError(f"cross_attention: q, k, v of types {q.dtype}, {k.dtype}, {v.dtype} (bf16; other types under bf16 autocast)")
    if q.shape[3] % 8 or q.shape[3] > 128:
        raise XqError(f"cross_attention: head dim {q.shape[3]} is not a multiple of 8 up to 128")
    _same_device("cross_attention", q, k, v, kv_lens, key_mask)
    kv_lens = None if kv_lens is None else kv_lens.contiguous()
    key_mask = None if key_mask is None else key_mask.contiguous()
    if not _wants_node(q, k, v):
        return _xattn_forward(_rows(q, q.shape[2] // k.shape[2]), _rows(k), _rows(v), kv_lens, key_mask, scale, False)[0]
    return CrossAttentionFn.apply(q, k, v, kv_lens, key_mask, scale)
