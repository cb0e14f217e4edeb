"""Operators of a training or serving step with 16-bit storage, over the C ABI (csrc/lookup.hip, linear_act.hip,
grad_clip.hip), next to the fp32 operators of plnlp_amd/ops.py:

  embedding_lookup   scale * table[ids], and the table's gradient summed by id
  linear_act         activation(x W^T + bias) + residual, and its gradients
  grad_norm          the norm of a list of gradients taken as one vector
  clip_grads         the gradients scaled so that this norm stays below a limit (in place, or into other tensors)

All sums are held in 32 bits or more and every result is rounded once; what linear_act's backward pass rounds on the way, its docstring
says.  All are deterministic.  Work is enqueued on the current stream of the current device, on which every tensor has to be; nothing
waits for it.  All may be captured into a graph (a backward pass, as any of torch's, only while no graph of the same leaves is alive
that was recorded before the capture).  Like the rest of the package there is no CPU path.  Gradients are those of reverse mode, of first order: second ones, and operands with
a forward-mode tangent, are refused."""
from __future__ import annotations

import math
from typing import List, Optional, Sequence

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L

_HALF = (torch.bfloat16, torch.float16)


def _stream(*tensors: Optional[torch.Tensor]) -> int:
    """the current stream, once every tensor is known to be on its device (L.require_device says what is wrong if one is not)"""
    device = tensors[0].get_device()
    if device < 0 or device != torch.cuda.current_device():
        L.require_device(*tensors)
    for t in tensors:
        if t is not None and t.get_device() != device:
            L.require_device(*tensors)
    return L.stream_ptr()


def _no_tangent(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """refuses operands with a forward-mode tangent, which no operator here carries on (the kernels see addresses alone); outside a
    dual level, where there are none, nothing is asked"""
    if getattr(forward_ad, "_current_level", 0) < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what}: there is no forward-mode derivative, and an operand carries a tangent")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """a matrix with consecutive elements along its rows and rows that do not overlap: t itself, or a contiguous copy"""
    if t.is_contiguous():
        return t
    rows, cols = t.shape
    if rows == 0 or cols == 0:
        return t
    if (cols > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < cols):
        return t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    """elements between the rows of a matrix as _rows gives it (a single row: any; then its width)"""
    rows, cols = t.shape
    return t.stride(0) if rows > 1 else cols


def _workspace(n_bytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(n_bytes, dtype=torch.uint8, device=device) if n_bytes > 0 else None


# ------------------------------------------------------------------ lookup ------
def _lookup_rows(table: torch.Tensor, ids: torch.Tensor, scale: float, out_dtype: torch.dtype) -> torch.Tensor:
    stream = _stream(table, ids)
    table, flat = _rows(table), ids.contiguous()
    rows, width = table.shape
    out = table.new_empty((*ids.shape, width), dtype=out_dtype)
    L.check(L.load().plnlp_embedding_lookup(table.data_ptr(), _ld(table), L.DTYPE_CODES[table.dtype], rows, width, flat.data_ptr(),
                                            flat.element_size(), flat.numel(), scale, out.data_ptr(), max(width, 1),
                                            L.DTYPE_CODES[out_dtype], stream), "plnlp_embedding_lookup")
    return out


def _lookup_grad(gy: torch.Tensor, ids: torch.Tensor, n_rows: int, padding: int, scale: float, dtype: torch.dtype) -> torch.Tensor:
    lib = L.load()
    width = gy.shape[-1]
    stream = _stream(gy, ids)
    gy = _rows(gy.reshape(ids.numel(), width))
    flat = ids.contiguous()
    grad = torch.empty(n_rows, width, dtype=dtype, device=gy.device)
    n_bytes = lib.plnlp_embedding_grad_workspace_bytes(flat.numel(), width)
    ws = _workspace(n_bytes, gy.device)
    L.check(lib.plnlp_embedding_grad(gy.data_ptr(), max(_ld(gy), width), L.DTYPE_CODES[gy.dtype], flat.data_ptr(), flat.element_size(),
                                     flat.numel(), padding, scale, grad.data_ptr(), max(width, 1), L.DTYPE_CODES[dtype], n_rows, width,
                                     L.ptr(ws), n_bytes, stream), "plnlp_embedding_grad")
    return grad


class EmbeddingLookupFn(torch.autograd.Function):
    """scale * table[ids]; the gradient adds the rows of equal ids in the order of their positions"""

    @staticmethod
    def forward(ctx, table, ids, scale: float, padding: int, out_dtype):
        ctx.save_for_backward(ids)
        ctx.rest = (table.shape[0], padding, scale, table.dtype)
        return _lookup_rows(table, ids, scale, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        n_rows, padding, scale, dtype = ctx.rest
        return _lookup_grad(gy, ctx.saved_tensors[0], n_rows, padding, scale, dtype), None, None, None, None


def embedding_lookup(table: torch.Tensor, ids: torch.Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None,
                     out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """out[..., :] = scale * table[ids[...], :].

    table: [V, D], bf16, fp16 or fp32 (rows may be strided); ids: int32 or int64 of any shape; out_dtype: the result's type
    (default: the table's).  An id outside [0, V) -- the -1 of a padded batch -- reads as a row of zeros and gives no
    gradient.  padding_idx: a row (negative: from the end) that is read like any other and gets no gradient, as in
    torch.nn.Embedding.  The gradient has the table's type and is dense: rows without an id are zero.  At most
    2^31 - 2 rows and ids."""
    if table.dim() != 2 or table.dtype not in L.DTYPE_CODES:
        raise ValueError(f"embedding_lookup: table must be a bf16, fp16 or fp32 matrix, not {table.dtype} {tuple(table.shape)}")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"embedding_lookup: ids must be int32 or int64, not {ids.dtype}")
    out_dtype = table.dtype if out_dtype is None else out_dtype
    if out_dtype not in L.DTYPE_CODES:
        raise TypeError(f"embedding_lookup: out_dtype must be bf16, fp16 or fp32, not {out_dtype}")
    padding = -1
    if padding_idx is not None:
        if not -table.shape[0] <= padding_idx < table.shape[0]:
            raise ValueError(f"embedding_lookup: padding_idx {padding_idx} is no row of a table of {table.shape[0]}")
        padding = padding_idx % table.shape[0]
    _no_tangent("embedding_lookup", table)
    if torch.is_grad_enabled() and table.requires_grad:
        return EmbeddingLookupFn.apply(table, ids, float(scale), padding, out_dtype)
    return _lookup_rows(table, ids, float(scale), out_dtype)


# ------------------------------------------------------------------ linear ------
def _linear_forward(x, weight, bias, residual, act: int, keep: bool):
    """(y [m, n], slope or None) of matrices as _rows gives them; the activation's derivative is kept where the backward pass will
    read it: int16 [m, n], as plnlp_linear_act codes it"""
    stream = _stream(x, weight, bias, residual)
    lib = L.load()
    m, k = x.shape
    n = weight.shape[0]
    out = x.new_empty((m, n))
    slope = x.new_empty((m, n), dtype=torch.int16) if keep else None
    n_bytes = lib.plnlp_linear_act_workspace_bytes(m, n, k)
    ws = _workspace(n_bytes, x.device)
    L.check(lib.plnlp_linear_act(x.data_ptr(), _ld(x), weight.data_ptr(), _ld(weight), L.ptr(bias), L.ptr(residual),
                                 0 if residual is None else _ld(residual), act, m, n, k, L.ptr(slope), n, out.data_ptr(), n,
                                 L.DTYPE_CODES[x.dtype], L.ptr(ws), n_bytes, stream), "plnlp_linear_act")
    return out, slope


class LinearActFn(torch.autograd.Function):
    """act(x W^T + bias) + residual on matrices (linear_act)"""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act: int):
        y, slope = _linear_forward(x, weight, bias, residual, act, act != L.ACTIVATIONS["none"])
        ctx.act = act
        ctx.save_for_backward(x, weight, slope)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        lib = L.load()
        x, weight, slope = ctx.saved_tensors
        need = ctx.needs_input_grad
        m, k = x.shape
        n = weight.shape[0]
        dx = torch.empty(m, k, dtype=x.dtype, device=x.device) if need[0] else None
        dw = torch.empty(n, k, dtype=x.dtype, device=x.device) if need[1] else None
        db = torch.empty(n, dtype=x.dtype, device=x.device) if need[2] else None
        if need[0] or need[1] or need[2]:
            stream = _stream(gy, x, weight)
            g = _rows(gy)
            n_bytes = lib.plnlp_linear_act_backward_workspace_bytes(m, n, k, ctx.act)
            ws = _workspace(n_bytes, x.device)
            L.check(lib.plnlp_linear_act_backward(g.data_ptr(), _ld(g), L.ptr(slope), n, ctx.act, x.data_ptr(), _ld(x), weight.data_ptr(),
                                                  _ld(weight), m, n, k, L.ptr(dx), k, L.ptr(dw), k, L.ptr(db), L.DTYPE_CODES[x.dtype],
                                                  L.ptr(ws), n_bytes, stream), "plnlp_linear_act_backward")
        return dx, dw, db, gy if need[3] else None, None


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
               residual: Optional[torch.Tensor] = None, activation: str = "none") -> torch.Tensor:
    """activation(x W^T + bias) + residual.

    x: [..., K]; weight: [N, K] (torch.nn.Linear's layout); bias: [N]; residual: the result's shape [..., N]; all bf16 or all
    fp16.  activation: "none", "relu", "gelu" (z Phi(z)), "gelu_tanh" or "silu".  The product is summed in fp32; bias,
    activation and residual act on the fp32 sums, which are rounded once.  The activation's derivative is kept
    for the backward pass in 16 bits, where a gradient is wanted: in steps of 2^-14, and between -2^-5 and 0 (saturated units) to
    2^-10 of itself.  The gradients of x and weight are products with dz = dy * derivative rounded to the operands' type, past whose
    range it is infinite (up to 16 384 elements of dz: kept in two terms, to the square of one rounding); bias' sums dz unrounded.
    fp32 matrices are the business of ops.LinearFn."""
    dtype = x.dtype
    if dtype not in _HALF:
        raise TypeError(f"linear_act: x must be bf16 or fp16, not {dtype} (ops.LinearFn is the fp32 layer)")
    act = L.ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"linear_act: activation must be one of {', '.join(L.ACTIVATIONS)}, not {activation!r}")
    shape = x.shape
    if len(shape) < 1 or weight.dim() != 2 or weight.shape[1] != shape[-1]:
        raise ValueError(f"linear_act: x {tuple(shape)} and weight {tuple(weight.shape)} do not match ([..., K] and [N, K])")
    n = weight.shape[0]
    out_shape = (*shape[:-1], n)
    grad = x.requires_grad or weight.requires_grad
    if weight.dtype != dtype:
        raise TypeError(f"linear_act: all operands must have x's type {dtype}; weight is {weight.dtype}")
    if bias is not None:
        if bias.shape != (n,):
            raise ValueError(f"linear_act: bias must have shape ({n},), not {tuple(bias.shape)}")
        if bias.dtype != dtype:
            raise TypeError(f"linear_act: all operands must have x's type {dtype}; bias is {bias.dtype}")
        grad = grad or bias.requires_grad
        bias = bias.contiguous()
    if residual is not None:
        if residual.shape != out_shape:
            raise ValueError(f"linear_act: residual must have the result's shape {out_shape}, not {tuple(residual.shape)}")
        if residual.dtype != dtype:
            raise TypeError(f"linear_act: all operands must have x's type {dtype}; residual is {residual.dtype}")
        grad = grad or residual.requires_grad
    _no_tangent("linear_act", x, weight, bias, residual)
    if len(shape) != 2:
        rows = math.prod(shape[:-1])
        x = x.reshape(rows, shape[-1])
        residual = None if residual is None else residual.reshape(rows, n)
    x, weight = _rows(x), _rows(weight)
    residual = None if residual is None else _rows(residual)
    if grad and torch.is_grad_enabled():
        y = LinearActFn.apply(x, weight, bias, residual, act)
    else:
        y = _linear_forward(x, weight, bias, residual, act, False)[0]
    return y if len(shape) == 2 else y.view(out_shape)


# ------------------------------------------------------------------ clipping ----
_DST_CODES = {t: c << 32 for t, c in L.DTYPE_CODES.items()}
_SIZES = np.array([4, 2, 2], dtype=np.int64)
_OVERLAP = "clip_grads: the memory of a clipped tensor overlaps another tensor of the call (a gradient listed twice?)"


def _norm_kind(norm_type) -> int:
    p = float(norm_type)
    if p == 2.0:
        return L.NORM_L2
    if p == 1.0:
        return L.NORM_L1
    if p == math.inf:
        return L.NORM_MAX
    raise ValueError(f"norm_type must be 1, 2 or inf, not {norm_type!r}")


def _pointers(tensors: Sequence[torch.Tensor], what: str):
    """(addresses, sizes, types) of a list of dense tensors of the three types on the current device"""
    try:
        ptrs = list(map(torch.Tensor.data_ptr, tensors))
    except RuntimeError:
        raise TypeError(f"{what} must be dense tensors") from None
    types = [t.dtype for t in tensors]
    for t in set(types):
        if t not in L.DTYPE_CODES:
            raise TypeError(f"{what} must be bf16, fp16 or fp32, not {t}")
    on = set(map(torch.Tensor.get_device, tensors))
    if on and (len(on) > 1 or -1 in on or torch.cuda.current_device() not in on):
        L.require_device(*tensors)
    return ptrs, list(map(torch.Tensor.numel, tensors)), types


def _codes(types, codes) -> list:
    return list(map(codes.__getitem__, types))


def _contiguous(tensors: List[torch.Tensor], fresh: bool = False) -> List[torch.Tensor]:
    """the list itself where all are contiguous, else with copies (fresh: uninitialised ones) in the place of those that are not"""
    if all(map(torch.Tensor.is_contiguous, tensors)):
        return tensors
    return [t if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format) if fresh else t.contiguous()
            for t in tensors]


def _overlap(src, dst, n, src_types, dst_types) -> bool:
    """whether a written range [dst, dst + n) meets another written range, or a read range [src, src + n) other than the one that is
    clipped in place (arrays of addresses, elements and type codes)"""
    some = n > 0
    if not some.all():
        src, dst, n, src_types, dst_types = src[some], dst[some], n[some], src_types[some], dst_types[some]
    end = dst + n * _SIZES[dst_types]
    order = np.argsort(dst)
    first, last = dst[order], end[order]
    if (last[:-1] > first[1:]).any():
        return True
    if src is dst or len(src) == 0 or (src == dst).all():
        return False
    # each read range against the written ones around its beginning, which do not overlap one another: the last that begins at or
    # before it and the next one; its own is meant to be there where it is clipped in place
    src_end = src + n * _SIZES[src_types]
    at = np.searchsorted(first, src, side="right")
    before, after = np.maximum(at - 1, 0), np.minimum(at, len(order) - 1)
    mine = (src == dst) & (order[before] == np.arange(len(src)))
    return bool(((at > 0) & (last[before] > src) & ~mine).any() or ((at < len(order)) & (first[after] < src_end)).any())


def grad_norm(grads: Sequence[torch.Tensor], *, norm_type: float = 2.0) -> torch.Tensor:
    """The norm (2, 1 or inf) of all elements of `grads` taken as one vector, as a 0-d fp32 tensor on the device.
    Any mix of bf16, fp16 and fp32, any shapes, empty tensors among them; NaN and infinities go through; the sums are fp64, so
    neither large nor tiny elements leave the range.  Tensors that are not contiguous are read through a copy.  Autograd
    does not follow: the norm has no graph."""
    kind = _norm_kind(norm_type)
    grads = list(grads)
    _no_tangent("grad_norm", *grads)
    ptrs, sizes, types = _pointers(grads, "grad_norm: gradients")
    flat = _contiguous(grads)
    if flat is not grads:
        ptrs = list(map(torch.Tensor.data_ptr, flat))
    return _run_clip(ptrs, ptrs, sizes, _codes(types, L.DTYPE_CODES), None, kind, None)


def _run_clip(src, dst, sizes, src_codes, dst_codes, kind: int, max_norm: Optional[float]) -> torch.Tensor:
    """grad_norm (max_norm None) or clip_grads on lists of addresses"""
    lib = L.load()
    n = len(src)
    types = src_codes if dst_codes is None else list(map(int.__or__, src_codes, dst_codes))
    # the rows of plnlp_grad_tensor: two addresses, a size, two 32-bit type codes
    rows = np.array([src, dst, sizes, types], dtype=np.int64)
    if max_norm is not None and (n > 1 or src is not dst):
        to = rows[3] >> 32
        if _overlap(rows[0], rows[0] if src is dst else rows[1], rows[2], rows[3] & 3, to):
            raise ValueError(_OVERLAP)
    rows = np.ascontiguousarray(rows.T)
    at = rows.ctypes.data
    need = lib.plnlp_grad_norm_workspace_doubles(at, n)
    device = torch.cuda.current_device()
    norm = torch.empty((), dtype=torch.float32, device=device)
    ws = torch.empty(need, dtype=torch.float64, device=device)
    if max_norm is None:
        L.check(lib.plnlp_grad_norm(at, n, kind, ws.data_ptr(), need, norm.data_ptr(), L.stream_ptr()), "plnlp_grad_norm")
    else:
        L.check(lib.plnlp_grad_clip(at, n, kind, max_norm, ws.data_ptr(), need, norm.data_ptr(), L.stream_ptr()), "plnlp_grad_clip")
    return norm


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, *, norm_type: float = 2.0,
               out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales all gradients by min(1, max_norm / (norm + 1e-6)), norm = grad_norm(grads), and returns that norm (a 0-d fp32
    tensor on the device; nothing is read back by the host).

    out: where the scaled gradients go -- one tensor of as many elements for each, of any of the three types: 16-bit gradients
    into the fp32 ones an optimiser of fp32 parameters reads; None: in place.  As torch.nn.utils.clip_grad_norm_ has it, a NaN
    norm makes every gradient NaN and an infinite one makes the finite elements zero.  A tensor listed twice, or one whose
    memory another one's result would overwrite, is refused, and so is a written tensor that is expanded.  Tensors that are not contiguous
    are handled through copies: what such views share with other tensors of the call is scaled once, from its old value."""
    kind = _norm_kind(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grads: max_norm must be 0 or more, not {max_norm}")
    grads = list(grads)
    to = grads if out is None else list(out)
    _no_tangent("clip_grads", *grads, *to)
    src, sizes, types = _pointers(grads, "clip_grads: gradients")
    if out is None:
        dst, to_types = src, types
    else:
        dst, to_sizes, to_types = _pointers(to, "clip_grads: out")
        if to_sizes != sizes:
            raise ValueError("clip_grads: out must hold one tensor of as many elements for each gradient")
    flat = _contiguous(grads)
    flat_to = flat if out is None else _contiguous(to, fresh=True)
    if flat is not grads:
        src = list(map(torch.Tensor.data_ptr, flat))
    if flat_to is not to:
        dst = src if out is None else list(map(torch.Tensor.data_ptr, flat_to))
    if flat_to is not to and len({t.data_ptr() for t in to if t.numel()}) < sum(t.numel() > 0 for t in to):
        raise ValueError(_OVERLAP)                   # (the copies of such tensors do not overlap)
    if flat_to is not to and any(s == 0 and n > 1 for t, c in zip(to, flat_to) if c is not t for s, n in zip(t.stride(), t.shape)):
        raise ValueError("clip_grads: the elements of an expanded tensor share memory and cannot be written")
    norm = _run_clip(src, dst, sizes, _codes(types, L.DTYPE_CODES), _codes(to_types, _DST_CODES), kind, max_norm)
    torch.autograd.graph.increment_version([t for t in to if not t.is_inference()])      # (written behind autograd's back)
    if flat_to is not to:
        with torch.no_grad():
            for t, c in zip(to, flat_to):
                if c is not t:
                    t.copy_(c)
    return norm
