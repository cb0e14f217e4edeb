"""Operators of a training or serving step with 16-bit storage, over the C ABI (csrc/lookup.hip, linear_act.hip,
grad_clip.hip), next to the fp32 operators of plnlp_amd/ops.py:

  embedding_lookup   scale * table[ids], and the table's gradient summed by id
  linear_act         activation(x W^T + bias) + residual, and its gradients
  grad_norm          the norm of a list of gradients taken as one vector
  clip_grads         the gradients scaled so that this norm stays below a limit (in place, or into other tensors)

All sums are held in 32 bits or more and every result is rounded once.  All are deterministic.  Work is enqueued on the current
stream of the current device, on which every tensor has to be; nothing waits for it.  All may be captured into a graph.
Like the rest of the package there is no CPU path."""
from __future__ import annotations

import ctypes as C
import math
from typing import List, Optional, Sequence

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from . import _lib as L

_HALF = (torch.bfloat16, torch.float16)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """a matrix with consecutive elements along its rows and rows that do not overlap: t itself, or a contiguous copy"""
    if t.shape[0] == 0 or t.shape[1] == 0:
        return t
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        return t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    """elements between the rows of a matrix as _rows gives it (a single row: any; then its width)"""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _workspace(n_bytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(n_bytes, dtype=torch.uint8, device=device) if n_bytes > 0 else None


# ------------------------------------------------------------------ lookup ------
def _lookup_rows(table: torch.Tensor, ids: torch.Tensor, scale: float, out_dtype: torch.dtype) -> torch.Tensor:
    table = _rows(table)
    out = torch.empty(*ids.shape, table.shape[1], dtype=out_dtype, device=table.device)
    flat = ids.contiguous()
    L.check(L.load().plnlp_embedding_lookup(table.data_ptr(), _ld(table), L.DTYPE_CODES[table.dtype], table.shape[0], table.shape[1],
                                            flat.data_ptr(), flat.element_size(), flat.numel(), scale, out.data_ptr(),
                                            max(table.shape[1], 1), L.DTYPE_CODES[out_dtype], L.stream_ptr()),
            "plnlp_embedding_lookup")
    return out


def _lookup_grad(gy: torch.Tensor, ids: torch.Tensor, n_rows: int, padding: int, scale: float, dtype: torch.dtype) -> torch.Tensor:
    lib = L.load()
    width = gy.shape[-1]
    gy = _rows(gy.reshape(ids.numel(), width))
    flat = ids.contiguous()
    L.require_device(gy, flat)
    grad = torch.empty(n_rows, width, dtype=dtype, device=gy.device)
    n_bytes = lib.plnlp_embedding_grad_workspace_bytes(flat.numel(), width)
    ws = _workspace(n_bytes, gy.device)
    L.check(lib.plnlp_embedding_grad(gy.data_ptr(), max(_ld(gy), width), L.DTYPE_CODES[gy.dtype], flat.data_ptr(), flat.element_size(),
                                     flat.numel(), padding, scale, grad.data_ptr(), max(width, 1), L.DTYPE_CODES[dtype], n_rows, width,
                                     L.ptr(ws), n_bytes, L.stream_ptr()), "plnlp_embedding_grad")
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
    L.require_device(table, ids)
    if torch.is_grad_enabled() and table.requires_grad:
        return EmbeddingLookupFn.apply(table, ids, float(scale), padding, out_dtype)
    return _lookup_rows(table, ids, float(scale), out_dtype)


# ------------------------------------------------------------------ linear ------
def _linear_forward(x, weight, bias, residual, act: int, keep: bool):
    """(y [m, n], slope or None) of matrices as _rows gives them; the activation's derivative is kept where the backward pass will
    read it: int16 [m, n] in steps of 2^-14"""
    lib = L.load()
    m, k = x.shape
    n = weight.shape[0]
    out = torch.empty(m, n, dtype=x.dtype, device=x.device)
    slope = torch.empty(m, n, dtype=torch.int16, device=x.device) if keep else None
    n_bytes = lib.plnlp_linear_act_workspace_bytes(m, n, k)
    ws = _workspace(n_bytes, x.device)
    L.check(lib.plnlp_linear_act(x.data_ptr(), _ld(x), weight.data_ptr(), _ld(weight), L.ptr(bias), L.ptr(residual),
                                 0 if residual is None else _ld(residual), act, m, n, k, L.ptr(slope), n, out.data_ptr(), n,
                                 L.DTYPE_CODES[x.dtype], L.ptr(ws), n_bytes, L.stream_ptr()), "plnlp_linear_act")
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
            g = _rows(gy)
            L.require_device(g, x, weight)
            n_bytes = lib.plnlp_linear_act_backward_workspace_bytes(m, n, k, ctx.act)
            ws = _workspace(n_bytes, x.device)
            L.check(lib.plnlp_linear_act_backward(g.data_ptr(), _ld(g), L.ptr(slope), n, ctx.act, x.data_ptr(), _ld(x), weight.data_ptr(),
                                                  _ld(weight), m, n, k, L.ptr(dx), k, L.ptr(dw), k, L.ptr(db), L.DTYPE_CODES[x.dtype],
                                                  L.ptr(ws), n_bytes, L.stream_ptr()), "plnlp_linear_act_backward")
        return dx, dw, db, gy if need[3] else None, None


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
               residual: Optional[torch.Tensor] = None, activation: str = "none") -> torch.Tensor:
    """activation(x W^T + bias) + residual.

    x: [..., K]; weight: [N, K] (torch.nn.Linear's layout); bias: [N]; residual: the result's shape [..., N]; all bf16 or all
    fp16.  activation: "none", "relu", "gelu" (z Phi(z)), "gelu_tanh" or "silu".  The product is summed in fp32; bias,
    activation and residual act on the fp32 sums, which are rounded once.  The activation's derivative is kept
    for the backward pass in steps of 2^-14, where a gradient is wanted.
    fp32 matrices are the business of ops.LinearFn."""
    if x.dtype not in _HALF:
        raise TypeError(f"linear_act: x must be bf16 or fp16, not {x.dtype} (ops.LinearFn is the fp32 layer)")
    if activation not in L.ACTIVATIONS:
        raise ValueError(f"linear_act: activation must be one of {', '.join(L.ACTIVATIONS)}, not {activation!r}")
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"linear_act: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match ([..., K] and [N, K])")
    n = weight.shape[0]
    shape = (*x.shape[:-1], n)
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"linear_act: bias must have shape ({n},), not {tuple(bias.shape)}")
    if residual is not None and tuple(residual.shape) != shape:
        raise ValueError(f"linear_act: residual must have the result's shape {shape}, not {tuple(residual.shape)}")
    for t in (weight, bias, residual):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"linear_act: all operands must have x's type {x.dtype}, not {t.dtype}")
    L.require_device(x, weight, bias, residual)
    rows = math.prod(x.shape[:-1])
    x2 = _rows(x.reshape(rows, x.shape[-1]))
    w2 = _rows(weight)
    b2 = bias if bias is None or bias.stride(0) == 1 or n <= 1 else bias.contiguous()
    r2 = None if residual is None else _rows(residual.reshape(rows, n))
    act = L.ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x2, w2, b2, r2)):
        y = LinearActFn.apply(x2, w2, b2, r2, act)
    else:
        y = _linear_forward(x2, w2, b2, r2, act, False)[0]
    return y.view(shape)


# ------------------------------------------------------------------ clipping ----
_GRAD_ROW = np.dtype([("src", np.uint64), ("dst", np.uint64), ("n", np.int64), ("src_dtype", np.int32), ("dst_dtype", np.int32)])
assert _GRAD_ROW.itemsize == C.sizeof(L.GradTensor)


def _norm_kind(norm_type) -> int:
    p = float(norm_type)
    if p == 2.0:
        return L.NORM_L2
    if p == 1.0:
        return L.NORM_L1
    if p == math.inf:
        return L.NORM_MAX
    raise ValueError(f"norm_type must be 1, 2 or inf, not {norm_type!r}")


def _check_list(tensors: Sequence[torch.Tensor], what: str) -> None:
    device = torch.cuda.current_device() if tensors and torch.cuda.is_available() else -1
    for t in tensors:
        if t.dtype not in L.DTYPE_CODES or t.layout is not torch.strided:
            raise TypeError(f"{what} must be dense bf16, fp16 or fp32 tensors, not {t.dtype}, {t.layout}")
        if t.get_device() != device or device < 0:
            L.require_device(t)


def _table(src: Sequence[torch.Tensor], dst: Optional[Sequence[torch.Tensor]]):
    rows = np.zeros(len(src), dtype=_GRAD_ROW)
    codes = L.DTYPE_CODES
    rows["src"] = [t.data_ptr() for t in src]
    rows["n"] = [t.numel() for t in src]
    rows["src_dtype"] = [codes[t.dtype] for t in src]
    if dst is not None:
        rows["dst"] = [t.data_ptr() for t in dst] if dst is not src else rows["src"]
        rows["dst_dtype"] = [codes[t.dtype] for t in dst] if dst is not src else rows["src_dtype"]
    return rows


def _refuse_overlaps(rows) -> None:
    """a written range that another entry reads or writes would be scaled twice, or read half scaled"""
    rows = rows[rows["n"] > 0]
    size = np.array([4, 2, 2])
    s0 = rows["src"].astype(np.int64)
    s1 = s0 + rows["n"] * size[rows["src_dtype"]]
    d0 = rows["dst"].astype(np.int64)
    d1 = d0 + rows["n"] * size[rows["dst_dtype"]]
    order = np.argsort(d0, kind="stable")
    bad = bool((d1[order][:-1] > d0[order][1:]).any())
    if not bad:
        same = s0 == d0
        # each source against the written ranges around its beginning (they do not overlap one another): the last that begins at or
        # before it and the next one; its own is meant to be there where it is clipped in place
        at = np.searchsorted(d0[order], s0, side="right")
        before, after = np.maximum(at - 1, 0), np.minimum(at, len(order) - 1)
        own = np.arange(len(rows))
        hit = (at > 0) & (d1[order][before] > s0) & ~(same & (order[before] == own))
        hit |= (at < len(order)) & (d0[order][after] < s1)
        bad = bool(hit.any())
    if bad:
        raise ValueError("clip_grads: the memory of a clipped tensor overlaps another tensor of the call (a gradient listed twice?)")


def grad_norm(grads: Sequence[torch.Tensor], *, norm_type: float = 2.0) -> torch.Tensor:
    """The norm (2, 1 or inf) of all elements of `grads` taken as one vector, as a 0-d fp32 tensor on the device.
    Any mix of bf16, fp16 and fp32, any shapes, empty tensors among them; NaN and infinities go through; the sums are fp64, so
    neither large nor tiny elements leave the range.  Tensors that are not contiguous are read through a copy."""
    kind = _norm_kind(norm_type)
    grads = list(grads)
    _check_list(grads, "grad_norm: gradients")
    return _norm(grads, kind)


def _norm(grads, kind: int) -> torch.Tensor:
    lib = L.load()
    grads = [t if t.is_contiguous() else t.contiguous() for t in grads]
    norm = torch.empty((), dtype=torch.float32, device="cuda")
    rows = _table(grads, None)
    arr = rows.ctypes.data_as(C.POINTER(L.GradTensor))
    need = lib.plnlp_grad_norm_workspace_doubles(arr, len(grads))
    ws = torch.empty(need, dtype=torch.float64, device="cuda")
    L.check(lib.plnlp_grad_norm(arr, len(grads), kind, ws.data_ptr(), need, norm.data_ptr(), L.stream_ptr()), "plnlp_grad_norm")
    return norm


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, *, norm_type: float = 2.0,
               out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales all gradients by min(1, max_norm / (norm + 1e-6)), norm = grad_norm(grads), and returns that norm (a 0-d fp32
    tensor on the device; nothing is read back by the host).

    out: where the scaled gradients go -- tensors of the same shapes, of any of the three types: 16-bit gradients into the fp32
    ones an optimiser of fp32 parameters reads; None: in place.  As torch.nn.utils.clip_grad_norm_ has it, a NaN norm makes
    every gradient NaN and an infinite one makes the finite elements zero.  A tensor listed twice, or one whose memory another
    one's result would overwrite, is refused.  Tensors that are not contiguous are handled through copies."""
    kind = _norm_kind(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grads: max_norm must be 0 or more, not {max_norm}")
    grads = list(grads)
    _check_list(grads, "clip_grads: gradients")
    lib = L.load()
    src = [t if t.is_contiguous() else t.contiguous() for t in grads]
    back = []
    if out is None:
        dst = src
        back = [(t, c) for t, c in zip(grads, src) if c is not t]
    else:
        out = list(out)
        _check_list(out, "clip_grads: out")
        if len(out) != len(grads) or any(o.shape != g.shape for o, g in zip(out, grads)):
            raise ValueError("clip_grads: out must hold one tensor of the same shape for each gradient")
        dst = [t if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format) for t in out]
        back = [(t, c) for t, c in zip(out, dst) if c is not t]
    rows = _table(src, dst)
    if len(rows) > 1 or out is not None:
        _refuse_overlaps(rows)
    arr = rows.ctypes.data_as(C.POINTER(L.GradTensor))
    need = lib.plnlp_grad_norm_workspace_doubles(arr, len(src))
    norm = torch.empty((), dtype=torch.float32, device="cuda")
    ws = torch.empty(need, dtype=torch.float64, device="cuda")
    L.check(lib.plnlp_grad_clip(arr, len(src), kind, max_norm, ws.data_ptr(), need, norm.data_ptr(), L.stream_ptr()), "plnlp_grad_clip")
    for t, c in back:
        t.copy_(c)
    return norm
