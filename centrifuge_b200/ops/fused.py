"""Python entry points of the fused sm_100a kernels.

Every function takes preallocated outputs where the training step reuses buffers.  CUDA tensors
go to the compiled kernels (``centrifuge_b200._kernels``); CPU tensors run the fp32 definitions
in :mod:`centrifuge_b200.ops.reference`.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence

import torch

from . import reference as ref
from ._ext import kernels


# ---------------------------------------------------------------- RMSNorm
def rmsnorm_fwd(x: torch.Tensor, w: torch.Tensor, eps: float, out: Optional[torch.Tensor] = None,
                rstd: Optional[torch.Tensor] = None):
    if out is None:
        out = torch.empty_like(x)
    if rstd is None:
        rstd = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    if not x.is_cuda:
        y, r = ref.rmsnorm(x, w, eps)
        out.copy_(y)
        rstd.copy_(r)
        return out, rstd
    kernels().rmsnorm_fwd(x, w, out, rstd, eps)
    return out, rstd


def rmsnorm_bwd(dy: torch.Tensor, x: torch.Tensor, rstd: torch.Tensor, w: torch.Tensor,
                dw_acc: torch.Tensor, x_rows: Optional[torch.Tensor] = None,
                dres: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    """``dx = dres + d(rmsnorm)/dx`` on the rows ``x[x_rows]``; ``dw_acc += dgamma`` (fp32)."""
    if out is None:
        out = torch.empty_like(dy)
    if not dy.is_cuda:
        xs = x if x_rows is None else x[x_rows.long()]
        rs = rstd if x_rows is None else rstd[x_rows.long()]
        dx, dw = ref.rmsnorm_bwd(dy, xs, rs, w, dres)
        out.copy_(dx)
        dw_acc += dw
        return out
    partial_rows = max(1, min(dy.shape[0], 148 * 2))
    kernels().rmsnorm_bwd(dy, x, x_rows, rstd, w, dres, out, dw_acc, partial_rows)
    return out


# ---------------------------------------------------------------- RoPE
def rope_(qkv: torch.Tensor, pos: torch.Tensor, n_heads: int, head_dim: int,
          table: torch.Tensor, inverse: bool = False) -> torch.Tensor:
    """In-place RoPE on heads ``[0, n_heads)`` of each ``qkv`` row at positions ``pos``."""
    if not qkv.is_cuda:
        rows = qkv.shape[0]
        view = qkv[:, : n_heads * head_dim].view(rows, n_heads, head_dim)
        view.copy_(ref.rope(view, pos, table, inverse))
        return qkv
    kernels().rope(qkv, pos, n_heads, head_dim, table, inverse)
    return qkv


# ---------------------------------------------------------------- SwiGLU
def swiglu_fwd(gu: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    F = gu.shape[1] // 2
    if out is None:
        out = torch.empty(gu.shape[0], F, dtype=gu.dtype, device=gu.device)
    if not gu.is_cuda:
        out.copy_(ref.swiglu(gu))
        return out
    kernels().swiglu_fwd(gu, out)
    return out


def swiglu_bwd(dh: torch.Tensor, gu: torch.Tensor, gu_rows: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None,
               h_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``d[gate; up]`` from ``dh`` and the saved ``gu`` rows ``gu_rows``.  With ``h_out``
    (``[rows, F]``) the same pass also writes ``h = silu(gate) * up`` of those rows, i.e. the
    forward activation of the kept rows, recomputed instead of gathered."""
    if out is None:
        out = torch.empty(dh.shape[0], 2 * dh.shape[1], dtype=dh.dtype, device=dh.device)
    if not dh.is_cuda:
        g = gu if gu_rows is None else gu[gu_rows.long()]
        out.copy_(ref.swiglu_bwd(dh, g))
        if h_out is not None:
            h_out.copy_(ref.swiglu(g.float()))
        return out
    kernels().swiglu_bwd(dh, gu, gu_rows, out, h_out)
    return out


# ---------------------------------------------------------------- gathers / embedding
def gather_rows(src: torch.Tensor, idx: torch.Tensor, out: Optional[torch.Tensor] = None):
    if out is None:
        out = torch.empty(idx.numel(), src.shape[1], dtype=src.dtype, device=src.device)
    if not src.is_cuda:
        out.copy_(src[idx.long()])
        return out
    kernels().gather_rows(src, idx, out)
    return out


def embedding_fwd(table: torch.Tensor, ids: torch.Tensor, out: Optional[torch.Tensor] = None):
    ids = ids.reshape(-1)
    if out is None:
        out = torch.empty(ids.numel(), table.shape[1], dtype=table.dtype, device=table.device)
    if not table.is_cuda:
        out.copy_(table[ids])
        return out
    kernels().embedding_fwd(table, ids.contiguous(), out)
    return out


def embedding_bwd(dy: torch.Tensor, ids: torch.Tensor, dtable: torch.Tensor,
                  id_rows: Optional[torch.Tensor] = None, deterministic: bool = True):
    """``dtable[ids[id_rows[r]]] += dy[r]``.  ``deterministic``: rows are sorted by token and
    each token's rows are summed in row order by one warp (same bits on every run); otherwise
    fp32 atomics, whose summation order varies from run to run."""
    ids = ids.reshape(-1)
    if not dy.is_cuda:
        sel = ids if id_rows is None else ids[id_rows.long()]
        dtable.index_add_(0, sel, dy.float())
        return dtable
    kernels().embedding_bwd(dy, ids.contiguous(), id_rows, dtable, deterministic)
    return dtable


_EMBED_MAX_H = 65535 * 128
_ROW_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _need(ok: bool, what: str, *args) -> None:
    if not ok:
        raise ValueError(what.format(*args))


def _rows2d(t: torch.Tensor, H: int) -> bool:
    """``t`` is ``[*, H]`` with columns next to each other and rows that do not overlap."""
    return t.dim() == 2 and t.shape[1] == H and (t.stride(1) == 1 or H <= 1) and (
        t.stride(0) >= H or t.shape[0] <= 1)


def _vector(t: torch.Tensor, H: int, dtype: torch.dtype) -> bool:
    return t.dim() == 1 and t.shape[0] == H and t.dtype == dtype and t.is_contiguous()


def _need_index(index: torch.Tensor, n: int, what: str) -> None:
    """CPU: an index outside ``[0, n)`` is an error (a negative one would count from the end)."""
    if index.numel() and not 0 <= int(index.min()) <= int(index.max()) < n:
        raise IndexError(f"{what} outside [0, {n})")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors, contiguous or row-major ``[rows, width]``, share bytes."""
    def layout(t):
        rows = t.dim() == 2 and t.shape[0] > 1 and not t.is_contiguous()
        step = t.stride(0) * t.element_size() if rows else 0
        width = (t.shape[1] if rows else t.numel()) * t.element_size()
        return t.data_ptr(), t.data_ptr() + (t.shape[0] - 1 if rows else 0) * step + width, step, width

    (lo, hi, step, width), (lo2, hi2, step2, width2) = layout(a), layout(b)
    if lo >= hi or lo2 >= hi2 or lo >= hi2 or lo2 >= hi:
        return False
    s = max(step, step2)  # both may be columns of one buffer's rows
    if s == 0 or step not in (0, s) or step2 not in (0, s):
        return True
    return (lo2 - lo) % s < width or (lo2 - lo) % s + width2 > s


def scaled_embedding_fwd(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[r] = scale * table[ids[r]]``, rounded once.

    ``table [V, H]`` and ``out [ids.numel(), H]`` are bf16, fp16 or fp32 (``out`` may have another
    type than the table, e.g. an fp32 residual stream) with unit column stride and any row stride,
    apart from each other, ``H`` up to 8388480; ``ids`` int64 or int32, any shape.  On the GPU an id
    outside the vocabulary records an error in the status block and gives a zero row; on the CPU it
    raises ``IndexError``."""
    if table.is_cuda:
        return kernels().scaled_embedding_fwd(table, ids, scale, out)
    _need(table.dim() == 2 and _rows2d(table, table.shape[1]) and table.dtype in _ROW_TYPES,
          "scaled_embedding_fwd: table must be a row-major bf16, fp16 or fp32 [V, H]")
    _need(table.shape[1] <= _EMBED_MAX_H, "scaled_embedding_fwd: hidden size {} is over {}",
          table.shape[1], _EMBED_MAX_H)
    _need(ids.dtype in (torch.int64, torch.int32), "scaled_embedding_fwd: ids must be int64 or int32")
    ids = ids.reshape(-1)
    H = table.shape[1]
    if out is None:
        out = torch.empty(ids.shape[0], H, dtype=table.dtype, device=table.device)
    else:
        _need(_rows2d(out, H) and out.shape[0] == ids.shape[0] and out.dtype in _ROW_TYPES,
              "scaled_embedding_fwd: out must be a row-major bf16, fp16 or fp32 [{}, {}]",
              ids.shape[0], H)
        _need(not _overlap(out, table) and not _overlap(out, ids),
              "scaled_embedding_fwd: out overlaps the table or the ids")
    _need_index(ids, table.shape[0], "scaled_embedding_fwd: an id is")
    return out.copy_(table[ids.long()].float() * scale)


def scaled_embedding_bwd(dy: torch.Tensor, ids: torch.Tensor, dtable: torch.Tensor,
                         scale: float = 1.0, id_rows: Optional[torch.Tensor] = None,
                         padding_idx: Optional[int] = None,
                         accumulate: bool = True) -> torch.Tensor:
    """``dtable[v] (+)= scale * sum of dy[r] over the rows r of token v``, in fp32 and in one fixed
    order (same bits on every run).

    Row ``r`` has token ``ids[id_rows[r]]`` (``ids[r]`` without ``id_rows``).  ``dy [R, H]`` is
    bf16, fp16 or fp32 and ``dtable [V, H]`` fp32, both with unit column stride and any row stride,
    apart from each other, ``H`` up to 8388480.  Rows of token ``padding_idx`` (below 2^31) add
    nothing.  Without ``accumulate`` the gradient replaces what ``dtable`` held: rows of tokens that
    do not occur become zero.  Where it is added, the GPU takes subnormal numbers (below 1.2e-38) as
    zeros.  On the GPU a token outside the table or a row id outside ``ids`` records an error in the
    status block and adds nothing; on the CPU it raises ``IndexError`` and ``dtable`` stays as it
    was."""
    if dy.is_cuda:
        kernels().scaled_embedding_bwd(dy, ids, dtable, scale, id_rows, padding_idx, accumulate)
        return dtable
    _need(dy.dim() == 2 and _rows2d(dy, dy.shape[1]) and dy.dtype in _ROW_TYPES,
          "scaled_embedding_bwd: dy must be a row-major bf16, fp16 or fp32 [R, H]")
    _need(ids.dtype in (torch.int64, torch.int32), "scaled_embedding_bwd: ids must be int64 or int32")
    _need(_rows2d(dtable, dy.shape[1]) and dtable.dtype == torch.float32,
          "scaled_embedding_bwd: dtable must be a row-major fp32 [V, {}]", dy.shape[1])
    _need(dtable.shape[0] > 0 or dy.shape[0] == 0, "scaled_embedding_bwd: a table of 0 rows")
    _need(dy.shape[1] <= _EMBED_MAX_H, "scaled_embedding_bwd: hidden size {} is over {}",
          dy.shape[1], _EMBED_MAX_H)
    _need(padding_idx is None or 0 <= padding_idx < 1 << 31,
          "scaled_embedding_bwd: padding_idx is negative or over 31 bits")
    ids = ids.reshape(-1)
    if id_rows is None:
        _need(ids.shape[0] == dy.shape[0], "scaled_embedding_bwd: {} ids for {} rows",
              ids.shape[0], dy.shape[0])
    else:
        _need(id_rows.dtype == torch.int32 and id_rows.dim() == 1 and id_rows.is_contiguous()
              and id_rows.shape[0] == dy.shape[0],
              "scaled_embedding_bwd: id_rows must be contiguous int32 [{}]", dy.shape[0])
    _need(not any(_overlap(dtable, t) for t in (dy, ids, id_rows) if t is not None),
          "scaled_embedding_bwd: dtable overlaps dy, the ids or id_rows")
    if id_rows is not None:
        _need_index(id_rows, ids.shape[0], "scaled_embedding_bwd: a row id is")
    tok = (ids if id_rows is None else ids[id_rows.long()]).long()
    g = dy.float() * scale
    if padding_idx is not None:
        g, tok = g[tok != padding_idx], tok[tok != padding_idx]
    _need_index(tok, dtable.shape[0], "scaled_embedding_bwd: a token is")
    if not accumulate:
        dtable.zero_()
    return dtable.index_add_(0, tok, g)


# ---------------------------------------------------------------- norms around a block
def _check_gate(name: str, gate: torch.Tensor, T: int, H: int, dtype: torch.dtype) -> None:
    if gate.dim() == 1:
        _need(_vector(gate, H, dtype), "{}: a channel's gate must be contiguous {} [{}]", name,
              dtype, H)
    elif gate.dim() == 2 and gate.shape[1] == 1 and gate.dtype == torch.float32:
        _need(gate.shape[0] == T, "{}: a token's gate must be fp32 [{}, 1]", name, T)
    else:
        _need(_rows2d(gate, H) and gate.shape[0] == T and gate.dtype == dtype,
              "{}: the gate must be [{}], fp32 [{}, 1] or {} [{}, {}]", name, H, T, dtype, T, H)


def block_norms_fwd(h: torch.Tensor, x: torch.Tensor, w_post: torch.Tensor,
                    w_pre: Optional[torch.Tensor], eps: float,
                    gate: Optional[torch.Tensor] = None, block_scale: float = 1.0,
                    resid_scale: float = 1.0):
    """The norm after a block, its gate, the residual sum and the norm before the next block::

        y = resid_scale * x + block_scale * gate * rmsnorm(h, w_post)
        n = rmsnorm(y, w_pre)

    in one pass (``n`` from the unrounded ``y``).  Returns ``(y, n, rstd_post, rstd_pre)``; without
    ``w_pre`` (the last block of a pipeline stage) ``n`` and ``rstd_pre`` are ``None``.

    ``h [T, H]`` (a block's output), ``n`` and the weights are bf16, fp16 or fp32; the residual
    stream ``x``, ``y`` has that type or fp32.  ``gate``: ``None``, a learned ``[H]``, a weight for
    each token (fp32 ``[T, 1]``), or ``[T, H]``.  ``h``, ``x`` and ``gate`` may have any row stride.
    ``H`` up to 16384."""
    if h.is_cuda:
        return kernels().block_norms_fwd(h, x, w_post, w_pre, eps, gate, block_scale, resid_scale)
    T, H = h.shape if h.dim() == 2 else (-1, -1)
    _need(T >= 0 and _rows2d(h, H) and h.dtype in _ROW_TYPES,
          "block_norms_fwd: h must be a row-major bf16, fp16 or fp32 [T, H]")
    _need(_rows2d(x, H) and x.shape[0] == T and x.dtype in (h.dtype, torch.float32),
          "block_norms_fwd: x must be a row-major {} or fp32 [{}, {}]", h.dtype, T, H)
    _need(_vector(w_post, H, h.dtype) and (w_pre is None or _vector(w_pre, H, h.dtype)),
          "block_norms_fwd: the weights must be contiguous {} [{}]", h.dtype, H)
    _need(H <= 16384, "block_norms_fwd: hidden size {} is over 16384", H)
    if gate is not None:
        _check_gate("block_norms_fwd", gate, T, H, h.dtype)
    y, n, rp, rq = ref.block_norms(h, x, w_post, w_pre, eps, gate, block_scale, resid_scale)
    return y.to(x.dtype), None if n is None else n.to(h.dtype), rp, rq


def block_norms_bwd(dy: Optional[torch.Tensor], dn: Optional[torch.Tensor], h: torch.Tensor,
                    y: Optional[torch.Tensor], rstd_post: torch.Tensor,
                    rstd_pre: Optional[torch.Tensor], w_post: torch.Tensor,
                    w_pre: Optional[torch.Tensor], dw_post: torch.Tensor,
                    dw_pre: Optional[torch.Tensor], gate: Optional[torch.Tensor] = None,
                    dgate: Optional[torch.Tensor] = None, block_scale: float = 1.0,
                    resid_scale: float = 1.0, rows: Optional[torch.Tensor] = None,
                    accumulate: bool = True):
    """Gradient of :func:`block_norms_fwd` on the rows ``rows`` of ``h``, ``y`` and the saved
    statistics (all when ``None``): ``(dx, dh, dgate)``.

    ``dy [R, H]`` is the gradient that reaches ``y`` past the next block (``None``: none does) and
    ``dn [R, H]`` that of ``n``; without ``w_pre``, ``dn``, ``y``, ``rstd_pre`` and ``dw_pre`` are
    ``None``.  ``dw_post``, ``dw_pre`` and, for a learned gate, ``dgate`` are fp32 ``[H]`` buffers,
    added to (written without ``accumulate``); a buffer given for two of them (one parameter in both
    places) gets the sum of both gradients, other overlaps are refused.  A token's or element's gate
    returns its gradient for the ``R`` rows.  On the GPU a row id outside ``h`` records an error in
    the status block and gives zero rows; on the CPU it raises ``IndexError``."""
    if h.is_cuda:
        return kernels().block_norms_bwd(dy, dn, h, y, rstd_post, rstd_pre, w_post, w_pre, dw_post,
                                         dw_pre, gate, dgate, block_scale, resid_scale, rows,
                                         accumulate)
    name = "block_norms_bwd"
    T, H = h.shape if h.dim() == 2 else (-1, -1)
    _need(T >= 0 and _rows2d(h, H) and h.dtype in _ROW_TYPES,
          "{}: h must be a row-major bf16, fp16 or fp32 [T, H]", name)
    pre = w_pre is not None
    _need((dn is not None) == pre and (y is not None) == pre and (rstd_pre is not None) == pre
          and (dw_pre is not None) == pre and (pre or dy is not None),
          "{}: dn, y, rstd_pre and dw_pre go with w_pre, and one of dy and dn is needed", name)
    R = (dy if dn is None else dn).shape[0]
    resid = (y if pre else dy).dtype
    _need(resid in (h.dtype, torch.float32), "{}: y and dy must be {} or fp32", name, h.dtype)
    if dy is not None:
        _need(_rows2d(dy, H) and dy.shape[0] == R and dy.dtype == resid,
              "{}: dy must be a row-major {} [{}, {}]", name, resid, R, H)
    if pre:
        _need(_rows2d(dn, H) and dn.dtype == h.dtype and _rows2d(y, H) and y.shape[0] == T,
              "{}: dn must be a row-major {} [R, {}] and y a row-major [{}, {}]", name, h.dtype, H,
              T, H)
        _need(_vector(rstd_pre, T, torch.float32) and _vector(w_pre, H, h.dtype)
              and _vector(dw_pre, H, torch.float32),
              "{}: rstd_pre must be fp32 [{}], w_pre {} [{}], dw_pre fp32 [{}]", name, T, h.dtype,
              H, H)
    _need(_vector(rstd_post, T, torch.float32) and _vector(w_post, H, h.dtype)
          and _vector(dw_post, H, torch.float32),
          "{}: rstd_post must be fp32 [{}], w_post {} [{}], dw_post fp32 [{}]", name, T, h.dtype, H,
          H)
    _need(H <= 16384, "{}: hidden size {} is over 16384", name, H)
    if rows is None:
        _need(R == T, "{}: {} gradient rows for {} rows", name, R, T)
    else:
        _need(rows.dtype == torch.int32 and rows.dim() == 1 and rows.shape[0] == R
              and rows.is_contiguous(), "{}: rows must be contiguous int32 [{}]", name, R)
    if gate is not None:
        _check_gate(name, gate, T, H, h.dtype)
    learned = gate is not None and gate.dim() == 1
    _need((dgate is not None) == learned and (not learned or _vector(dgate, H, torch.float32)),
          "{}: dgate is the fp32 [{}] buffer of a learned gate", name, H)
    sums = [t for t in (dw_post, dw_pre, dgate) if t is not None]
    params = [t for t in (w_post, w_pre, gate if learned else None) if t is not None]
    for i, s in enumerate(sums):
        _need(all(s.data_ptr() == t.data_ptr() or not _overlap(s, t) for t in sums[:i]),
              "{}: dw_post, dw_pre and dgate overlap in part", name)
        _need(not any(_overlap(s, t) for t in params),
              "{}: dw_post, dw_pre or dgate overlaps a weight or the gate", name)
    if rows is not None:
        _need_index(rows, T, f"{name}: a row id is")
        at = rows.long()
        h, rstd_post = h[at], rstd_post[at]
        y, rstd_pre = (y[at], rstd_pre[at]) if pre else (None, None)
        gate = gate if gate is None or learned else gate[at]
    dx, dh, dp, dq, dg = ref.block_norms_bwd(dy, dn, h, y, rstd_post, rstd_pre, w_post, w_pre,
                                             gate, block_scale, resid_scale)
    written = set()
    for acc, d in ((dw_pre, dq), (dw_post, dp), (dgate, dg if learned else None)):
        if acc is not None:
            acc.copy_(acc + d if accumulate or acc.data_ptr() in written else d)
            written.add(acc.data_ptr())
    return (dx.to(resid), dh.to(h.dtype),
            dgate if gate is None or learned else dg.to(gate.dtype))


# ---------------------------------------------------------------- layer norm
def _check_apart(name: str, what: str, out: torch.Tensor, inputs,
                 in_place: Optional[torch.Tensor] = None) -> None:
    for t in inputs:
        same = t is not None and t is in_place and t.data_ptr() == out.data_ptr() and (
            t.stride() == out.stride())
        _need(t is None or same or not _overlap(out, t), "{}: {} overlaps another tensor of the call",
              name, what)


def layernorm_fwd(x: torch.Tensor, w: Optional[torch.Tensor], b: Optional[torch.Tensor], eps: float,
                  out: Optional[torch.Tensor] = None):
    """``y = (x - mean) rstd w + b`` with ``rstd = (mean of (x - mean)^2 + eps)^-1/2`` of each row:
    ``(y, mean, rstd)``, the last two fp32 ``[T]``.

    ``w`` and ``b`` (contiguous ``[H]``; without one it is one, or zero) and ``y`` are bf16, fp16 or
    fp32, and ``x [T, H]`` has their type or is an fp32 residual stream (without both, ``y`` has the
    type of ``out``, or of ``x``).  ``x`` and ``out`` may have any row stride and alignment, and do
    not overlap.  ``H`` up to 16384."""
    if x.is_cuda:
        return kernels().layernorm_fwd(x, w, b, eps, out)
    name = "layernorm_fwd"
    T, H = x.shape if x.dim() == 2 else (-1, -1)
    _need(T >= 0 and _rows2d(x, H), "{}: x must be row-major [T, H]", name)
    _need(H <= 16384, "{}: hidden size {} is over 16384", name, H)
    dtype = next(t for t in (w, b, out, x) if t is not None).dtype
    _need(dtype in _ROW_TYPES and x.dtype in (dtype, torch.float32), "{}: x must be {} or fp32", name,
          dtype)
    _need(all(t is None or _vector(t, H, dtype) for t in (w, b)),
          "{}: w and b must be contiguous {} [{}]", name, dtype, H)
    if out is not None:
        _need(_rows2d(out, H) and out.shape[0] == T and out.dtype == dtype,
              "{}: out must be row-major {} [{}, {}]", name, dtype, T, H)
        _check_apart(name, "out", out, (x, w, b))
    y, mean, rstd = ref.layernorm(x, w, b, eps)
    return y.to(dtype) if out is None else out.copy_(y), mean, rstd


def layernorm_bwd(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                  w: Optional[torch.Tensor], dw: Optional[torch.Tensor],
                  db: Optional[torch.Tensor], rows: Optional[torch.Tensor] = None,
                  dres: Optional[torch.Tensor] = None, accumulate: bool = True) -> torch.Tensor:
    """``dx = dres + d(layernorm)/dx`` on the rows ``rows`` of ``x`` and the saved statistics (int32
    ``[R]``; all when ``None``).

    ``dy [R, H]`` and ``w`` are bf16, fp16 or fp32; ``x``, ``dres [R, H]`` (the gradient that reaches
    ``x`` past the norm, or ``None``) and ``dx`` have that type or fp32.  ``dw`` and ``db`` are fp32
    ``[H]`` buffers (``None``: not wanted), added to (written without ``accumulate``) in a fixed
    order; what is written overlaps nothing else.  On the GPU a row id outside ``x`` records an error
    in the status block, gives a zero row and adds nothing; on the CPU it raises ``IndexError``."""
    if dy.is_cuda:
        return kernels().layernorm_bwd(dy, x, mean, rstd, w, dw, db, rows, dres, accumulate)
    name = "layernorm_bwd"
    T, H = x.shape if x.dim() == 2 else (-1, -1)
    _need(T >= 0 and _rows2d(x, H) and _rows2d(dy, H),
          "{}: dy must be row-major [R, H] and x [T, H]", name)
    R = dy.shape[0]
    _need(H <= 16384, "{}: hidden size {} is over 16384", name, H)
    _need(dy.dtype in _ROW_TYPES and x.dtype in (dy.dtype, torch.float32),
          "{}: x must be {} or fp32", name, dy.dtype)
    _need(_vector(mean, T, torch.float32) and _vector(rstd, T, torch.float32),
          "{}: mean and rstd must be contiguous fp32 [{}]", name, T)
    _need(w is None or _vector(w, H, dy.dtype), "{}: w must be contiguous {} [{}]", name, dy.dtype, H)
    _need(dres is None or _rows2d(dres, H) and dres.shape[0] == R and dres.dtype == x.dtype,
          "{}: dres must be row-major {} [{}, {}]", name, x.dtype, R, H)
    if rows is None:
        _need(R == T, "{}: {} gradient rows for {} rows", name, R, T)
    else:
        _need(rows.dtype == torch.int32 and rows.dim() == 1 and rows.shape[0] == R
              and rows.is_contiguous(), "{}: rows must be contiguous int32 [{}]", name, R)
    for what, t, other in (("dw", dw, None), ("db", db, dw)):
        if t is not None:
            _need(_vector(t, H, torch.float32), "{}: {} must be contiguous fp32 [{}]", name, what, H)
            _check_apart(name, what, t, (dy, x, mean, rstd, w, rows, dres, other))
    if rows is not None:
        _need_index(rows, T, f"{name}: a row id is")
        x, mean, rstd = x[rows.long()], mean[rows.long()], rstd[rows.long()]
    dx, gw, gb = ref.layernorm_bwd(dy, x, mean, rstd, w, dres)
    for t, g in ((dw, gw), (db, gb)):
        if t is not None:
            t.copy_(t + g if accumulate else g)
    return dx.to(x.dtype)


# ---------------------------------------------------------------- distillation
def _check_distill(name: str, logits, top_ids, top_logits, temperature: float, labels) -> None:
    T, V = logits.shape if logits.dim() == 2 else (-1, -1)
    _need(T >= 0 and _rows2d(logits, V) and logits.dtype in _ROW_TYPES,
          "{}: logits must be row-major bf16, fp16 or fp32 [T, V]", name)
    _need(0 < V <= 1 << 20, "{}: {} logits a row, not 1 to {}", name, V, 1 << 20)
    K = top_ids.shape[1] if top_ids.dim() == 2 else -1
    _need(0 < K <= 1024, "{}: {} listed logits a row, not 1 to 1024", name, K)
    _need(top_ids.dtype in (torch.int64, torch.int32) and _rows2d(top_ids, K)
          and top_ids.shape[0] == T, "{}: top_ids must be int64 or int32 [{}, K]", name, T)
    _need(top_logits.dtype in _ROW_TYPES and _rows2d(top_logits, K) and top_logits.shape[0] == T,
          "{}: top_logits must be bf16, fp16 or fp32 [{}, {}]", name, T, K)
    _need(2.0 ** -100 <= temperature <= 2.0 ** 100, "{}: temperature = {} is not from 2^-100 to 2^100",
          name, temperature)
    _need(labels is None or _vector(labels, T, torch.int64), "{}: labels must be int64 [{}]", name, T)


def distill_fwd(logits: torch.Tensor, top_ids: torch.Tensor, top_logits: torch.Tensor,
                temperature: float = 1.0, top_lse: Optional[torch.Tensor] = None,
                labels: Optional[torch.Tensor] = None):
    """Per-token divergence of a student from a teacher of whom the top logits are known, and the
    labels' cross entropy, in one pass over the student's logits: ``(kd, ce, lse, stats)``.

    ``logits [T, V]`` are the student's; the teacher's ``top_logits [T, K]`` belong to the tokens
    ``top_ids [T, K]`` (int64 or int32; a negative id leaves an entry out, so lists may be of any
    length, and a token named twice has the sum of its shares).  With ``q = softmax(logits / tau)``,
    ``tau = temperature``:

    * without ``top_lse`` the teacher's shares are ``p = softmax(top_logits / tau)`` over the list and
      ``kd = sum p (log p - log q)``; an empty list, or one of ``-inf`` alone, gives 0.
    * ``top_lse [T]`` (fp32) is ``log sum exp`` of *all* the teacher's logits ``/ tau``; then
      ``p = exp(top_logits / tau - top_lse)``, and what is left of 1 is compared with the student's
      share of all tokens outside the list (where the student gives them any: one whose logarithm is
      2^23 or more below the list's, as of masked logits, counts as none).

    ``kd`` is not scaled by ``tau^2``.  With ``labels`` (int64 ``[T]``; negative: ignored, 0), ``ce``
    and ``lse`` are those of :func:`ce_fwd`, without them ``None``.  ``stats`` (fp32 ``[T, 4]``:
    ``log sum exp(logits / tau)``, the same of the tokens outside the list, their share less the
    teacher's (times what makes up for the rounding of a large value before it), and the teacher's
    normaliser) is what :func:`distill_bwd` needs.

    ``tau`` is from ``2^-100`` to ``2^100``, and no logit (for kd: over ``tau``) is above ``2^29``.  A row
    whose logits are all near 1e4 in size loses the last fp32 digits of its statistics: 5e-4 of the shares
    of listed tokens and labels in the gradient.

    Logits may be masked by ``-inf`` or by their type's lowest value: a finite logit (for kd: over
    ``tau``) below ``-2^30 log 2`` counts as being there, so that a row of such masks alone is a uniform
    distribution.

    Logits and ``top_logits`` are bf16, fp16 or fp32 with any row stride and alignment, ``V`` up to
    1048576, ``K`` up to 1024.  On the GPU an id or label outside the vocabulary records an error in
    the status block and is left out; on the CPU it raises ``IndexError``."""
    if logits.is_cuda:
        return kernels().distill_fwd(logits, top_ids, top_logits, temperature, top_lse, labels)
    name = "distill_fwd"
    _check_distill(name, logits, top_ids, top_logits, temperature, labels)
    T, V = logits.shape
    _need(top_lse is None or _vector(top_lse, T, torch.float32), "{}: top_lse must be fp32 [{}]", name,
          T)
    _need_index(top_ids.clamp(min=0), V, f"{name}: an id is")
    if labels is not None:
        _need_index(labels.clamp(min=0), V, f"{name}: a label is")
    return tuple(None if t is None else t.float()
                 for t in ref.distill(logits, top_ids, top_logits, temperature, top_lse, labels))


def distill_bwd(logits: torch.Tensor, top_ids: torch.Tensor, top_logits: torch.Tensor,
                stats: torch.Tensor, dkd: torch.Tensor, temperature: float = 1.0,
                labels: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                dce: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dlogits of ``sum dkd kd + dce ce`` (:func:`distill_fwd`) for the rows ``rows`` (int32 ``[R]``;
    all when ``None``), rounded once: what both losses give, in one pass.

    ``dkd [R]`` and ``dce [R]`` are fp32; ``labels``, ``lse`` (of the forward) and ``dce`` go
    together.  A weight of zero adds nothing, whatever the row holds.  Relative to a logarithm of 2^23 or
    more in size (a row of masks alone) exponentials count as zero, since fp32 statistics do not hold
    its digits.  ``out [R, V]`` has the type of
    the logits and any row stride, and may be the logits themselves without ``rows``; other overlaps
    are refused.  On the GPU a row id outside the logits records an error in the status block and
    gives a zero row; on the CPU it raises ``IndexError``."""
    if logits.is_cuda:
        return kernels().distill_bwd(logits, top_ids, top_logits, stats, dkd, temperature, labels, lse,
                                     dce, rows, out)
    name = "distill_bwd"
    _check_distill(name, logits, top_ids, top_logits, temperature, labels)
    T, V = logits.shape
    _need(dkd.dim() == 1 and _vector(dkd, dkd.shape[0], torch.float32), "{}: dkd must be fp32 [R]",
          name)
    R = dkd.shape[0]
    _need(stats.shape == (T, 4) and stats.dtype == torch.float32 and stats.is_contiguous(),
          "{}: stats must be contiguous fp32 [{}, 4]", name, T)
    _need((lse is None) == (labels is None) and (dce is None) == (labels is None),
          "{}: labels, lse and dce go together", name)
    _need(labels is None or _vector(lse, T, torch.float32) and _vector(dce, R, torch.float32),
          "{}: lse must be fp32 [{}] and dce fp32 [{}]", name, T, R)
    if rows is None:
        _need(R == T, "{}: {} gradient rows for {} rows", name, R, T)
    else:
        _need(_vector(rows, R, torch.int32), "{}: rows must be contiguous int32 [{}]", name, R)
    if out is not None:
        _need(_rows2d(out, V) and out.shape[0] == R and out.dtype == logits.dtype,
              "{}: out must be row-major {} [{}, {}]", name, logits.dtype, R, V)
        _check_apart(name, "out", out,
                     (logits, top_ids, top_logits, stats, dkd, labels, lse, dce, rows),
                     logits if rows is None else None)
    if rows is not None:
        _need_index(rows, T, f"{name}: a row id is")
        at = rows.long()
        logits, top_ids, top_logits, stats = logits[at], top_ids[at], top_logits[at], stats[at]
        labels, lse = (None, None) if labels is None else (labels[at], lse[at])
    _need_index(top_ids.clamp(min=0), V, f"{name}: an id is")
    if labels is not None:
        _need_index(labels.clamp(min=0), V, f"{name}: a label is")
    g = ref.distill_bwd(logits, top_ids, top_logits, stats, dkd, temperature, labels, lse, dce)
    return g.to(logits.dtype) if out is None else out.copy_(g)


# ---------------------------------------------------------------- cross entropy
def ce_fwd(logits: torch.Tensor, labels: torch.Tensor, loss: Optional[torch.Tensor] = None,
           lse: Optional[torch.Tensor] = None):
    rows = logits.shape[0]
    if loss is None:
        loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
    if lse is None:
        lse = torch.empty(rows, dtype=torch.float32, device=logits.device)
    if not logits.is_cuda:
        l, s = ref.cross_entropy(logits, labels)
        loss.copy_(l)
        lse.copy_(s)
        return loss, lse
    kernels().ce_fwd(logits, labels, loss, lse)
    return loss, lse


def ce_bwd(logits: torch.Tensor, labels: torch.Tensor, lse: torch.Tensor, dloss: torch.Tensor,
           rows: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
           vocab_start: int = 0):
    """dlogits of the rows ``rows`` (all when None); with a vocabulary shard the logits'
    columns are the global ids ``vocab_start + j`` and ``lse`` is the full-vocabulary lse."""
    n = dloss.numel()
    if out is None:
        out = torch.empty(n, logits.shape[1], dtype=logits.dtype, device=logits.device)
    if not logits.is_cuda:
        r = torch.arange(logits.shape[0]) if rows is None else rows.long()
        lab = labels[r]
        V = logits.shape[1]
        p = torch.exp(logits[r].float() - lse[r].unsqueeze(-1))
        loc = lab - vocab_start
        hit = (lab >= 0) & (loc >= 0) & (loc < V)
        p[hit, loc[hit]] -= 1.0
        p = p * dloss.unsqueeze(-1)
        p[lab < 0] = 0
        out.copy_(p)
        return out
    kernels().ce_bwd(logits, rows, labels, lse, dloss, out, vocab_start)
    return out


def ce_partial(logits: torch.Tensor, labels: torch.Tensor, vocab_start: int, out=None):
    """Per-row (max, sum exp(logit - max), label logit or 0) of one vocabulary shard;
    ``out``: three fp32 ``[rows]`` tensors to write them into."""
    rows = logits.shape[0]
    f32 = dict(dtype=torch.float32, device=logits.device)
    pmax, psum, ptgt = out if out is not None else (torch.empty(rows, **f32) for _ in range(3))
    if not logits.is_cuda:
        lf = logits.float()
        pmax.copy_(lf.max(-1).values)
        psum.copy_(torch.exp(lf - pmax.unsqueeze(-1)).sum(-1))
        loc = labels - vocab_start
        hit = (labels >= 0) & (loc >= 0) & (loc < lf.shape[1])
        t = torch.zeros(rows, **f32)
        t[hit] = lf[hit, loc[hit]]
        ptgt.copy_(t)
        return pmax, psum, ptgt
    kernels().ce_partial(logits, labels, pmax, psum, ptgt, vocab_start)
    return pmax, psum, ptgt


# ---------------------------------------------------------------- optimizer
def adamw_(master, grad, m, v, param, lr, beta1, beta2, eps, wd, step, grad_scale=None):
    """Fused AdamW step on flat fp32 buffers; writes the bf16 copy into ``param``."""
    bc1 = 1.0 - beta1 ** step
    bc2 = 1.0 - beta2 ** step
    if not master.is_cuda:
        g = grad * (grad_scale if grad_scale is not None else 1.0)
        master.mul_(1 - lr * wd)
        m.mul_(beta1).add_(g, alpha=1 - beta1)
        v.mul_(beta2).addcmul_(g, g, value=1 - beta2)
        denom = (v.sqrt() / math.sqrt(bc2)).add_(eps)
        master.addcdiv_(m, denom, value=-lr / bc1)
        param.copy_(master)
        return
    kernels().adamw(master, grad, m, v, param, lr, beta1, beta2, eps, wd, bc1, bc2, grad_scale)


def grad_norm_clip_coef(grad: torch.Tensor, max_norm: float, extra_scale: float,
                        coef: torch.Tensor, norm: torch.Tensor,
                        partial: Optional[torch.Tensor] = None,
                        extra_sumsq: Optional[torch.Tensor] = None):
    """On-device ``coef = clip(max_norm / ||g * extra_scale||) * extra_scale``.

    ``extra_sumsq`` lets data-parallel ranks add the squared norms of the other shards (it is
    the all-reduced sum of the per-rank partial sums).
    """
    if not grad.is_cuda:
        s = grad.float().pow(2).sum()
        if extra_sumsq is not None:
            s = extra_sumsq.sum()
        n = s.sqrt() * extra_scale
        c = 1.0
        if max_norm > 0 and n > max_norm:
            c = max_norm / (float(n) + 1e-6)
        coef.fill_(c * extra_scale)
        norm.fill_(float(n))
        return coef
    k = kernels()
    if extra_sumsq is None:
        if partial is None:
            partial = torch.empty(148 * 4, dtype=torch.float32, device=grad.device)
        k.sumsq(grad, partial)
        extra_sumsq = partial
    k.clip_coef(extra_sumsq, max_norm, extra_scale, coef, norm)
    return coef


def grad_list_sumsq(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """Sum of squares of all elements of a list of tensors, as fp32 partial sums whose total it is.
    Ranks that hold different parameters add their totals (an all-reduce of ``.sum()``) and give the
    result to :func:`grad_list_clip_` as ``extra_sumsq``."""
    grads = list(grads)
    if grads and grads[0].is_cuda:
        return kernels().grad_list_sumsq(grads)
    _need(len(grads) > 0, "grad_list_sumsq: empty list")
    _check_grads("grad_list_sumsq", grads)
    return sum(g.double().pow(2).sum() for g in grads).float().view(1)


def _check_grads(name: str, grads: List[torch.Tensor], dev: Optional[torch.device] = None) -> None:
    dev = dev or grads[0].device
    for i, g in enumerate(grads):
        if g.dtype not in _ROW_TYPES or g.device != dev or g.layout != torch.strided:
            raise ValueError(f"{name}: tensor {i} must be a dense bf16, fp16 or fp32 tensor on {dev}")


def _check_spans(grads: List[torch.Tensor], outs: List[torch.Tensor],
                 norm: Optional[torch.Tensor], extra_sumsq: Optional[torch.Tensor]) -> None:
    """Outputs shaped like their gradients and dense; nothing that is written (the outputs and the
    norm) overlaps anything else."""
    spans, end, end_written = [], 0, 0

    def add(t: torch.Tensor, name: str, written: bool) -> None:
        lo = t.data_ptr()
        if t.numel():
            spans.append((lo, lo + t.numel() * t.element_size(), name, written))

    for i, (g, o) in enumerate(zip(grads, outs)):
        _need(o.shape == g.shape and (o.stride() == g.stride()
                                      or o.is_contiguous() and g.is_contiguous()),
              "grad_list_clip_: output {} must have the sizes and strides of its gradient", i)
        _need(torch.ops.aten.is_non_overlapping_and_dense.default(g),
              "grad_list_clip_: tensor {} has gaps or overlaps itself", i)
        if not (o.data_ptr() == g.data_ptr() and o.dtype == g.dtype):
            add(g, f"tensor {i}", False)
        add(o, f"tensor {i}", True)
    if norm is not None:
        add(norm, "norm", True)
    if extra_sumsq is not None:
        add(extra_sumsq, "extra_sumsq", False)
    for lo, hi, name, written in sorted(spans):
        _need(lo >= (end if written else end_written),
              "grad_list_clip_: {} and another tensor overlap, and one of them is written", name)
        end, end_written = max(end, hi), max(end_written, hi) if written else end_written


def grad_list_clip_(grads: Sequence[torch.Tensor], max_norm: float, extra_scale: float = 1.0,
                    out: Optional[Sequence[torch.Tensor]] = None,
                    norm: Optional[torch.Tensor] = None,
                    extra_sumsq: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Clip a list of gradients by their global norm, without a host synchronisation::

        norm   = extra_scale * sqrt(sum of all squares)
        out[i] = grads[i] * extra_scale * min(1, max_norm / (norm + 1e-6))

    in place, or into the tensors ``out`` (which may have other types: bf16 gradients into the
    optimizer's fp32 buffer).  Returns ``norm`` (fp32 ``[1]``).  ``max_norm <= 0`` sets no limit.
    A norm that is infinite or no number is returned as such, and carries over to the gradients as
    the formula says.  ``extra_sumsq``: fp32 partial sums of squares to use instead of the list's
    own (see :func:`grad_list_sumsq`); the norm is theirs for an empty list too.

    Tensors are bf16, fp16 or fp32, of any size and alignment, in any dense layout (``out[i]``
    in that of ``grads[i]``); the list may mix types.  Tensors with gaps are refused, and so are
    outputs and a ``norm`` that overlap anything else of the call.  The
    squares and their partial sums are fp32: a norm (before ``extra_scale``) above 1.8e19 may come
    out infinite, and elements below 1e-19 count with fewer bits, below 2.6e-23 not at all."""
    grads = list(grads)
    if not extra_scale > 0:
        raise ValueError(f"grad_list_clip_: extra_scale = {extra_scale} is not positive")
    outs = grads if out is None else list(out)
    _need(len(outs) == len(grads), "grad_list_clip_: {} gradients, {} outputs", len(grads),
          len(outs))
    if not grads and extra_sumsq is None:
        return torch.zeros(1) if norm is None else norm.zero_()
    first = grads[0] if grads else extra_sumsq
    if first.is_cuda:
        return kernels().grad_list_clip(grads, None if out is None else outs, max_norm, extra_scale,
                                        norm, extra_sumsq)
    if grads:
        _check_grads("grad_list_clip_", grads)
        _check_grads("grad_list_clip_", outs, first.device)
    for name, t in (("norm", norm), ("extra_sumsq", extra_sumsq)):
        _need(t is None or t.dtype == torch.float32 and t.is_contiguous() and t.numel() > 0
              and t.device == first.device, "grad_list_clip_: {} must be contiguous fp32 on {}", name,
              first.device)
    _need(norm is None or norm.numel() == 1, "grad_list_clip_: norm has more than one element")
    _check_spans(grads, outs, norm, extra_sumsq)
    if norm is None:
        norm = torch.empty(1, dtype=torch.float32, device=first.device)
    if extra_sumsq is None:
        extra_sumsq = grad_list_sumsq(grads)
    norm.copy_((extra_sumsq.double().sum().sqrt() * extra_scale).view(norm.shape))
    k = extra_scale
    if max_norm > 0:
        k = (max_norm / (norm.view(()) + 1e-6)).clamp(max=1.0) * extra_scale
    for g, o in zip(grads, outs):
        o.copy_(g.float() * k)
    return norm


def grad_list_clip_coef(grads: Sequence[torch.Tensor], max_norm: float, extra_scale: float,
                        coef: torch.Tensor, norm: torch.Tensor) -> torch.Tensor:
    """:func:`grad_norm_clip_coef` of a list of tensors: ``coef`` and ``norm`` for an optimizer that
    takes the factor itself (:func:`adamw_`'s ``grad_scale``); the gradients are only read.  ``coef``
    and ``norm`` are one fp32 element each, on the device of the list."""
    grads = list(grads)
    sums = grad_list_sumsq(grads)
    for name, t in (("coef", coef), ("norm", norm)):
        _need(t.dtype == torch.float32 and t.numel() == 1 and t.device == sums.device,
              "grad_list_clip_coef: {} must be one fp32 element on {}", name, sums.device)
    return grad_norm_clip_coef(sums, max_norm, extra_scale, coef, norm, extra_sumsq=sums)


# ---------------------------------------------------------------- attention
def attn_fwd(qkv: torch.Tensor, B: int, S: int, nh: int, nkv: int, hd: int,
             out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
             scale: Optional[float] = None):
    """Causal GQA attention over the fused ``qkv [B*S, (nh+2nkv)*hd]`` rows.

    Returns ``o [B*S, nh*hd]`` (bf16) and ``lse [B*S, nh]`` (fp32).
    """
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    T = B * S
    if out is None:
        out = torch.empty(T, nh * hd, dtype=qkv.dtype, device=qkv.device)
    if lse is None:
        lse = torch.empty(T, nh, dtype=torch.float32, device=qkv.device)
    if not qkv.is_cuda:
        q = qkv[:, : nh * hd].reshape(B, S, nh, hd)
        k = qkv[:, nh * hd:(nh + nkv) * hd].reshape(B, S, nkv, hd)
        v = qkv[:, (nh + nkv) * hd:(nh + 2 * nkv) * hd].reshape(B, S, nkv, hd)
        o, l = ref.attention(q, k, v, True, scale)
        out.copy_(o.reshape(T, nh * hd))
        lse.copy_(l.reshape(T, nh))
        return out, lse
    kernels().attn_fwd(qkv, out, lse, B, S, nh, nkv, hd, scale)
    return out, lse


def attn_bwd(qkv_k: torch.Tensor, qkv_full: torch.Tensor, o_k: torch.Tensor, do_k: torch.Tensor,
             lse_k: torch.Tensor, pos_k: torch.Tensor, B: int, S: int, Sk: int, nh: int,
             nkv: int, hd: int, dqkv_k: Optional[torch.Tensor] = None,
             scale: Optional[float] = None,
             rope_table: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Filtered (restore-Q) attention backward; returns ``dqkv_k [B*Sk, ld]``.

    With ``rope_table`` the q and k gradients come out with the RoPE backward applied (rotated
    back to the pre-RoPE projection outputs at the kept rows' positions)."""
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    if dqkv_k is None:
        dqkv_k = torch.empty_like(qkv_k)
    if not qkv_k.is_cuda:
        q = qkv_k[:, : nh * hd].reshape(B, Sk, nh, hd)
        k = qkv_full[:, nh * hd:(nh + nkv) * hd].reshape(B, S, nkv, hd)
        v = qkv_full[:, (nh + nkv) * hd:(nh + 2 * nkv) * hd].reshape(B, S, nkv, hd)
        dq, dk, dv = ref.attention_bwd_filtered(
            q, k, v, o_k.reshape(B, Sk, nh, hd), do_k.reshape(B, Sk, nh, hd),
            lse_k.reshape(B, Sk, nh), pos_k.reshape(B, Sk), scale)
        dq = dq.reshape(B * Sk, nh, hd)
        dk = dk.reshape(B * Sk, nkv, hd)
        if rope_table is not None:
            pf = pos_k.reshape(-1)
            dq = ref.rope(dq, pf, rope_table, inverse=True)
            dk = ref.rope(dk, pf, rope_table, inverse=True)
        dqkv_k[:, : nh * hd] = dq.reshape(B * Sk, nh * hd)
        dqkv_k[:, nh * hd:(nh + nkv) * hd] = dk.reshape(B * Sk, nkv * hd)
        dqkv_k[:, (nh + nkv) * hd:(nh + 2 * nkv) * hd] = dv.reshape(B * Sk, nkv * hd)
        return dqkv_k
    delta = torch.empty(B * Sk * nh, dtype=torch.float32, device=qkv_k.device)
    kernels().attn_bwd(qkv_k, qkv_full, o_k, do_k, lse_k, pos_k, dqkv_k, delta, B, S, Sk, nh, nkv,
                       hd, scale, rope_table)
    return dqkv_k
    delta = torch.empty(B * Sk * nh, dtype=torch.float32, device=qkv_k.device)
    kernels().attn_bwd(qkv_k, qkv_full, o_k, do_k, lse_k, pos_k, dqkv_k, delta, B, S, Sk, nh, nkv,
                       hd, scale)
    return dqkv_k
