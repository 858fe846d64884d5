"""Linear-layer GEMMs on the tcgen05 kernel (csrc/kernels/gemm_sm100.cu).

Shapes follow the PyTorch ``F.linear`` convention: ``x [T, K]``, ``w [N, K]``, ``y [T, N]``.

* ``linear_fwd``     y  = x w^T            (both operands K-major)
* ``linear_dgrad``   dx = dy w             (w read MN-major: no transpose copy)
* ``linear_wgrad``   dW (+)= dy^T x        (both read MN-major; fp32 accumulate epilogue)

Layers with a bias and an activation (csrc/kernels/linear_act.cu), bf16 or fp16, of any size:

* ``linear_act_fwd``     z = x w^T + bias,  y = act(z) + resid
* ``linear_act_dgrad``   dz = (dy w) act'(z)   (through a layer into the activation below it)
* ``linear_bias_wgrad``  dW (+)= dy^T x,  dbias (+)= sum of the rows of dy

CPU tensors run the fp32 reference (``torch.matmul``); CUDA tensors always run the kernel.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._ext import kernels

EPI_BF16, EPI_BF16_RESID, EPI_F32, EPI_F32_ACC = 0, 1, 2, 3


def gemm(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor, a_mn: bool, b_mn: bool,
         epi: int = EPI_BF16, resid: Optional[torch.Tensor] = None, alpha: float = 1.0,
         bn: int = 0, max_ctas: int = 0) -> torch.Tensor:
    """``out = epi(alpha * op(a) @ op(b))`` with op(a) ``[M, K]`` and op(b) ``[K, N]``."""
    if not a.is_cuda:
        A = (a.t() if a_mn else a).float()
        B = (b if b_mn else b.t()).float()
        r = alpha * (A @ B)
        if epi == EPI_BF16_RESID:
            r = r + resid.float()
        if epi == EPI_F32_ACC:
            out += r
        else:
            out.copy_(r)
        return out
    _check_gemm_operands(a, b, out, b_mn)
    kernels().gemm(a, b, out, a_mn, b_mn, epi, resid, alpha, bn, max_ctas)
    return out


def _check_gemm_operands(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor, b_mn: bool):
    """Shape and alignment rules of the tcgen05 GEMM (TMA rows start on 16 bytes, the epilogue
    stores 32-column chunks), checked before the launch so a bad call raises here."""
    N = b.shape[1] if b_mn else b.shape[0]
    if N % 32:
        raise ValueError(f"gemm: N = {N} is not a multiple of 32")
    for name, t in (("a", a), ("b", b), ("out", out)):
        if t.dim() != 2 or t.stride(1) != 1:
            raise ValueError(f"gemm: {name} must be 2-D with unit column stride")
        if t.data_ptr() % 16:
            raise ValueError(f"gemm: {name} is not 16-byte aligned")
    if a.stride(0) % 8 or b.stride(0) % 8:
        raise ValueError("gemm: row strides of a and b must be multiples of 8 elements")


def linear_fwd(x: torch.Tensor, w: torch.Tensor, out: Optional[torch.Tensor] = None,
               resid: Optional[torch.Tensor] = None) -> torch.Tensor:
    if out is None:
        out = torch.empty(x.shape[0], w.shape[0], dtype=x.dtype, device=x.device)
    return gemm(x, w, out, False, False, EPI_BF16_RESID if resid is not None else EPI_BF16,
                resid)


def linear_fwd_ce(x: torch.Tensor, w: torch.Tensor, labels: torch.Tensor):
    """Per-token cross entropy of ``logits = x w^T`` against ``labels`` (< 0: ignored, loss 0)
    without storing the logits: the GEMM epilogue reduces every 256-column tile of a row to
    (max, sum of exp, label logit) and a combine kernel forms ``lse`` and the loss.
    Returns ``(loss [M], lse [M])`` in fp32."""
    M, N = x.shape[0], w.shape[0]
    f32 = dict(dtype=torch.float32, device=x.device)
    if not x.is_cuda:
        from . import reference as ref
        return ref.cross_entropy(x.float() @ w.float().t(), labels)
    nt = (N + 255) // 256
    pmax = torch.empty(M, nt, **f32)
    psum = torch.empty(M, nt, **f32)
    ptgt = torch.empty(M, **f32)
    loss, lse = torch.empty(M, **f32), torch.empty(M, **f32)
    k = kernels()
    k.gemm_ce_part(x, w, labels, pmax, psum, ptgt)
    k.ce_combine(pmax, psum, ptgt, labels, N, loss, lse)
    return loss, lse


def linear_ce_grad(x: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, lse: torch.Tensor,
                   dloss: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dlogits = (softmax(x w^T) - onehot(labels)) * dloss`` (bf16 ``[M, N]``) with the logits
    recomputed inside the GEMM (rows with ``labels < 0`` are zero)."""
    M, N = x.shape[0], w.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=x.dtype, device=x.device)
    if not x.is_cuda:
        from . import reference as ref
        out.copy_(ref.cross_entropy_bwd(x.float() @ w.float().t(), labels, lse, dloss))
        return out
    kernels().gemm_ce_grad(x, w, labels, lse.contiguous(), dloss.contiguous(), out)
    return out


def linear_fwd_rope(x: torch.Tensor, w: torch.Tensor, pos: torch.Tensor, table: torch.Tensor,
                    rope_cols: int, head_dim: int, out: Optional[torch.Tensor] = None
                    ) -> torch.Tensor:
    """``y = x w^T`` with rotate-half RoPE applied to columns ``[0, rope_cols)`` (heads of
    ``head_dim``) at positions ``pos [T]``, fused into the GEMM epilogue (the q and k heads of a
    fused qkv projection)."""
    if out is None:
        out = torch.empty(x.shape[0], w.shape[0], dtype=x.dtype, device=x.device)
    if not x.is_cuda:
        from . import reference as ref
        y = x.float() @ w.float().t()
        n = rope_cols // head_dim
        q = y[:, :rope_cols].view(-1, n, head_dim)
        y[:, :rope_cols] = ref.rope(q, pos, table).reshape(-1, rope_cols)
        out.copy_(y)
        return out
    kernels().gemm_rope(x, w, out, pos, table, rope_cols, head_dim)
    return out


def linear_fwd_swiglu(x: torch.Tensor, w: torch.Tensor):
    """``gu = x w^T`` for ``w = [gate; up]`` and ``h = silu(gate) * up`` from the same kernel
    (SwiGLU in the GEMM epilogue).  Returns ``(gu [T, 2F], h [T, F])``; ``gu`` is what the
    backward needs."""
    F = w.shape[0] // 2
    gu = torch.empty(x.shape[0], 2 * F, dtype=x.dtype, device=x.device)
    h = torch.empty(x.shape[0], F, dtype=x.dtype, device=x.device)
    if not x.is_cuda or F % 128:
        gu = gemm(x, w, gu, False, False)
        from . import fused
        return gu, fused.swiglu_fwd(gu, out=h)
    kernels().gemm_swiglu(x, w, gu, h)
    return gu, h


def linear_dgrad_swiglu(dy: torch.Tensor, wd: torch.Tensor, gu: torch.Tensor,
                        gu_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``d[gate; up]`` of ``h = silu(gate) * up`` given ``dy`` at the down projection's output:
    ``dh = dy wd`` (``wd [H, F]``) feeds the SwiGLU backward in the GEMM epilogue, with the saved
    ``gu`` rows ``gu_rows`` (kept rows of the forward's ``gu``; all rows when ``None``).
    Returns ``dgu [T, 2F]``; ``dh`` is never materialised."""
    F = wd.shape[1]
    dgu = torch.empty(dy.shape[0], 2 * F, dtype=dy.dtype, device=dy.device)
    if not dy.is_cuda:
        from . import fused
        dh = (dy.float() @ wd.float()).to(dy.dtype)
        return fused.swiglu_bwd(dh, gu, gu_rows, out=dgu)
    if F % 32:
        raise ValueError(f"linear_dgrad_swiglu: F = {F} is not a multiple of 32")
    kernels().gemm_swiglu_bwd(dy, wd, gu, gu_rows, dgu)
    return dgu


def linear_dgrad(dy: torch.Tensor, w: torch.Tensor, out: Optional[torch.Tensor] = None,
                 resid: Optional[torch.Tensor] = None) -> torch.Tensor:
    if out is None:
        out = torch.empty(dy.shape[0], w.shape[1], dtype=dy.dtype, device=dy.device)
    return gemm(dy, w, out, False, True, EPI_BF16_RESID if resid is not None else EPI_BF16,
                resid)


def linear_wgrad(dy: torch.Tensor, x: torch.Tensor, dw: torch.Tensor,
                 accumulate: bool = True, alpha: float = 1.0) -> torch.Tensor:
    """``dw (+)= alpha * dy^T x``; ``dw`` is fp32 ``[N, K]`` (the flat gradient bucket)."""
    return gemm(dy, x, dw, True, True, EPI_F32_ACC if accumulate else EPI_F32, None, alpha)


ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")
_HALF_TYPES = (torch.bfloat16, torch.float16)


def _act_code(name: str, act: str) -> int:
    if act not in ACTIVATIONS:
        raise ValueError(f"{name}: act = {act!r} is none of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS.index(act)


def _check_out(name: str, what: str, out: torch.Tensor, shape, dtype: torch.dtype, inputs,
               in_place: Optional[torch.Tensor] = None):
    from .fused import _need, _overlap, _rows2d
    _need(_rows2d(out, shape[1]) and out.shape[0] == shape[0] and out.dtype == dtype,
          "{}: {} must be row-major {} {}", name, what, dtype, list(shape))
    for t in inputs:
        same = t is in_place and t is not None and t.data_ptr() == out.data_ptr() and (
            t.stride() == out.stride() and t.dtype == out.dtype)
        _need(t is None or same or not _overlap(out, t), "{}: {} overlaps another tensor of the call",
              name, what)


def linear_act_fwd(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   act: str = "none", resid: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None,
                   z: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y = act(x w^T + bias) + resid``, rounded once.

    ``x [T, K]``, ``w [N, K]`` and ``resid [T, N]`` are bf16 or fp16 of one type, row-major with any
    row stride and alignment (rows that do not start on 16 bytes are laid out anew for the call);
    ``bias [N]`` is contiguous; any ``T``, ``N`` and ``K > 0``.  ``act``: one of :data:`ACTIVATIONS`
    (``gelu`` by the normal distribution, ``gelu_tanh`` by its approximation).  ``z [T, N]``, when
    given, receives the rounded ``x w^T + bias``, which :func:`linear_act_dgrad` needs.  ``out`` may
    be ``resid`` itself; other overlaps are refused.  CPU tensors may be fp32 too, as the definition
    that the others are compared with."""
    code = _act_code("linear_act_fwd", act)
    if x.is_cuda:
        return kernels().linear_act_fwd(x, w, bias, code, resid, out, z)
    from . import reference as ref
    from .fused import _need, _rows2d, _vector
    name = "linear_act_fwd"
    _need(x.dtype in _HALF_TYPES + (torch.float32,), "{}: x must be bfloat16 or float16", name)
    _need(x.dim() == 2 and w.dim() == 2 and _rows2d(x, x.shape[1]) and _rows2d(w, x.shape[1])
          and w.dtype == x.dtype, "{}: x must be row-major [T, K] and w {} [N, K]", name, x.dtype)
    _need(x.shape[1] > 0, "{}: x has no columns", name)
    shape = (x.shape[0], w.shape[0])
    _need(bias is None or _vector(bias, shape[1], x.dtype), "{}: bias must be contiguous {} [{}]",
          name, x.dtype, shape[1])
    _need(resid is None or _rows2d(resid, shape[1]) and resid.shape[0] == shape[0]
          and resid.dtype == x.dtype, "{}: resid must be row-major {} {}", name, x.dtype, shape)
    if z is not None:
        _check_out(name, "z", z, shape, x.dtype, (x, w, bias, resid, out))
    if out is not None:
        _check_out(name, "out", out, shape, x.dtype, (x, w, bias, resid), resid)
    y, zf = ref.linear_act(x, w, bias, act, resid)
    if z is not None:
        z.copy_(zf)
    return y.to(x.dtype) if out is None else out.copy_(y)


def linear_act_dgrad(dy: torch.Tensor, w: torch.Tensor, z: torch.Tensor, act: str,
                     z_rows: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dz = (dy w) act'(z[z_rows])``: the gradient ``dy [R, K]`` of a layer's output through its
    weight ``w [K, N]`` and the activation that made its input, whose argument ``z [T, N]`` the
    forward kept; on the rows ``z_rows`` (int32 ``[R]``; all when ``None``).  The product is not
    stored or rounded.  Types and layouts as in :func:`linear_act_fwd`; ``out`` may be ``z`` itself
    without ``z_rows``.  On the GPU a row id outside ``z`` records an error in the status block and
    gives a zero row; on the CPU it raises ``IndexError``."""
    code = _act_code("linear_act_dgrad", act)
    if dy.is_cuda:
        return kernels().linear_act_dgrad(dy, w, z, code, z_rows, out)
    from . import reference as ref
    from .fused import _need, _need_index, _rows2d
    name = "linear_act_dgrad"
    _need(dy.dtype in _HALF_TYPES + (torch.float32,), "{}: dy must be bfloat16 or float16", name)
    _need(dy.dim() == 2 and w.dim() == 2 and _rows2d(dy, dy.shape[1]) and _rows2d(w, w.shape[1])
          and w.shape[0] == dy.shape[1] and w.dtype == dy.dtype,
          "{}: dy must be row-major [R, K] and w {} [K, N]", name, dy.dtype)
    _need(dy.shape[1] > 0, "{}: dy has no columns", name)
    shape = (dy.shape[0], w.shape[1])
    _need(_rows2d(z, shape[1]) and z.dtype == dy.dtype, "{}: z must be row-major {} [T, {}]", name,
          dy.dtype, shape[1])
    if z_rows is None:
        _need(z.shape[0] == shape[0], "{}: {} gradient rows for {} rows of z", name, shape[0],
              z.shape[0])
    else:
        _need(z_rows.dtype == torch.int32 and z_rows.dim() == 1 and z_rows.is_contiguous()
              and z_rows.shape[0] == shape[0], "{}: z_rows must be contiguous int32 [{}]", name,
              shape[0])
    if out is not None:
        _check_out(name, "out", out, shape, dy.dtype, (dy, w, z, z_rows),
                   z if z_rows is None else None)
    if z_rows is not None:
        _need_index(z_rows, z.shape[0], f"{name}: a row id is")
    dz = ref.linear_act_dgrad(dy, w, z if z_rows is None else z[z_rows.long()], act)
    return dz.to(dy.dtype) if out is None else out.copy_(dz)


def linear_bias_wgrad(dy: torch.Tensor, x: torch.Tensor, dw: torch.Tensor,
                      dbias: Optional[torch.Tensor] = None,
                      accumulate: bool = True) -> torch.Tensor:
    """``dw (+)= dy^T x`` and ``dbias (+)= sum of the rows of dy`` (written without ``accumulate``),
    each summed in fp32 in a fixed order.  ``dy [R, N]`` and ``x [R, K]`` as in
    :func:`linear_act_fwd` (without rows nothing is added), ``dw [N, K]`` fp32 with any row stride,
    ``dbias [N]`` contiguous fp32; what is written overlaps nothing else.  Sums below 1.2e-38 may count
    as zero on the GPU."""
    if dy.is_cuda:
        kernels().linear_bias_wgrad(dy, x, dw, dbias, accumulate)
        return dw
    from .fused import _need, _overlap, _rows2d, _vector
    name = "linear_bias_wgrad"
    _need(dy.dtype in _HALF_TYPES + (torch.float32,), "{}: dy must be bfloat16 or float16", name)
    _need(dy.dim() == 2 and x.dim() == 2 and _rows2d(dy, dy.shape[1]) and _rows2d(x, x.shape[1])
          and x.shape[0] == dy.shape[0] and x.dtype == dy.dtype,
          "{}: dy must be row-major [R, N] and x {} [R, K]", name, dy.dtype)
    _check_out(name, "dw", dw, (dy.shape[1], x.shape[1]), torch.float32, (dy, x, dbias))
    if dbias is not None:
        _need(_vector(dbias, dy.shape[1], torch.float32), "{}: dbias must be contiguous fp32 [{}]",
              name, dy.shape[1])
        _need(not _overlap(dbias, dy) and not _overlap(dbias, x),
              "{}: dbias overlaps another tensor of the call", name)
    g = dy.float()
    dw.copy_(g.t() @ x.float() + (dw if accumulate else 0.0))
    if dbias is not None:
        dbias.copy_(g.sum(0) + (dbias if accumulate else 0.0))
    return dw
