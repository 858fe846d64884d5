"""Plain-PyTorch fp32 definitions of every fused op.

These are the numerical oracles the sm_100a kernels are tested against, and the code path the
ops take on CPU tensors (unit tests and the CPU filtered-gradient oracle run here).
"""
from __future__ import annotations

import math
from typing import Optional

import torch


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float):
    xf = x.float()
    rstd = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (xf * rstd * w.float()), rstd.squeeze(-1)


def rmsnorm_bwd(dy, x, rstd, w, dres=None):
    dyf, xf, wf = dy.float(), x.float(), w.float()
    r = rstd.float().unsqueeze(-1)
    H = x.shape[-1]
    dot = (wf * dyf * xf).sum(-1, keepdim=True)
    dx = r * wf * dyf - xf * dot * r.pow(3) / H
    if dres is not None:
        dx = dx + dres.float()
    dw = (dyf * xf * r).sum(0)
    return dx, dw


def block_norms(h, x, w_post, w_pre, eps, gate=None, block_scale=1.0, resid_scale=1.0):
    """Norm after a block, gate, residual sum and the norm before the next block (fp32):
    ``(y, n, rstd_post, rstd_pre)``, the last two ``None`` without ``w_pre``."""
    b, rstd_post = rmsnorm(h, w_post, eps)
    if gate is not None:
        b = b * gate.float()
    y = resid_scale * x.float() + block_scale * b
    if w_pre is None:
        return y, None, rstd_post, None
    n, rstd_pre = rmsnorm(y, w_pre, eps)
    return y, n, rstd_post, rstd_pre


def block_norms_bwd(dy, dn, h, y, rstd_post, rstd_pre, w_post, w_pre, gate=None, block_scale=1.0,
                    resid_scale=1.0):
    """Gradient of :func:`block_norms` (fp32): ``(dx, dh, dw_post, dw_pre, dgate)``."""
    dY, dw_pre = (None if dy is None else dy.float()), None
    if w_pre is not None:
        dY, dw_pre = rmsnorm_bwd(dn, y, rstd_pre, w_pre, dY)
    t = block_scale * dY
    db = t if gate is None else t * gate.float()
    dh, dw_post = rmsnorm_bwd(db, h, rstd_post, w_post)
    dgate = None
    if gate is not None:
        dgate = t * h.float() * rstd_post.unsqueeze(-1) * w_post.float()
        if gate.dim() == 1:
            dgate = dgate.sum(0)
        elif gate.shape[1] == 1 and gate.dtype == torch.float32:
            dgate = dgate.sum(-1, keepdim=True)
    return resid_scale * dY, dh, dw_post, dw_pre, dgate


def layernorm(x, w, b, eps):
    """``(y, mean, rstd)`` (fp32)."""
    xf = x.float()
    mean = xf.mean(-1)
    d = xf - mean.unsqueeze(-1)
    rstd = torch.rsqrt(d.pow(2).mean(-1) + eps)
    y = d * rstd.unsqueeze(-1)
    if w is not None:
        y = y * w.float()
    return y if b is None else y + b.float(), mean, rstd


def layernorm_bwd(dy, x, mean, rstd, w, dres=None):
    """``(dx, dw, db)`` (fp32)."""
    r = rstd.unsqueeze(-1)
    n = (x.float() - mean.unsqueeze(-1)) * r
    g = dy.float() if w is None else dy.float() * w.float()
    dx = r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    if dres is not None:
        dx = dx + dres.float()
    return dx, (dy.float() * n).sum(0), dy.float().sum(0)


def activation(z: torch.Tensor, act: str) -> torch.Tensor:
    if act == "relu":
        return torch.relu(z)
    if act == "silu":
        return torch.nn.functional.silu(z)
    if act == "gelu":  # (1 + erf would lose the small values)
        return 0.5 * z * torch.erfc(z * -math.sqrt(0.5))
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
    return z


def activation_grad(z: torch.Tensor, act: str) -> torch.Tensor:
    if act == "none":
        return torch.ones_like(z)
    with torch.enable_grad():
        z = z.detach().requires_grad_()
        return torch.autograd.grad(activation(z, act).sum(), z)[0]


def linear_act(x, w, bias, act, resid):
    """``(act(z) + resid, z)`` with ``z = x w^T + bias`` (fp32)."""
    z = x.float() @ w.float().t()
    if bias is not None:
        z = z + bias.float()
    y = activation(z, act)
    return y if resid is None else y + resid.float(), z


def linear_act_dgrad(dy, w, z, act):
    return (dy.float() @ w.float()) * activation_grad(z.float(), act)


# From here on fp32 has no digits behind the point: a rest of the vocabulary that lies so far below the
# list counts as none, and an exponential relative to such a logarithm of a sum as zero.
NO_DIGITS = 2.0 ** 23
# Finite logits below this (masks by the type's lowest value) count as being there.
LOWEST = -2.0 ** 30 * math.log(2.0)


def _with_masks(x):
    return torch.where((x < LOWEST) & (x > -math.inf), torch.full_like(x, LOWEST), x)


def distill(logits, top_ids, top_logits, temperature, top_lse=None, labels=None):
    """Divergence of the student from a teacher's top logits and the labels' cross entropy (fp64):
    ``(kd, ce, lse, stats)``; entries with a negative id are left out."""
    z, ids = logits.double(), top_ids.long()
    ok, inf = ids >= 0, float("inf")
    x = _with_masks(z / temperature)
    lse = torch.logsumexp(x, -1)
    t = (top_logits.double() / temperature).masked_fill(~ok, -inf)
    norm = torch.logsumexp(t, -1) if top_lse is None else top_lse.double()
    none = norm == -inf if top_lse is None else torch.zeros_like(norm, dtype=torch.bool)
    log_p = (t - norm.unsqueeze(-1)).masked_fill(none.unsqueeze(-1), -inf)
    p = log_p.exp()
    log_q = x.gather(-1, ids.clamp(min=0)) - lse.unsqueeze(-1)
    kd = (p * (log_p - log_q)).masked_fill(p == 0, 0.0).sum(-1)
    base, coef = lse, (~none).double()
    if top_lse is not None:
        others = torch.cat([x, x[:, :1]], -1).scatter(-1, ids.masked_fill(~ok, x.shape[-1]), -inf)
        others = others[:, :-1]
        gap = others.amax(-1) - x.amax(-1)
        base = torch.logsumexp(others, -1).masked_fill(gap < -NO_DIGITS, -inf)
        share = p.sum(-1)
        left = (1.0 - share).clamp(min=0.0)
        rest = (base - lse).masked_fill(base == -inf, -inf)
        kd = kd + (left * (left.log() - rest)).masked_fill((left == 0) | (base == -inf), 0.0)
        rounded = base.float().double()  # as a statistic, and what makes up for it
        coef = (share.clamp(min=1.0) * rest.exp() - left) * (rounded - base).clamp(-2.0, 2.0).exp()
        coef, base = coef.masked_fill(base == -inf, 0.0), rounded
    stats = torch.stack([lse, base, coef, norm], -1)
    if labels is None:
        return kd, None, None, stats
    z = _with_masks(z)
    full = torch.logsumexp(z, -1)
    ce = full - z.gather(-1, labels.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    return kd, ce.masked_fill(labels < 0, 0.0), full, stats


def _exp_from(x, log_sum):
    return torch.exp(x - log_sum).masked_fill(log_sum.abs() >= NO_DIGITS, 0.0)


def distill_bwd(logits, top_ids, top_logits, stats, dkd, temperature, labels=None, lse=None,
                dce=None):
    """Gradient of ``sum dkd kd + dce ce`` (fp64).  A weight of zero adds nothing."""
    z, ids, st = logits.double(), top_ids.long(), stats.double()
    V, inf = z.shape[-1], float("inf")
    ok = ids >= 0
    k = (dkd.double() / temperature).unsqueeze(-1)
    k = k.masked_fill((st[:, 3:4] == -inf) & (st[:, 2:3] == 0), 0.0)  # a list without a share
    x = z / temperature
    spread = k * st[:, 2:3]
    g = (_exp_from(x, st[:, 1:2]) * spread).masked_fill(spread == 0, 0.0)
    t = (top_logits.double() / temperature).masked_fill(~ok, -inf)
    p = torch.exp(t - st[:, 3:4]).masked_fill(~ok, 0.0)
    g = torch.cat([g, g[:, :1]], -1)
    at = ids.masked_fill(~ok, V)
    q = _exp_from(x.gather(-1, ids.clamp(min=0)), st[:, 0:1])
    whole = p.sum(-1, keepdim=True)  # what the teacher's terms add up to: one, but for a list of all
    whole = torch.where(st[:, 1:2] == -inf, whole, whole.clamp(min=1.0))
    g.scatter_(-1, at, k * q * whole).scatter_add_(-1, at, -k * p)
    g = g[:, :V].masked_fill((k == 0), 0.0)
    if labels is not None:
        w = dce.double().masked_fill(labels < 0, 0.0).unsqueeze(-1)
        soft = _exp_from(z, lse.double().unsqueeze(-1))
        soft.scatter_add_(-1, labels.clamp(min=0).unsqueeze(-1), -torch.ones_like(w))
        g = g + (w * soft).masked_fill(w == 0, 0.0)
    return g


def rope_table(max_pos: int, head_dim: int, theta: float, device=None) -> torch.Tensor:
    """``[max_pos, head_dim/2, 2]`` fp32 (cos, sin) of ``pos * theta^(-2i/d)`` (HF convention)."""
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.int64).float() / head_dim))
    pos = torch.arange(max_pos, dtype=torch.float32)
    freqs = torch.outer(pos, inv_freq)
    return torch.stack([freqs.cos(), freqs.sin()], dim=-1).contiguous().to(device)


def rope(x: torch.Tensor, pos: torch.Tensor, table: torch.Tensor, inverse: bool = False):
    """Rotate-half RoPE of ``x [rows, n_heads, hd]`` at positions ``pos [rows]``."""
    hd = x.shape[-1]
    half = hd // 2
    cs = table[pos.long()]  # [rows, half, 2]
    c = cs[..., 0].unsqueeze(1)
    s = cs[..., 1].unsqueeze(1)
    if inverse:
        s = -s
    x1, x2 = x[..., :half].float(), x[..., half:].float()
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)


def swiglu(gu: torch.Tensor):
    F = gu.shape[-1] // 2
    g, u = gu[..., :F].float(), gu[..., F:].float()
    return torch.nn.functional.silu(g) * u


def swiglu_bwd(dh, gu):
    F = gu.shape[-1] // 2
    g, u, d = gu[..., :F].float(), gu[..., F:].float(), dh.float()
    s = torch.sigmoid(g)
    du = d * g * s
    dg = d * u * s * (1 + g * (1 - s))
    return torch.cat([dg, du], dim=-1)


def cross_entropy(logits: torch.Tensor, labels: torch.Tensor):
    lf = logits.float()
    lse = torch.logsumexp(lf, dim=-1)
    safe = labels.clamp(min=0)
    loss = lse - lf.gather(-1, safe.unsqueeze(-1)).squeeze(-1)
    loss = torch.where(labels >= 0, loss, torch.zeros_like(loss))
    return loss, lse


def cross_entropy_bwd(logits, labels, lse, dloss):
    p = torch.exp(logits.float() - lse.unsqueeze(-1))
    onehot = torch.zeros_like(p)
    valid = labels >= 0
    onehot[valid, labels[valid]] = 1.0
    g = (p - onehot) * dloss.unsqueeze(-1)
    g[~valid] = 0
    return g


def attention(q, k, v, causal: bool = True, scale: Optional[float] = None):
    """``q [B, S, nh, hd]``, ``k, v [B, S, nkv, hd]`` -> ``(o [B, S, nh, hd], lse [B, S, nh])``."""
    B, S, nh, hd = q.shape
    nkv = k.shape[2]
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    rep = nh // nkv
    kf = k.float().repeat_interleave(rep, dim=2)
    vf = v.float().repeat_interleave(rep, dim=2)
    s = torch.einsum("bqhd,bkhd->bhqk", q.float(), kf) * scale
    if causal:
        m = torch.ones(S, S, dtype=torch.bool, device=q.device).triu(1)
        s = s.masked_fill(m, float("-inf"))
    lse = torch.logsumexp(s, dim=-1)  # [B, nh, S]
    p = torch.exp(s - lse.unsqueeze(-1))
    o = torch.einsum("bhqk,bkhd->bqhd", p, vf)
    return o, lse.permute(0, 2, 1)


def attention_bwd_filtered(q_k, k_full, v_full, o_k, do_k, lse_k, pos_k, scale=None):
    """Restore-Q filtered attention backward (fp32).

    ``q_k/o_k/do_k [B, Sk, nh, hd]`` are the kept query rows, ``k_full/v_full [B, S, nkv, hd]``
    every key, ``lse_k [B, Sk, nh]``, ``pos_k [B, Sk]`` the kept positions.  Returns
    ``dq_k [B, Sk, nh, hd]`` (all keys contribute) and ``dk_k, dv_k [B, Sk, nkv, hd]``
    (kept keys, kept queries only).
    """
    B, Sk, nh, hd = q_k.shape
    S, nkv = k_full.shape[1], k_full.shape[2]
    rep = nh // nkv
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    kf = k_full.float().repeat_interleave(rep, dim=2)
    vf = v_full.float().repeat_interleave(rep, dim=2)
    qf, of, dof = q_k.float(), o_k.float(), do_k.float()
    s = torch.einsum("bqhd,bkhd->bhqk", qf, kf) * scale  # [B, nh, Sk, S]
    keys = torch.arange(S, device=q_k.device)
    valid = keys.view(1, 1, S) <= pos_k.long().view(B, Sk, 1)  # [B, Sk, S]
    p = torch.exp(s - lse_k.float().permute(0, 2, 1).unsqueeze(-1))
    p = torch.where(valid.unsqueeze(1), p, torch.zeros_like(p))
    dp = torch.einsum("bqhd,bkhd->bhqk", dof, vf)
    delta = (dof * of).sum(-1).permute(0, 2, 1).unsqueeze(-1)  # [B, nh, Sk, 1]
    ds = p * (dp - delta)
    dq = torch.einsum("bhqk,bkhd->bqhd", ds, kf) * scale
    # kept keys only: gather key columns at the kept positions
    idx = pos_k.long().view(B, 1, 1, Sk).expand(B, nh, Sk, Sk)
    ds_kk = torch.gather(ds, 3, idx)  # [B, nh, Sk(q), Sk(k)]
    p_kk = torch.gather(p, 3, idx)
    dk = torch.einsum("bhqk,bqhd->bkhd", ds_kk, qf) * scale
    dv = torch.einsum("bhqk,bqhd->bkhd", p_kk, dof)
    dk = dk.view(B, Sk, nkv, rep, hd).sum(3)
    dv = dv.view(B, Sk, nkv, rep, hd).sum(3)
    return dq, dk, dv
