"""The row operators around the blocks of a training step, as cases to be measured.

* scaled embedding lookup, and its gradient over the kept rows;
* the norms after and before a block with the block's gate and the residual scale, and their
  gradient over the kept rows;
* the global gradient norm over a list of tensors, with clipping.

``run`` computes an operator in elementary torch operations, or, with ``own`` set, through
:mod:`centrifuge_b200.ops.fused`.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # two sequences of 128 tokens through a unit-test model: launch latency
        {"name": "embed fwd small", "op": "embed_fwd", "vocab": 1024, "hidden": 256, "rows": 256,
         "dtype": "bf16", "out": "bf16"},
        # a micro-batch of TinyLlama-1.1B, 8 x 2048 tokens
        {"name": "embed fwd 8x2048", "op": "embed_fwd", "vocab": 32000, "hidden": 2048,
         "rows": 16384, "dtype": "bf16", "out": "bf16"},
        # half of the tokens of the small batch kept by the filter
        {"name": "embed bwd small", "op": "embed_bwd", "vocab": 1024, "hidden": 256, "tokens": 256,
         "rows": 128, "dtype": "bf16", "pad": 0.0},
        # half of a TinyLlama micro-batch kept, token frequencies of natural text
        {"name": "embed bwd 8x2048 kept", "op": "embed_bwd", "vocab": 32000, "hidden": 2048,
         "tokens": 16384, "rows": 8192, "dtype": "bf16", "pad": 0.0},
        # Llama-3-8B's table, two sequences of 4096 of which a third is one padding token
        {"name": "embed bwd 2x4096 padded", "op": "embed_bwd", "vocab": 128256, "hidden": 4096,
         "tokens": 8192, "rows": 8192, "dtype": "bf16", "pad": 0.35},
        # the small batch's norms
        {"name": "norms fwd small", "op": "norms_fwd", "rows": 256, "hidden": 256, "dtype": "bf16",
         "resid": "bf16", "gate": "none", "pre": True},
        # a TinyLlama micro-batch, a learned gate for each channel
        {"name": "norms fwd 8x2048", "op": "norms_fwd", "rows": 16384, "hidden": 2048,
         "dtype": "bf16", "resid": "bf16", "gate": "channel", "pre": True},
        # Llama-3-8B's width, ragged rows, the residual stream in fp32, one weight for each token
        {"name": "norms fwd wide fp32 stream", "op": "norms_fwd", "rows": 8190, "hidden": 4096,
         "dtype": "bf16", "resid": "fp32", "gate": "token", "pre": True},
        # few kept rows of an odd batch at a width that is no power of two
        {"name": "norms bwd small", "op": "norms_bwd", "tokens": 399, "rows": 200, "hidden": 1000,
         "dtype": "fp16", "resid": "fp16", "gate": "none", "pre": True, "dy": True},
        # half of a TinyLlama micro-batch kept, a learned gate for each channel
        {"name": "norms bwd 8x2048 kept", "op": "norms_bwd", "tokens": 16384, "rows": 8192,
         "hidden": 2048, "dtype": "bf16", "resid": "bf16", "gate": "channel", "pre": True,
         "dy": True},
        # gradients of a unit-test model in fp32, under the limit, in place
        {"name": "clip small in place", "op": "clip", "layers": 2, "hidden": 128, "ffn": 256,
         "vocab": 512, "kv": 64, "dtype": "fp32", "out": "same", "over": 0.5},
        # bf16 gradients of TinyLlama-1.1B, over the limit, into the optimizer's fp32 buffer
        {"name": "clip TinyLlama to fp32", "op": "clip", "layers": 22, "hidden": 2048, "ffn": 5632,
         "vocab": 32000, "kv": 256, "dtype": "bf16", "out": "fp32", "over": 3.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed_fwd", "embed_bwd", "norms_fwd", "norms_bwd", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    hidden = _log(rng, 96, 4096)
    if rng.random() < 0.7:  # most widths are whole vectors, some are odd
        hidden = max(8, hidden // 8 * 8)
    tokens = _log(rng, 1, 16384)
    rows = max(1, int(tokens * rng.uniform(0.3, 1.0)))
    if op == "embed_fwd":
        return {"op": op, "vocab": _log(rng, 300, 128256), "hidden": hidden, "rows": tokens,
                "dtype": dtype, "out": rng.choice([dtype, "fp32"])}
    if op == "embed_bwd":
        return {"op": op, "vocab": _log(rng, 300, 64000), "hidden": hidden, "tokens": tokens,
                "rows": rows, "dtype": dtype, "pad": rng.choice([0.0, 0.0, 0.2, 0.9])}
    gate = rng.choice(["none", "channel", "token", "element"])
    resid = rng.choice([dtype, "fp32"])
    if op == "norms_fwd":
        return {"op": op, "rows": tokens, "hidden": hidden, "dtype": dtype, "resid": resid,
                "gate": gate, "pre": rng.random() < 0.8}
    if op == "norms_bwd":
        pre = rng.random() < 0.8
        return {"op": op, "tokens": tokens, "rows": rows, "hidden": hidden, "dtype": dtype,
                "resid": resid, "gate": gate, "pre": pre, "dy": not pre or rng.random() < 0.7}
    c = {"op": op, "layers": rng.randint(1, 24), "hidden": hidden, "ffn": _log(rng, 200, 5632),
         "vocab": _log(rng, 300, 32000), "kv": rng.randint(16, 256), "dtype": dtype,
         "out": rng.choice(["same", "fp32"]), "over": rng.choice([0.3, 2.0, 50.0])}
    # no more bytes than the largest listed case
    c["layers"] = max(1, min(c["layers"], int(c["layers"] * 5e9 / work(c)["bytes"])))
    return c


def _grad_shapes(c):
    h, f, kv = c["hidden"], c["ffn"], c["kv"]
    layer = [(h, h), (kv, h), (kv, h), (h, h), (f, h), (f, h), (h, f), (h,), (h,)]
    return [(c["vocab"], h)] + layer * c["layers"] + [(h,), (c["vocab"], h)]


def _writes(c):
    """Whether clipping has anything to write: in place only a norm over the limit scales."""
    return c["out"] == "fp32" or c["over"] > 1.0


def work(case):
    c, op = case, case["op"]
    if op == "embed_fwd":
        n = c["rows"] * c["hidden"]
        return {"bytes": n * (SIZE[c["dtype"]] + SIZE[c["out"]]) + 8 * c["rows"], "flops": n}
    if op == "embed_bwd":
        n = c["rows"] * c["hidden"]
        return {"bytes": n * SIZE[c["dtype"]] + 12 * c["rows"] + 4 * c["vocab"] * c["hidden"],
                "flops": 2 * n}
    if op in ("norms_fwd", "norms_bwd"):
        n, e, r = c["rows"] * c["hidden"], SIZE[c["dtype"]], SIZE[c["resid"]]
        g = {"none": 0, "channel": e * c["hidden"], "token": 4 * c["rows"], "element": e * n}
        if op == "norms_fwd":  # h, x, gate read; y, n written
            b = n * (e + 2 * r + (e if c["pre"] else 0)) + g[c["gate"]] + 8 * c["rows"]
            return {"bytes": b, "flops": 12 * n}
        # h, y (where the norm before needs it), dn, dy, gate read; dx, dh, dgate written
        b = n * (2 * e + r + ((e + r) if c["pre"] else 0) + (r if c["dy"] else 0))
        return {"bytes": b + 2 * g[c["gate"]] + 12 * c["rows"], "flops": 24 * n}
    n = sum(math.prod(s) for s in _grad_shapes(c))
    out = SIZE["fp32"] if c["out"] == "fp32" else SIZE[c["dtype"]]
    return {"bytes": n * SIZE[c["dtype"]] + (n * out if _writes(c) else 0), "flops": 3 * n}


# ---------------------------------------------------------------- inputs
def _tokens(g, n, vocab, pad=0.0):
    """Token ids with the 1 / rank frequencies of text, and a share `pad` of one more token."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(vocab)) - 1).long().clamp_(0, vocab - 1)
    if pad:
        p = torch.rand(n, generator=g, device="cuda")
        ids = torch.where(p < pad, torch.full_like(ids, vocab // 2), ids)
    return ids


def _kept(g, tokens, rows):
    return torch.randperm(tokens, generator=g, device="cuda")[:rows].sort().values.int()


def _normal(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def prepare(case, seed):
    c, op = case, case["op"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[c["dtype"]]
    H = c["hidden"]
    s = {"op": op}
    if op == "embed_fwd":
        s.update(table=_normal(g, c["vocab"], H, dtype=dt, scale=0.02),
                 ids=_tokens(g, c["rows"], c["vocab"]), scale=math.sqrt(H), out=TYPES[c["out"]])
    elif op == "embed_bwd":
        s.update(dy=_normal(g, c["rows"], H, dtype=dt), scale=math.sqrt(H),
                 ids=_tokens(g, c["tokens"], c["vocab"], c["pad"]),
                 kept=_kept(g, c["tokens"], c["rows"]),
                 dtable=torch.empty(c["vocab"], H, device="cuda"))
    elif op in ("norms_fwd", "norms_bwd"):
        rt = TYPES[c["resid"]]
        T = c["rows"] if op == "norms_fwd" else c["tokens"]
        s.update(h=_normal(g, T, H, dtype=dt), block_scale=0.5, resid_scale=0.9,
                 w_post=_normal(g, H, dtype=dt, scale=0.1, shift=1.0),
                 w_pre=_normal(g, H, dtype=dt, scale=0.1, shift=1.0) if c["pre"] else None)
        s["gate"] = {"none": lambda: None,
                     "channel": lambda: _normal(g, H, dtype=dt, scale=0.2, shift=0.5),
                     "token": lambda: torch.rand(T, 1, generator=g, device="cuda"),
                     "element": lambda: torch.rand(T, H, generator=g, device="cuda").to(dt),
                     }[c["gate"]]()
        x = _normal(g, T, H, dtype=rt, scale=2.0)
        if op == "norms_fwd":
            s["x"] = x
        else:
            s["y"], _, s["rstd_post"], s["rstd_pre"] = _norms_fwd({**s, "x": x})
            s["dn"] = _normal(g, c["rows"], H, dtype=dt) if c["pre"] else None
            s["dy"] = _normal(g, c["rows"], H, dtype=rt) if c["dy"] else None
            s["kept"] = _kept(g, T, c["rows"])
            s["dw"] = torch.empty(3, H, device="cuda")  # the weights' and the gate's gradients
    else:
        shapes = _grad_shapes(c)
        n = sum(math.prod(x) for x in shapes)
        s["grads"] = [_normal(g, *x, dtype=dt, scale=1e-3) for x in shapes]
        s["max_norm"] = 1e-3 * math.sqrt(n) / c["over"]
        s["flat"] = torch.empty(n, device="cuda") if c["out"] == "fp32" else None
        if c["out"] == "fp32":
            parts = s["flat"].split([math.prod(x) for x in shapes])
            s["outs"] = [p.view(x) for p, x in zip(parts, shapes)]
        else:
            s["outs"] = [torch.empty_like(t) for t in s["grads"]] if c["over"] > 1.0 else None
    return s


# ---------------------------------------------------------------- plain forms
def _embed_fwd(s):
    return (s["table"][s["ids"]].float() * s["scale"]).to(s["out"])


def _embed_bwd(s):
    tok = s["ids"][s["kept"].long()]
    s["dtable"].zero_()
    return s["dtable"].index_add_(0, tok, s["dy"].float() * s["scale"])


def _norms_fwd(s):
    h = s["h"].float()
    rstd_post = torch.rsqrt(h.square().mean(-1) + EPS)
    b = h * rstd_post[:, None] * s["w_post"].float()
    if s["gate"] is not None:
        b = b * s["gate"].float()
    y = s["resid_scale"] * s["x"].float() + s["block_scale"] * b
    if s["w_pre"] is None:
        return y.to(s["x"].dtype), None, rstd_post, None
    rstd_pre = torch.rsqrt(y.square().mean(-1) + EPS)
    n = y * rstd_pre[:, None] * s["w_pre"].float()
    return y.to(s["x"].dtype), n.to(s["h"].dtype), rstd_post, rstd_pre


def _norms_bwd(s):
    kept, gate = s["kept"].long(), s["gate"]
    h, rp = s["h"][kept].float(), s["rstd_post"][kept][:, None]
    dY = 0.0 if s["dy"] is None else s["dy"].float()
    dw_pre = None
    if s["w_pre"] is not None:
        y, rq, dn = s["y"][kept].float(), s["rstd_pre"][kept][:, None], s["dn"].float()
        a = dn * s["w_pre"].float()
        dY = dY + rq * a - y * (rq ** 3) * (a * y).mean(-1, keepdim=True)
        dw_pre = (dn * y * rq).sum(0)
    w = s["w_post"].float()
    hat = h * rp
    t = s["block_scale"] * dY
    if gate is None:
        gf, dgate = 1.0, None
    elif gate.dim() == 1:
        gf, dgate = gate.float(), (t * hat * w).sum(0)
    elif gate.shape[1] == 1:
        gf, dgate = gate[kept].float(), (t * hat * w).sum(-1, keepdim=True)
    else:
        gf, dgate = gate[kept].float(), (t * hat * w).to(gate.dtype)
    b = t * gf
    dw_post = (b * hat).sum(0)
    a = b * w
    dh = rp * a - h * (rp ** 3) * (a * h).mean(-1, keepdim=True)
    dx = s["resid_scale"] * dY
    return dx.to(s["y"].dtype), dh.to(s["h"].dtype), dw_post, dw_pre, dgate


def _clip(s):
    total = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["grads"]]).sum()
    norm = total.sqrt().float()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    if s["outs"] is not None:
        torch._foreach_copy_(s["outs"], [g.float() * coef for g in s["grads"]])
    return norm.view(1)


def _clipped(s, norm):
    """The norm, and the gradients: the whole buffer, or the first sixty tensors of a list."""
    if s["flat"] is not None:
        return {"norm": norm, "flat": s["flat"]}
    return {"norm": norm, "grads": (s["outs"] if s["outs"] is not None else s["grads"])[:60]}


# ---------------------------------------------------------------- one pass
def run(s):
    op = s["op"]
    if own:
        from centrifuge_b200.ops import fused
    if op == "embed_fwd":
        if not own:
            return _embed_fwd(s)
        out = None
        if s["out"] != s["table"].dtype:
            out = torch.empty(s["ids"].numel(), s["table"].shape[1], dtype=s["out"], device="cuda")
        return fused.scaled_embedding_fwd(s["table"], s["ids"], s["scale"], out=out)
    if op == "embed_bwd":
        if not own:
            return _embed_bwd(s)
        return fused.scaled_embedding_bwd(s["dy"], s["ids"], s["dtable"], s["scale"],
                                          id_rows=s["kept"], accumulate=False)
    if op == "norms_fwd":
        if not own:
            return _norms_fwd(s)
        return fused.block_norms_fwd(s["h"], s["x"], s["w_post"], s["w_pre"], EPS, gate=s["gate"],
                                     block_scale=s["block_scale"], resid_scale=s["resid_scale"])
    if op == "norms_bwd":
        if not own:
            return _norms_bwd(s)
        gate, pre = s["gate"], s["w_pre"] is not None
        dw_post, dw_pre = s["dw"][0], s["dw"][1] if pre else None
        dgate = s["dw"][2] if gate is not None and gate.dim() == 1 else None
        dx, dh, dgate = fused.block_norms_bwd(
            s["dy"], s["dn"], s["h"], s["y"] if pre else None, s["rstd_post"], s["rstd_pre"],
            s["w_post"], s["w_pre"], dw_post, dw_pre, gate=gate, dgate=dgate,
            block_scale=s["block_scale"], resid_scale=s["resid_scale"], rows=s["kept"],
            accumulate=False)
        return dx, dh, dw_post, dw_pre, dgate
    if own:
        return _clipped(s, fused.grad_list_clip_(s["grads"], s["max_norm"], out=s["outs"]))
    return _clipped(s, _clip(s))


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    c, op = case, case["op"]
    s = prepare(case, seed)
    if op == "embed_fwd":
        rows = torch.index_select(s["table"], 0, s["ids"])
        return torch.mul(rows.double(), float(s["scale"]))
    if op == "embed_bwd":
        tok = torch.index_select(s["ids"], 0, s["kept"].long())
        order = torch.argsort(tok, stable=True)
        uniq, count = torch.unique_consecutive(tok[order], return_counts=True)
        pre = torch.zeros(tok.numel() + 1, c["hidden"], dtype=torch.float64, device="cuda")
        torch.cumsum(s["dy"].double()[order], 0, out=pre[1:])
        end = count.cumsum(0)
        full = torch.zeros(c["vocab"], c["hidden"], dtype=torch.float64, device="cuda")
        full[uniq] = (pre[end] - pre[end - count]) * s["scale"]
        return full
    if op == "norms_fwd":
        d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
        ms = torch.einsum("th,th->t", d["h"], d["h"]) / c["hidden"] + EPS
        branch = torch.einsum("th,h,t->th", d["h"], d["w_post"], ms.pow(-0.5)) * s["block_scale"]
        branch = branch * d["gate"] if "gate" in d else branch
        y = torch.add(branch, d["x"], alpha=s["resid_scale"])
        if not c["pre"]:
            return y, None, ms.pow(-0.5), None
        mq = torch.einsum("th,th->t", y, y) / c["hidden"] + EPS
        return y, torch.einsum("th,h,t->th", y, d["w_pre"], mq.pow(-0.5)), ms.pow(-0.5), mq.pow(-0.5)
    if op == "norms_bwd":
        return _exact_norms_bwd(c, s)
    sq = [torch.linalg.vector_norm(g.reshape(-1), dtype=torch.float64) for g in s["grads"]]
    norm = torch.linalg.vector_norm(torch.stack(sq))
    k = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    norm = norm.view(1)
    if s["flat"] is not None:
        flat = torch.cat([g.reshape(-1) for g in s["grads"]])
        s.clear()
        return {"norm": norm, "flat": flat.double().mul_(k)}
    return {"norm": norm, "grads": [g.double() * (k if c["over"] > 1.0 else 1.0)
                                    for g in s["grads"][:60]]}


def _exact_norms_bwd(c, s):
    """The gradient through an orthogonal projection: d(v / |v|) has no part along v."""
    at = s["kept"].long()
    H = c["hidden"]
    h, w = s["h"].index_select(0, at).double(), s["w_post"].double()
    rp = s["rstd_post"].index_select(0, at).double().unsqueeze(1)
    up = torch.zeros_like(h) if s["dy"] is None else s["dy"].double()
    dw_pre = None
    if c["pre"]:
        y = s["y"].index_select(0, at).double()
        rq = s["rstd_pre"].index_select(0, at).double().unsqueeze(1)
        dn, yh = s["dn"].double(), y * rq
        dw_pre = torch.einsum("th,th->h", dn, yh)
        v = dn * s["w_pre"].double()
        up = up + (v - yh * torch.einsum("th,th->t", v, yh).unsqueeze(1) / H) * rq
    hh = h * rp
    gate = s["gate"]
    if gate is None:
        gv = torch.ones((), dtype=torch.float64, device="cuda")
    else:
        gv = gate.double() if gate.dim() == 1 else gate.index_select(0, at).double()
    per = up * hh * s["block_scale"]  # the gradient of gate times weight, element by element
    dgate = None
    if gate is not None:
        dgate = per * w
        if gate.dim() == 1:
            dgate = dgate.sum(0)
        elif gate.shape[1] == 1:
            dgate = dgate.sum(1, keepdim=True)
    v = up * gv * w * s["block_scale"]
    dh = (v - hh * torch.einsum("th,th->t", v, hh).unsqueeze(1) / H) * rp
    return up * s["resid_scale"], dh, (per * gv).sum(0), dw_pre, dgate
