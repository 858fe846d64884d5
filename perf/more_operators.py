"""Operators of blocks with layer norms and biased linear layers, and of a student's loss.

* linear layers with bias, activation and residual: forward, the gradient through the weight and
  the activation below it, the weight's and the bias's gradient;
* layer norm, and its gradient over the kept rows;
* distillation from a teacher's top logits beside the labels' cross entropy, and its gradient over
  the kept rows.

``run`` computes an operator in elementary torch operations, or, with ``own`` set, through
:mod:`centrifuge_b200.ops`.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the up projection of a unit-test model over two sequences of 128 tokens: launch latency
        {"name": "linear fwd small", "op": "linear_fwd", "rows": 256, "inner": 256, "cols": 512,
         "dtype": "bf16", "act": "gelu", "bias": True, "resid": False, "z": True},
        # the up projection of a micro-batch at TinyLlama's widths, 8 x 2048 tokens
        {"name": "linear fwd 8x2048 up", "op": "linear_fwd", "rows": 16384, "inner": 2048,
         "cols": 5632, "dtype": "bf16", "act": "gelu_tanh", "bias": True, "resid": False, "z": True},
        # few kept rows of an odd batch, widths that are no multiples of a tile
        {"name": "linear dgrad odd", "op": "linear_dgrad", "tokens": 399, "rows": 200,
         "inner": 1000, "cols": 2730, "dtype": "fp16", "act": "silu"},
        # half of a micro-batch kept, through the down projection into the activation below
        {"name": "linear dgrad 8x2048 kept", "op": "linear_dgrad", "tokens": 16384, "rows": 8192,
         "inner": 2048, "cols": 5632, "dtype": "bf16", "act": "gelu_tanh"},
        # the up projection's weight and bias over the kept half of a micro-batch
        {"name": "linear wgrad 8x2048 kept", "op": "linear_wgrad", "rows": 8192, "inner": 2048,
         "cols": 5632, "dtype": "bf16", "bias": True},
        # a micro-batch at TinyLlama's width
        {"name": "layernorm fwd 8x2048", "op": "ln_fwd", "rows": 16384, "hidden": 2048,
         "dtype": "bf16", "stream": "bf16", "bias": True},
        # few kept rows of an odd batch at a width that is no power of two
        {"name": "layernorm bwd small", "op": "ln_bwd", "tokens": 399, "rows": 200, "hidden": 1000,
         "dtype": "fp16", "stream": "fp16", "bias": True, "dres": True},
        # half of two sequences of 8192 at Llama-3-8B's width, the residual stream in fp32
        {"name": "layernorm bwd wide fp32 stream", "op": "ln_bwd", "tokens": 16384, "rows": 8190,
         "hidden": 4096, "dtype": "bf16", "stream": "fp32", "bias": True, "dres": True},
        # a unit-test model's logits, eight of a teacher's
        {"name": "distill fwd small", "op": "distill_fwd", "rows": 256, "vocab": 1024, "top": 8,
         "dtype": "bf16", "temperature": 1.0, "tail": False, "labels": False, "ragged": 0.0},
        # a micro-batch of TinyLlama's logits, 32 of a teacher's and the mass of its tail, with labels
        {"name": "distill fwd 8x2048", "op": "distill_fwd", "rows": 16384, "vocab": 32000, "top": 32,
         "dtype": "bf16", "temperature": 2.0, "tail": True, "labels": True, "ragged": 0.0},
        # its gradient over the kept half of the tokens
        {"name": "distill bwd 8x2048 kept", "op": "distill_bwd", "tokens": 16384, "rows": 8192,
         "vocab": 32000, "top": 32, "dtype": "bf16", "temperature": 2.0, "tail": True,
         "labels": True, "ragged": 0.0},
        # fp32 logits of Llama-3's vocabulary, an odd number of rows, lists of different lengths
        {"name": "distill bwd wide fp32", "op": "distill_bwd", "tokens": 2048, "rows": 1021,
         "vocab": 128256, "top": 64, "dtype": "fp32", "temperature": 1.0, "tail": False,
         "labels": True, "ragged": 0.3},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, of=8):
    n = _log(rng, lo, hi)
    return max(of, n // of * of) if rng.random() < 0.7 else n  # most are whole vectors, some odd


def draw(rng):
    op = rng.choice(["linear_fwd", "linear_dgrad", "linear_wgrad", "ln_fwd", "ln_bwd",
                     "distill_fwd", "distill_bwd"])
    tokens = _log(rng, 1, 16384)
    rows = max(1, int(tokens * rng.uniform(0.3, 1.0)))
    if op.startswith("linear"):
        c = {"op": op, "inner": _width(rng, 32, 8192), "cols": _width(rng, 32, 8192),
             "dtype": rng.choice(["bf16", "bf16", "fp16"])}
        limit = 16384 * 2048 * 5632 // (c["inner"] * c["cols"])  # the largest listed product
        c["rows"] = min(rows, limit)
        if op == "linear_wgrad":
            return {**c, "bias": rng.random() < 0.8}
        if op == "linear_dgrad":
            return {**c, "tokens": max(c["rows"], min(tokens, 2 * limit)),
                    "act": rng.choice(ACTS[1:])}
        return {**c, "act": rng.choice(ACTS), "bias": rng.random() < 0.8,
                "resid": rng.random() < 0.4, "z": rng.random() < 0.5}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op.startswith("ln"):
        c = {"op": op, "hidden": _width(rng, 96, 4096), "dtype": dtype,
             "stream": rng.choice([dtype, "fp32"]), "bias": rng.random() < 0.8}
        if op == "ln_fwd":
            return {**c, "rows": tokens}
        return {**c, "tokens": tokens, "rows": rows, "dres": rng.random() < 0.7}
    vocab = _width(rng, 300, 128256)
    c = {"op": op, "vocab": vocab, "top": min(vocab, _log(rng, 1, 128)), "dtype": dtype,
         "temperature": rng.choice([1.0, 1.0, 2.0, 0.7]), "tail": rng.random() < 0.5,
         "labels": rng.random() < 0.6, "ragged": rng.choice([0.0, 0.0, 0.3])}
    limit = 16384 * 32000 * 2 // (SIZE[dtype] * vocab)  # the largest listed logits
    if op == "distill_fwd":
        return {**c, "rows": max(1, min(tokens, limit))}
    return {**c, "tokens": max(1, min(tokens, limit)), "rows": max(1, min(rows, limit // 2))}


def work(case):
    c, op = case, case["op"]
    e = SIZE[c["dtype"]]
    if op.startswith("linear"):
        r, k, n = c["rows"], c["inner"], c["cols"]
        flops = 2 * r * k * n
        if op == "linear_fwd":
            b = e * (r * k + n * k + r * n * (1 + c["resid"] + c["z"]) + (n if c["bias"] else 0))
        elif op == "linear_dgrad":  # dy, w, z at the kept rows, their ids; dz
            b = e * (r * k + n * k + 2 * r * n) + 4 * r
        else:  # dy, x; dw and dbias in fp32
            b = e * (r * k + r * n) + 4 * (n * k + (n if c["bias"] else 0))
        return {"bytes": b, "flops": flops}
    if op.startswith("ln"):
        n, x = c["rows"] * c["hidden"], SIZE[c["stream"]]
        if op == "ln_fwd":  # x; y and the two statistics
            return {"bytes": n * (x + e) + 8 * c["rows"], "flops": 8 * n}
        # dy, x, dres, statistics and ids of the kept rows; dx
        return {"bytes": n * (e + 2 * x + (x if c["dres"] else 0)) + 12 * c["rows"],
                "flops": 14 * n}
    n, lists = c["rows"] * c["vocab"], 8 * c["rows"] * c["top"]
    if op == "distill_fwd":
        return {"bytes": n * e + lists + 32 * c["rows"], "flops": 6 * n}
    return {"bytes": 2 * n * e + lists + 40 * c["rows"], "flops": 8 * n}


# ---------------------------------------------------------------- inputs
def _kept(g, tokens, rows):
    return torch.randperm(tokens, generator=g, device="cuda")[:rows].sort().values.int()


def _normal(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def _student(g, T, V, dt):
    """Logits of a language model: noise, and some tokens of each row far above it."""
    n = min(V, 64)
    z = torch.randn(T, V, generator=g, device="cuda", dtype=dt) * 1.5
    rank = torch.arange(n, device="cuda")
    at = (torch.randint(0, V, (T, 1), generator=g, device="cuda") + rank * (V // n)) % V
    above = 16.0 - 2.0 * (rank + 1).log()
    above = above * (0.6 + 0.4 * torch.rand(T, 1, generator=g, device="cuda"))
    return z.scatter_(1, at, (above + _normal(g, T, n)).to(dt))


def _teacher(g, logits, c):
    """A teacher that mostly agrees with the student: its top logits, their ids (-1 behind the end
    of a short list) and the log of its whole softmax's sum."""
    T, V = logits.shape
    ids = torch.empty(T, c["top"], dtype=torch.int32, device="cuda")
    top = torch.empty(T, c["top"], device="cuda")
    lse = torch.empty(T, device="cuda")
    step = max(1, (1 << 26) // V)
    for i in range(0, T, step):
        t = logits[i:i + step].float()
        t += _normal(g, *t.shape, scale=0.8)
        v, at = t.topk(c["top"], dim=1)
        top[i:i + step], ids[i:i + step] = v, at
        lse[i:i + step] = (t / c["temperature"]).logsumexp(1)
    if c["ragged"]:
        length = torch.randint(0, c["top"] + 1, (T, 1), generator=g, device="cuda")
        short = torch.rand(T, 1, generator=g, device="cuda") < c["ragged"]
        ids[short & (torch.arange(c["top"], device="cuda") >= length)] = -1
    return ids, top, lse


def prepare(case, seed):
    c, op = case, case["op"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[c["dtype"]]
    s = {"op": op}
    if op.startswith("linear"):
        r, k, n = c["rows"], c["inner"], c["cols"]
        if op == "linear_wgrad":
            s.update(dy=_normal(g, r, n, dtype=dt), x=_normal(g, r, k, dtype=dt),
                     dw=torch.empty(n, k, device="cuda"),
                     dbias=torch.empty(n, device="cuda") if c["bias"] else None)
            return s
        # a weight [outputs, inputs]: the gradient comes in at its outputs
        shape = (n, k) if op == "linear_fwd" else (k, n)
        s.update(act=c["act"], w=_normal(g, *shape, dtype=dt, scale=1.0 / math.sqrt(k)))
        if op == "linear_fwd":
            s.update(x=_normal(g, r, k, dtype=dt),
                     bias=_normal(g, n, dtype=dt, scale=0.5) if c["bias"] else None,
                     resid=_normal(g, r, n, dtype=dt, scale=2.0) if c["resid"] else None,
                     save=c["z"])
        else:
            s.update(dy=_normal(g, r, k, dtype=dt), z=_normal(g, c["tokens"], n, dtype=dt),
                     kept=_kept(g, c["tokens"], r))
    elif op.startswith("ln"):
        H, xt = c["hidden"], TYPES[c["stream"]]
        T = c["rows"] if op == "ln_fwd" else c["tokens"]
        s.update(x=_normal(g, T, H, dtype=xt, scale=2.0, shift=0.3),
                 w=_normal(g, H, dtype=dt, scale=0.1, shift=1.0),
                 b=_normal(g, H, dtype=dt, scale=0.1) if c["bias"] else None)
        if op == "ln_bwd":
            _, s["mean"], s["rstd"] = _ln_fwd(s)
            s.update(dy=_normal(g, c["rows"], H, dtype=dt), kept=_kept(g, T, c["rows"]),
                     dres=_normal(g, c["rows"], H, dtype=xt) if c["dres"] else None,
                     dw=torch.empty(H, device="cuda"),
                     db=torch.empty(H, device="cuda") if c["bias"] else None)
    else:
        T = c["rows"] if op == "distill_fwd" else c["tokens"]
        s.update(logits=_student(g, T, c["vocab"], dt),
                 temperature=c["temperature"], labels=None)
        s["ids"], s["top"], lse = _teacher(g, s["logits"], c)
        s["top_lse"] = lse if c["tail"] else None
        if c["labels"]:
            labels = torch.randint(0, c["vocab"], (T,), generator=g, device="cuda")
            best = torch.rand(T, generator=g, device="cuda") < 0.5  # often what the teacher names
            labels = torch.where(best & (s["ids"][:, 0] >= 0), s["ids"][:, 0].long(), labels)
            pad = torch.rand(T, generator=g, device="cuda") < 0.05
            s["labels"] = torch.where(pad, torch.full_like(labels, -1), labels)
        if op == "distill_bwd":
            _, _, s["lse"], s["stats"] = _distill_fwd(s)
            s["kept"] = _kept(g, T, c["rows"])
            s["dkd"] = torch.rand(c["rows"], generator=g, device="cuda") / c["rows"]
            s["dce"] = None
            if c["labels"]:
                s["dce"] = torch.rand(c["rows"], generator=g, device="cuda") / c["rows"]
    return s


# ---------------------------------------------------------------- plain forms
def _act(z, act):
    if act == "relu":
        return z.clamp(min=0.0)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * torch.erfc(z * -math.sqrt(0.5))
    if act == "gelu_tanh":
        u = math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)
        return z / (1.0 + torch.exp(-2.0 * u))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0.0).float()
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return p * (1.0 + z * (1.0 - p))
    if act == "gelu":
        density = torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
        return 0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * density
    k = math.sqrt(2.0 / math.pi)
    p = 1.0 / (1.0 + torch.exp(-2.0 * k * (z + 0.044715 * z * z * z)))
    return p + z * p * (1.0 - p) * 2.0 * k * (1.0 + 3 * 0.044715 * z * z)


def _linear_fwd(s):
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, s["act"])
    if s["resid"] is not None:
        y = y + s["resid"].float()
    return y.to(s["x"].dtype), z.to(s["x"].dtype) if s["save"] else None


def _linear_dgrad(s):
    dh = s["dy"].float() @ s["w"].float()
    return (dh * _act_grad(s["z"][s["kept"].long()].float(), s["act"])).to(s["dy"].dtype)


def _linear_wgrad(s):
    dy = s["dy"].float()
    return dy.t() @ s["x"].float(), dy.sum(0) if s["dbias"] is not None else None


def _ln_fwd(s):
    x = s["x"].float()
    mean = x.mean(-1)
    d = x - mean[:, None]
    rstd = torch.rsqrt(d.square().mean(-1) + EPS)
    y = d * rstd[:, None] * s["w"].float()
    if s["b"] is not None:
        y = y + s["b"].float()
    return y.to(s["w"].dtype), mean, rstd


def _ln_bwd(s):
    at = s["kept"].long()
    r = s["rstd"][at][:, None]
    n = (s["x"][at].float() - s["mean"][at][:, None]) * r
    dy = s["dy"].float()
    a = dy * s["w"].float()
    dx = r * (a - a.mean(-1, keepdim=True) - n * (a * n).mean(-1, keepdim=True))
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    return dx.to(s["x"].dtype), (dy * n).sum(0), dy.sum(0) if s["db"] is not None else None


def _lse(x):
    """In 64 bits from the sum on: a divergence is the small difference of two of these."""
    m = x.amax(-1)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)  # of nothing: -inf
    return m.double() + torch.exp(x - m[:, None]).sum(-1).double().log()


def _picked(x, ids, none):
    """x at the ids of each row's list, `none` behind a list's end."""
    v = x.gather(1, ids.long().clamp(min=0))
    return torch.where(ids >= 0, v, torch.full_like(v, none))


def _share(s):
    """The teacher's shares of its listed tokens and the log of what divides them, in 64 bits: what
    is left of the whole is small beside it."""
    ids, top = s["ids"], s["top"].double() / s["temperature"]
    top = torch.where(ids >= 0, top, torch.full_like(top, -math.inf))
    if s["top_lse"] is not None:
        norm = s["top_lse"].double()
    else:
        norm = _lse(top)
    p = torch.where(ids >= 0, torch.exp(top - norm[:, None]), torch.zeros_like(top))
    return p, top, norm


def _distill_fwd(s):
    z, ids, labels = s["logits"].float(), s["ids"], s["labels"]
    x = z / s["temperature"]
    lse = _lse(x)
    p, top, norm = _share(s)
    q = _picked(x, ids, 0.0) - lse[:, None]
    kd = torch.where(p > 0, p * (top - norm[:, None] - q), torch.zeros_like(p)).sum(-1)
    base, coef = lse, torch.ones_like(lse)
    if s["top_lse"] is not None:
        out = torch.cat([x, x.new_zeros(x.shape[0], 1)], 1)
        out.scatter_(1, torch.where(ids >= 0, ids, x.shape[1]).long(), -math.inf)
        base = _lse(out[:, :-1])
        left = (1.0 - p.sum(-1)).clamp(min=0.0)
        some = (left > 0) & (base > -math.inf)
        log_q = base - lse
        kd = kd + torch.where(some, left * (left.log() - log_q), torch.zeros_like(left))
        coef = torch.where(base > -math.inf, log_q.exp() - left, torch.zeros_like(left))
    none = (ids < 0).all(-1)
    if s["top_lse"] is None:  # nothing to learn from an empty list
        kd = torch.where(none, torch.zeros_like(kd), kd)
        coef = torch.where(none, torch.zeros_like(coef), coef)
    kd, stats = kd.float(), torch.stack([lse, base, coef, norm], 1).float()
    if labels is None:
        return kd, None, None, stats
    full = lse if s["temperature"] == 1.0 else _lse(z)
    ce = full - z.gather(1, labels.clamp(min=0)[:, None])[:, 0]
    return kd, torch.where(labels >= 0, ce, torch.zeros_like(ce)).float(), full.float(), stats


def _distill_bwd(s):
    at = s["kept"].long()
    z, ids, st = s["logits"][at].float(), s["ids"][at], s["stats"][at]
    part = {**s, "ids": ids, "top": s["top"][at],
            "top_lse": None if s["top_lse"] is None else s["top_lse"][at]}
    p, _, _ = _share(part)
    V = z.shape[1]
    x = torch.cat([z / s["temperature"], z.new_zeros(z.shape[0], 1)], 1)
    g = torch.exp(x - st[:, 1:2]) * st[:, 2:3]
    col = torch.where(ids >= 0, ids, V).long()
    g.scatter_(1, col, torch.exp(x.gather(1, col) - st[:, 0:1]))
    g.scatter_add_(1, col, -p.float())
    g = g[:, :V] * (s["dkd"] / s["temperature"])[:, None]
    if s["labels"] is not None:
        labels = s["labels"][at]
        dce = torch.where(labels >= 0, s["dce"], torch.zeros_like(s["dce"]))[:, None]
        g = g + torch.exp(z - s["lse"][at][:, None]) * dce
        g.scatter_add_(1, labels.clamp(min=0)[:, None], -dce)
    return g.to(s["logits"].dtype)


# ---------------------------------------------------------------- one pass
def run(s):
    op = s["op"]
    if own:
        from centrifuge_b200.ops import fused, gemm
    if op == "linear_fwd":
        if not own:
            return _linear_fwd(s)
        z = None
        if s["save"]:
            z = torch.empty(s["x"].shape[0], s["w"].shape[0], dtype=s["x"].dtype, device="cuda")
        y = gemm.linear_act_fwd(s["x"], s["w"], s["bias"], act=s["act"], resid=s["resid"], z=z)
        return y, z
    if op == "linear_dgrad":
        if not own:
            return _linear_dgrad(s)
        return gemm.linear_act_dgrad(s["dy"], s["w"], s["z"], s["act"], z_rows=s["kept"])
    if op == "linear_wgrad":
        if not own:
            return _linear_wgrad(s)
        gemm.linear_bias_wgrad(s["dy"], s["x"], s["dw"], s["dbias"], accumulate=False)
        return s["dw"], s["dbias"]
    if op == "ln_fwd":
        if not own:
            return _ln_fwd(s)
        return fused.layernorm_fwd(s["x"], s["w"], s["b"], EPS)
    if op == "ln_bwd":
        if not own:
            return _ln_bwd(s)
        dx = fused.layernorm_bwd(s["dy"], s["x"], s["mean"], s["rstd"], s["w"], s["dw"], s["db"],
                                 rows=s["kept"], dres=s["dres"], accumulate=False)
        return dx, s["dw"], s["db"]
    if op == "distill_fwd":
        if not own:
            return _distill_fwd(s)
        return fused.distill_fwd(s["logits"], s["ids"], s["top"], s["temperature"],
                                 top_lse=s["top_lse"], labels=s["labels"])
    if not own:
        return _distill_bwd(s)
    return fused.distill_bwd(s["logits"], s["ids"], s["top"], s["stats"], s["dkd"],
                             s["temperature"], labels=s["labels"], lse=s["lse"], dce=s["dce"],
                             rows=s["kept"])


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    c, op = case, case["op"]
    s = prepare(case, seed)
    if op.startswith("linear"):
        return _exact_linear(c, s)
    if op == "ln_fwd":
        var, mean = torch.var_mean(s["x"].double(), dim=1, correction=0)
        rstd = (var + EPS).pow(-0.5)
        y = torch.einsum("th,t,h->th", s["x"].double() - mean.unsqueeze(1), rstd, s["w"].double())
        return y if s["b"] is None else y + s["b"].double(), mean, rstd
    if op == "ln_bwd":
        # the normalised row is its projection off the ones, scaled: so is its gradient
        k, H = s["kept"].long(), c["hidden"]
        r = s["rstd"].index_select(0, k).double().unsqueeze(1)
        n = torch.addcmul(-s["mean"].index_select(0, k).double().unsqueeze(1) * r,
                          s["x"].index_select(0, k).double(), r)
        dy = s["dy"].double()
        v = torch.einsum("th,h->th", dy, s["w"].double())
        along = torch.einsum("th,th->t", v, n).unsqueeze(1) / H
        dx = (v - v.sum(1, keepdim=True) / H - n * along) * r
        if s["dres"] is not None:
            dx += s["dres"].double()
        ones = torch.ones(c["rows"], dtype=torch.float64, device="cuda")
        return dx, torch.einsum("th,th->h", dy, n), ones @ dy if c["bias"] else None
    at = s["kept"].long() if op == "distill_bwd" else None
    parts, step = [], max(1, (1 << 27) // c["vocab"])
    for i in range(0, c["rows"], step):
        rows = torch.arange(i, min(i + step, c["rows"]), device="cuda")
        parts.append(_exact_distill(c, s, rows if at is None else at[rows], rows))
    if op == "distill_bwd":
        return torch.cat(parts)
    return tuple(None if x[0] is None else torch.cat(x) for x in zip(*parts))


def _exact_linear(c, s):
    if c["op"] == "linear_wgrad":
        dy = s["dy"].double()
        ones = torch.ones(c["rows"], dtype=torch.float64, device="cuda")
        return torch.einsum("rn,rk->nk", dy, s["x"].double()), ones @ dy if c["bias"] else None
    if c["op"] == "linear_fwd":
        z = torch.einsum("rk,nk->rn", s["x"].double(), s["w"].double())
        if s["bias"] is not None:
            z += s["bias"].double()
        y = z * _slope(z, c["act"]) if c["act"] != "none" else z
        return y if s["resid"] is None else y + s["resid"].double(), z if c["z"] else None
    dh = torch.einsum("rk,kn->rn", s["dy"].double(), s["w"].double())
    z = s["z"].index_select(0, s["kept"].long()).double()
    if c["act"] == "relu":
        return torch.where(z > 0, dh, torch.zeros_like(dh))
    with torch.enable_grad():
        z.requires_grad_()
        return torch.autograd.grad(z * _slope(z, c["act"]), z, dh)[0]


def _slope(z, act):
    """What an activation multiplies its argument by."""
    if act == "relu":
        return (z > 0).double()
    if act == "silu":
        return torch.sigmoid(z)
    if act == "gelu":
        return torch.special.ndtr(z)
    return torch.sigmoid(1.5957691216057308 * z + 0.07135481282922578 * z.pow(3))


def _exact_distill(c, s, at, rows):
    """Both losses of the rows `at` (and their gradient for the weights `rows`) from a dense
    distribution of the teacher over the listed tokens and one more for all the others."""
    V, tau = c["vocab"], c["temperature"]
    z, ids = s["logits"][at].double(), s["ids"][at].long()
    logq = torch.log_softmax(z / tau, 1)
    ok = ids >= 0
    top = (s["top"][at].double() / tau).masked_fill(~ok, -math.inf)
    norm = s["top_lse"][at].double() if c["tail"] else top.logsumexp(1)
    logp = top - norm.unsqueeze(1)
    p = logp.exp().masked_fill(~ok, 0.0)
    dense = z.new_zeros(z.shape[0], V + 1)
    dense.scatter_add_(1, ids.masked_fill(~ok, V), p)
    dense = dense[:, :V]
    inside = torch.zeros(z.shape[0], V + 1, dtype=torch.bool, device="cuda")
    inside.scatter_(1, ids.masked_fill(~ok, V), True)
    inside = inside[:, :V]
    picked = logq.gather(1, ids.clamp(min=0))
    kd = (p * (logp - picked)).masked_fill(~ok | (p == 0), 0.0).sum(1)
    lse = (z / tau).logsumexp(1)
    empty = ~ok.any(1)
    if c["tail"]:
        tail = (1.0 - p.sum(1)).clamp(min=0.0)
        log_rest = logq.masked_fill(inside, -math.inf).logsumexp(1)
        some = (tail > 0) & (log_rest > -math.inf)
        kd = kd + (tail * (tail.log() - log_rest)).masked_fill(~some, 0.0)
        base = lse + log_rest
        coef = (log_rest.exp() - tail).masked_fill(log_rest == -math.inf, 0.0)
    else:
        base, coef = lse, (~empty).double()
        kd = kd.masked_fill(empty, 0.0)
    lab = s["labels"][at] if c["labels"] else None
    if c["op"] == "distill_fwd":
        stats = torch.stack([lse, base, coef, norm], 1)
        if lab is None:
            return kd, None, None, stats
        ce = -torch.log_softmax(z, 1).gather(1, lab.clamp(min=0).unsqueeze(1)).squeeze(1)
        return kd, ce.masked_fill(lab < 0, 0.0), z.logsumexp(1), stats
    q = logq.exp()
    if c["tail"]:
        other = q - tail.unsqueeze(1) * torch.exp(logq - log_rest.unsqueeze(1))
        g = torch.where(inside, q - dense, other)
    else:
        g = (q - dense) * coef.unsqueeze(1)
    g *= s["dkd"][rows].double().unsqueeze(1) / tau
    if lab is not None:
        soft = torch.softmax(z, 1)
        soft.scatter_add_(1, lab.clamp(min=0).unsqueeze(1), -torch.ones_like(soft[:, :1]))
        g += soft * s["dce"][rows].double().masked_fill(lab < 0, 0.0).unsqueeze(1)
    return g
