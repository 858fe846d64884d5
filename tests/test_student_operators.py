"""Linear layers with bias, activation and residual, layer norm, and distillation from a teacher's top
logits, against their formulas in 64 bits.

Tolerances are bounds on the rounding errors of the arithmetic, element by element: u = 2^-24 for an
fp32 operation, k u sum|x| for a sum whose longest chain has k additions (2 k u where the tensor cores
add, which need not round to nearest), and half a step of the output's type for its one rounding.
"""
import math

import pytest
import torch

from centrifuge_b200.ops import fused, gemm
from centrifuge_b200.ops import reference as ref

U = 2.0 ** -24
EPS = 1e-5
CPU_GPU = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
BF, HF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
ACTS = gemm.ACTIVATIONS


def close(got, want, tol, what):
    """|got - want| <= tol everywhere, after the rounding to got's type."""
    info = torch.finfo(got.dtype)
    tiny = info.smallest_normal * info.eps / 2
    bound = tol + info.eps / 2 * (want.abs() + tol) + tiny
    off = (got.double() - want).abs()
    bad = ~((off <= bound) | ((got.double() == want) & want.isinf()))
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, at {i}: got "
                             f"{float(got[i])}, want {float(want[i])}, bound {float(bound[i])}")


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def rand(g, *shape, dtype=F32, scale=1.0, shift=0.0, pad=0, skew=0):
    """Normal values; the rows `pad` elements longer than asked for and begun at element `skew`."""
    if len(shape) == 2 and (pad or skew):
        t = torch.randn(shape[0], shape[1] + pad + skew, generator=g, device=g.device)
        return (t * scale + shift).to(dtype)[:, skew:skew + shape[1]]
    return (torch.randn(*shape, generator=g, device=g.device) * scale + shift).to(dtype)


def empty(dev, rows, cols, dtype, pad=0, skew=0):
    """A buffer of 9s around the [rows, cols] that a call writes, and that view of it."""
    t = torch.full((rows, cols + pad + skew), 9.0, dtype=dtype, device=dev)
    return t, t[:, skew:skew + cols]


def untouched(buf, cols, skew):
    return bool((buf[:, :skew] == 9.0).all()) and bool((buf[:, skew + cols:] == 9.0).all())


def kept(g, T, R):
    return torch.randperm(T, generator=g, device=g.device)[:R].sort().values.int()


# ---------------------------------------------------------------- linear layers
def act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * torch.erfc(-z * math.sqrt(0.5)) / 2
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def slope64(z, act):
    z = z.clone().requires_grad_()
    if act == "relu":
        return (z > 0).double()
    return torch.autograd.grad(act64(z, act).sum(), z)[0]


# The activations: exponentials of arguments up to 60 that are rounded once or twice (2 * 60 ln 2 u),
# the hardware's exponential and reciprocal (2^-22 each), a fit with 1.2e-6 (gelu): below 2^-16 in all.
ACT_REL = 2.0 ** -16


def act_tol(z, act):
    return 0.0 if act in ("none", "relu") else ACT_REL * act64(z, act).abs()


def slope_tol(z, act):
    """Both terms of the slope with the same relative error, and 1 - p of p near one."""
    if act in ("none", "relu"):
        return torch.zeros_like(z)
    if act == "gelu":
        return ACT_REL * (torch.erfc(-z * math.sqrt(0.5)) / 2 + z.abs() * torch.exp(-z * z / 2) * 0.4)
    u = z if act == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    du = torch.ones_like(z) if act == "silu" else 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z * z)
    p = torch.sigmoid(u)
    return ACT_REL * p * (1 + z.abs() * (1 - p) * du) + 4 * U * p * z.abs() * du


LINEAR = [
    (256, 256, 512), (1, 64, 32), (1, 8, 1), (3, 1, 5), (130, 72, 200), (257, 100, 130), (64, 33, 40),
    (300, 130, 257), (128, 64, 64), (129, 65, 65), (5, 2048, 96), (700, 40, 1000), (17, 1000, 2730),
    (2, 7, 300), (513, 264, 520),
]


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("T,K,N", LINEAR)
@pytest.mark.parametrize("act,bias,resid,save", [
    ("none", True, False, False), ("gelu", True, True, True), ("gelu_tanh", False, True, True),
    ("silu", True, False, True), ("relu", True, True, False), ("none", False, True, True)])
@pytest.mark.parametrize("dtype,pad,skew", [(BF, 0, 0), (HF, 0, 0), (BF, 8, 0), (HF, 5, 1)])
def test_linear_act_fwd(dev, T, K, N, act, bias, resid, save, dtype, pad, skew):
    g = gen(dev, T + K + N)
    x = rand(g, T, K, dtype=dtype, pad=pad, skew=skew)
    w = rand(g, N, K, dtype=dtype, scale=2.0 / math.sqrt(K), pad=pad, skew=skew)
    b = rand(g, N, dtype=dtype) if bias else None
    r = rand(g, T, N, dtype=dtype, pad=pad, skew=skew) if resid else None
    z_buf, z = empty(dev, T, N, dtype, pad, skew)
    o_buf, o = empty(dev, T, N, dtype, pad, skew)
    got = gemm.linear_act_fwd(x, w, b, act=act, resid=r, out=o if pad else None,
                              z=z if save else None)
    assert got.dtype == dtype and got.shape == (T, N) and (not pad or got is o)
    want_z = x.double() @ w.double().t()
    tol = 2 * (K + 2) * U * (x.double().abs() @ w.double().abs().t())
    if bias:
        want_z = want_z + b.double()
        tol = tol + U * want_z.abs()
    want = act64(want_z, act)
    tol_y = 1.13 * tol + act_tol(want_z, act)
    if resid:
        want = want + r.double()
        tol_y = tol_y + 2 * U * (want.abs() + r.double().abs())
    close(got, want, tol_y, "y")
    if save:
        close(z, want_z, tol, "z")
        assert untouched(z_buf, N, skew)
    if pad:
        assert untouched(o_buf, N, skew)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("R,K,N", LINEAR)
@pytest.mark.parametrize("act,dtype,pad,skew,some", [
    ("gelu", BF, 0, 0, True), ("gelu_tanh", HF, 0, 0, False), ("silu", BF, 8, 0, True),
    ("relu", HF, 5, 1, True), ("none", BF, 5, 1, False), ("silu", HF, 0, 0, False)])
def test_linear_act_dgrad(dev, R, K, N, act, dtype, pad, skew, some):
    g = gen(dev, R + 2 * K + N)
    T = 2 * R + 1 if some else R
    dy = rand(g, R, K, dtype=dtype, pad=pad, skew=skew)
    w = rand(g, K, N, dtype=dtype, scale=1.0 / math.sqrt(K), pad=pad, skew=skew)
    z = rand(g, T, N, dtype=dtype, scale=2.0, pad=pad, skew=skew)
    rows = kept(g, T, R) if some else None
    buf, o = empty(dev, R, N, dtype, pad, skew)
    got = gemm.linear_act_dgrad(dy, w, z, act, z_rows=rows, out=o if pad else None)
    assert got.dtype == dtype and got.shape == (R, N) and (not pad or got is o)
    zk = (z if rows is None else z[rows.long()]).double()
    dh, s = dy.double() @ w.double(), slope64(zk, act)
    tol = 2 * (K + 2) * U * (dy.double().abs() @ w.double().abs())
    close(got, dh * s, 1.13 * tol + (dh.abs() + tol) * slope_tol(zk, act) + 2 * U * (dh * s).abs(), "dz")
    assert not pad or untouched(buf, N, skew)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("N,K,R", [(b, a, c) for a, b, c in LINEAR] + [(64, 96, 0), (40, 300, 1500)])
@pytest.mark.parametrize("dtype,bias,accumulate,pad,skew", [
    (BF, True, True, 0, 0), (HF, True, False, 0, 0), (BF, False, False, 8, 0), (HF, True, True, 5, 1)])
def test_linear_bias_wgrad(dev, N, K, R, dtype, bias, accumulate, pad, skew):
    g = gen(dev, R + K + 3 * N)
    dy = rand(g, R, N, dtype=dtype, pad=pad, skew=skew)
    x = rand(g, R, K, dtype=dtype, pad=pad, skew=skew)
    buf, dw = empty(dev, N, K, F32, pad, skew)
    dw.copy_(rand(g, N, K))
    db = rand(g, N) if bias else None
    before, before_b = dw.clone(), None if db is None else db.clone()
    assert gemm.linear_bias_wgrad(dy, x, dw, db, accumulate=accumulate) is dw
    want = dy.double().t() @ x.double()
    tol = 2 * (R + 2) * U * (dy.double().abs().t() @ x.double().abs())
    if accumulate:
        want = want + before.double()
        tol = tol + U * want.abs()
    close(dw, want, tol, "dw")
    assert untouched(buf, K, skew)
    if bias:
        want = dy.double().sum(0)
        tol = (R + 2) * U * dy.double().abs().sum(0)
        if accumulate:
            want = want + before_b.double()
            tol = tol + U * want.abs()
        close(db, want, tol, "dbias")


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,kind", [
    (4096, 5632, 512, "fwd"), (2100, 2049, 264, "fwd"), (2048, 5632, 512, "dgrad"),
    (1500, 5000, 136, "dgrad"), (5632, 2048, 1000, "wgrad"), (3000, 2500, 70, "wgrad"),
    (20000, 300, 64, "fwd")])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_over_many_tiles(M, N, K, kind, dtype):
    """More tiles than SMs: each block takes several, with both accumulators in turn."""
    g = gen("cuda", M + N + K)
    if kind == "fwd":
        x, w = rand(g, M, K, dtype=dtype), rand(g, N, K, dtype=dtype, scale=K ** -0.5)
        got = gemm.linear_act_fwd(x, w)
        want, mass = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    elif kind == "dgrad":
        dy, w = rand(g, M, K, dtype=dtype), rand(g, K, N, dtype=dtype, scale=K ** -0.5)
        z = rand(g, M, N, dtype=dtype)
        got = gemm.linear_act_dgrad(dy, w, z, "relu")
        live = (z > 0).double()
        want, mass = dy.double() @ w.double() * live, dy.double().abs() @ w.double().abs()
    else:
        dy, x = rand(g, K, M, dtype=dtype), rand(g, K, N, dtype=dtype)
        got = torch.empty(M, N, device="cuda")
        runs = []
        for _ in range(2):
            gemm.linear_bias_wgrad(dy, x, got, accumulate=False)
            runs.append(got.clone())
        assert torch.equal(*runs)  # a fixed order
        want, mass = dy.double().t() @ x.double(), dy.double().abs().t() @ x.double().abs()
    close(got, want, 2 * (K + 2) * U * mass, kind)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_activations_over_their_range(dev, act, dtype):
    """Large and small arguments through an identity weight, in both directions."""
    v = torch.cat([torch.linspace(-12, 12, 1531), torch.tensor([0.0, -0.0, 1e-4, -1e-4, 30.0, -30.0]),
                   torch.tensor([88.0, -88.0, 200.0, -200.0, 6e4, -6e4])])
    v = torch.cat([v, v.new_zeros(-v.numel() % 32)]).to(dtype).to(dev).view(-1, 32)
    eye = torch.eye(32, dtype=dtype, device=dev)
    z = torch.empty_like(v)
    y = gemm.linear_act_fwd(v, eye, act=act, z=z)
    assert torch.equal(z, v)
    # an exponential below the smallest normal fp32 number may come out as zero; |z| du at most
    # multiplies it (du: the slope of what gelu_tanh takes the exponential of, for the others smaller)
    du = 1.6 * (1 + 0.135 * v.double() ** 2)
    flush = 2.0 ** -126 * (1 + v.double().abs() * (1 + du))
    close(y, act64(v.double(), act), act_tol(v.double(), act) + flush, "y")
    one = torch.ones(v.shape[0], 1, dtype=dtype, device=dev)
    dz = gemm.linear_act_dgrad(one, torch.ones(1, 32, dtype=dtype, device=dev), v, act)
    d = v.double()
    close(dz, slope64(d, act), slope_tol(d, act) + flush, "slope")


@pytest.mark.parametrize("dev", CPU_GPU)
def test_linear_odd_values(dev):
    """A NaN or infinity stays in its row (forward, dgrad) or column (wgrad)."""
    g = gen(dev, 3)
    x, w = rand(g, 70, 48, dtype=BF), rand(g, 40, 48, dtype=BF)
    x[5, 3], x[9, 0] = float("nan"), float("inf")
    for act in ACTS:
        y = gemm.linear_act_fwd(x, w, act=act)
        assert bool(y[5].isnan().all()) and not bool(y[9].isfinite().logical_and(y[9] != 0).any())
        y[5], y[9] = 0.0, 0.0
        assert bool(y.isfinite().all())
    z = rand(g, 70, 48, dtype=BF)
    z[2, 7] = float("nan")
    dz = gemm.linear_act_dgrad(torch.ones(70, 40, dtype=BF, device=dev), w, z, "gelu")
    assert bool(dz[2, 7].isnan()) and int(dz.isfinite().logical_not().sum()) == 1
    dw, db = torch.empty(48, 40, device=dev), torch.empty(48, device=dev)
    gemm.linear_bias_wgrad(x, rand(g, 70, 40, dtype=BF), dw, db, accumulate=False)
    assert bool(dw[3].isnan().all()) and bool(db[3].isnan()) and bool(db[0].isinf())
    assert bool(dw[4:].isfinite().all()) and bool(db[4:].isfinite().all())


@pytest.mark.parametrize("dev", CPU_GPU)
def test_linear_in_place(dev):
    g = gen(dev, 4)
    x, w = rand(g, 200, 64, dtype=BF), rand(g, 96, 64, dtype=BF)
    r = rand(g, 200, 96, dtype=BF)
    want = gemm.linear_act_fwd(x, w, act="gelu", resid=r)
    assert torch.equal(gemm.linear_act_fwd(x, w, act="gelu", resid=r, out=r), want)
    z, dy = rand(g, 200, 64, dtype=BF), rand(g, 200, 96, dtype=BF)
    want = gemm.linear_act_dgrad(dy, w, z, "silu")
    assert torch.equal(gemm.linear_act_dgrad(dy, w, z, "silu", out=z), want)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_linear_without_rows(dev):
    x, w = torch.empty(0, 64, dtype=BF, device=dev), torch.ones(32, 64, dtype=BF, device=dev)
    assert gemm.linear_act_fwd(x, w, act="gelu").shape == (0, 32)
    assert gemm.linear_act_dgrad(torch.empty(0, 32, dtype=BF, device=dev), w,
                                 torch.ones(5, 64, dtype=BF, device=dev), "gelu",
                                 z_rows=torch.empty(0, dtype=torch.int32, device=dev)).shape == (0, 64)
    buf, dw = empty(dev, 32, 64, F32, 3, 2)
    db = torch.ones(32, device=dev)
    dy = torch.empty(0, 32, dtype=BF, device=dev)
    gemm.linear_bias_wgrad(dy, x, dw, db)
    assert bool((buf == 9.0).all()) and bool((db == 1.0).all())
    gemm.linear_bias_wgrad(dy, x, dw, db, accumulate=False)
    assert not dw.any() and not db.any() and untouched(buf, 64, 2)
    # a layer without outputs or inputs
    assert gemm.linear_act_fwd(w, w[:0]).shape == (32, 0)
    db = torch.zeros(64, device=dev)
    gemm.linear_bias_wgrad(w, torch.empty(32, 0, dtype=BF, device=dev),
                           torch.empty(64, 0, device=dev), db)
    assert bool((db == 32.0).all())


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("rows", [0, 3])
def test_single_output_row_has_no_stride(dev, rows):
    """A weight gradient of one row, whose stride says nothing, with and without rows to sum."""
    g = gen(dev, 5)
    dy, x = rand(g, rows, 1, dtype=BF), rand(g, rows, 24, dtype=BF)
    buf = torch.full((40,), 9.0, device=dev)
    dw, db = buf.as_strided((1, 24), (1, 1), 8), torch.full((1,), 9.0, device=dev)
    gemm.linear_bias_wgrad(dy, x, dw, db, accumulate=False)
    want = dy.double().t() @ x.double()
    close(dw, want, 2 * rows * U * (dy.double().abs().t() @ x.double().abs()), "dw")
    close(db, dy.double().sum(0), rows * U * dy.double().abs().sum(0), "dbias")
    assert bool((buf[:8] == 9.0).all()) and bool((buf[32:] == 9.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("R,N,K", [(4096, 64, 64), (2000, 512, 256), (70, 136, 2100), (600, 2048, 2304)])
def test_weight_gradients_in_a_row(R, N, K):
    """Small integers, whose sums are exact: every call adds its whole product and column sums before
    what follows it on the stream reads them, eagerly and in a graph."""
    g = gen("cuda", 6)
    dy = torch.randint(-2, 3, (R, N), generator=g, device="cuda").to(BF)
    x = torch.randint(-2, 3, (R, K), generator=g, device="cuda").to(BF)
    want_w, want_b = (dy.double().t() @ x.double()).float(), dy.double().sum(0).float()
    dw, db = torch.zeros(N, K, device="cuda"), torch.zeros(N, device="cuda")
    seen = [(torch.empty_like(dw), torch.empty_like(db)) for _ in range(8)]

    def steps():
        for w, b in seen:
            gemm.linear_bias_wgrad(dy, x, dw, db)
            w.copy_(dw)
            b.copy_(db)

    def check():
        for i, (w, b) in enumerate(seen):
            assert torch.equal(w, (i + 1) * want_w) and torch.equal(b, (i + 1) * want_b)
            w.zero_(), b.zero_()
        dw.zero_(), db.zero_()

    steps()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps()
    for _ in range(3):
        graph.replay()
        check()


# ---------------------------------------------------------------- layer norm
def ln64(x, w, b):
    mean = x.mean(-1, keepdim=True)
    r = ((x - mean).square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = (x - mean) * r
    y = n if w is None else n * w
    return (y if b is None else y + b), mean, r, n


LN_CASES = [
    (256, 256, BF, BF, True, True), (1, 8, BF, BF, True, True), (3, 1, F32, F32, True, True),
    (17, 33, HF, HF, True, False), (300, 250, BF, F32, True, True), (200, 1000, HF, HF, False, False),
    (65, 512, BF, F32, True, True), (129, 768, F32, F32, False, True), (77, 2048, BF, BF, True, True),
    (300, 2048, HF, F32, True, True), (40, 2049, BF, BF, True, True), (33, 4096, BF, F32, True, True),
    (19, 5632, HF, F32, True, True), (12, 8192, F32, F32, True, True), (9, 8200, BF, BF, True, True),
    (5, 16384, F32, F32, True, True), (4, 16383, BF, BF, True, True), (2500, 64, BF, BF, True, True),
    (1300, 512, BF, BF, True, True), (1300, 1024, HF, HF, True, True), (1300, 2048, BF, BF, True, True),
    (1200, 3000, BF, BF, True, True), (2, 24, BF, BF, True, True), (1300, 250, BF, BF, True, True),
]
CHAIN = 160  # the longest chain of additions over a row: 128 of one thread, and the exchanges


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("T,H,dtype,stream,scale,bias", LN_CASES)
@pytest.mark.parametrize("pad,skew,shift", [(0, 0, 0.0), (8, 0, 3.0), (5, 1, -20.0)])
def test_layernorm_fwd(dev, T, H, dtype, stream, scale, bias, pad, skew, shift):
    g = gen(dev, T + H)
    x = rand(g, T, H, dtype=stream, scale=2.0, shift=shift, pad=pad, skew=skew)
    w = rand(g, H, dtype=dtype, scale=0.2, shift=1.0) if scale else None
    b = rand(g, H, dtype=dtype) if bias else None
    buf, o = empty(dev, T, H, dtype, pad, skew)
    given = pad or (w is None and b is None)
    y, mean, rstd = fused.layernorm_fwd(x, w, b, EPS, out=o if given else None)
    assert y.dtype == dtype and mean.dtype == rstd.dtype == F32 and (not given or y is o)
    xd = x.double()
    want, m, r, n = ln64(xd, None if w is None else w.double(), None if b is None else b.double())
    d = xd - m
    tol_m = CHAIN * U * xd.abs().mean(-1, keepdim=True)
    # the mean's error moves the squares' mean by its square alone, the rounding of x - mean by 2 u
    var = d.square().mean(-1, keepdim=True)
    tol_r = r * (((CHAIN + 6) * U * var + tol_m ** 2) / (2 * (var + EPS)) + 4 * U)
    tol = d.abs() * tol_r + r * (tol_m + 4 * U * d.abs())
    if w is not None:
        tol = tol * w.double().abs() + U * want.abs()
    if b is not None:
        tol = tol + U * (want.abs() + b.double().abs())
    close(mean, m[:, 0], tol_m[:, 0], "mean")
    close(rstd, r[:, 0], tol_r[:, 0], "rstd")
    close(y, want, tol, "y")
    assert not given or untouched(buf, H, skew)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("T,H,dtype,stream,scale,bias", LN_CASES)
@pytest.mark.parametrize("some,accumulate,res,pad,skew", [
    (True, False, True, 0, 0), (False, True, False, 8, 0), (True, True, True, 5, 1)])
def test_layernorm_bwd(dev, T, H, dtype, stream, scale, bias, some, accumulate, res, pad, skew):
    g = gen(dev, T + 2 * H)
    R = (T + 1) // 2 if some else T
    x = rand(g, T, H, dtype=stream, scale=2.0, shift=0.5, pad=pad, skew=skew)
    w = rand(g, H, dtype=dtype, scale=0.2, shift=1.0) if scale else None
    dy = rand(g, R, H, dtype=dtype, pad=pad, skew=skew)
    dres = rand(g, R, H, dtype=stream, pad=pad, skew=skew) if res else None
    rows = kept(g, T, R) if some else None
    _, m, r, _ = ln64(x.double(), None, None)
    mean, rstd = m[:, 0].float(), r[:, 0].float()
    dw, db = rand(g, H), rand(g, H) if bias else None
    before, before_b = dw.clone(), None if db is None else db.clone()
    dx = fused.layernorm_bwd(dy, x, mean, rstd, w, dw, db, rows=rows, dres=dres,
                             accumulate=accumulate)
    assert dx.dtype == stream and dx.shape == (R, H)
    at = slice(None) if rows is None else rows.long()
    xd, md, rd = x[at].double(), mean[at].double()[:, None], rstd[at].double()[:, None]
    n, dyd = (xd - md) * rd, dy.double()
    gr = dyd if w is None else dyd * w.double()
    m1, m2 = gr.mean(-1, keepdim=True), (gr * n).mean(-1, keepdim=True)
    want = rd * (gr - m1 - n * m2)
    k = (CHAIN + 6) * U
    tol = rd * (k * gr.abs().mean(-1, keepdim=True) + n.abs() * k * (gr * n).abs().mean(-1, keepdim=True)
                + 6 * U * (gr.abs() + m1.abs() + (n * m2).abs()))
    if res:
        want = want + dres.double()
        tol = tol + U * (want.abs() + dres.double().abs())
    close(dx, want, tol, "dx")
    for name, got, old, s in (("dw", dw, before, dyd * n), ("db", db, before_b, dyd)):
        if got is None:
            continue
        want, tol = s.sum(0), (R + 6) * U * s.abs().sum(0)
        if accumulate:
            want = want + old.double()
            tol = tol + U * want.abs()
        close(got, want, tol, name)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_layernorm_gradient_against_differences(dev):
    g = gen(dev, 8)
    T, H, h = 6, 40, 2.0 ** -10
    x, dy = rand(g, T, H), rand(g, T, H)
    w, b = rand(g, H), rand(g, H)
    _, mean, rstd = fused.layernorm_fwd(x, w, b, EPS)
    dw, db = torch.empty(H, device=dev), torch.empty(H, device=dev)
    dx = fused.layernorm_bwd(dy, x, mean, rstd, w, dw, db, accumulate=False)

    def total(xx, ww, bb):
        return float((ln64(xx, ww, bb)[0] * dy.double()).sum())

    leaves = [x.double(), w.double(), b.double()]
    for i, grad in enumerate((dx, dw, db)):
        d = rand(g, *leaves[i].shape).double()
        up, down = list(leaves), list(leaves)
        up[i], down[i] = leaves[i] + h * d, leaves[i] - h * d
        slope = (total(*up) - total(*down)) / (2 * h)
        # the difference's own error is h^2 / 6 of a third derivative that stays below 1e3 here
        assert abs(float((grad.double() * d).sum()) - slope) < 1e3 * h * h + 1e-4


@pytest.mark.parametrize("dev", CPU_GPU)
def test_layernorm_odd_rows(dev):
    """Constant rows, values far from zero, infinities and NaN; without rows and without columns."""
    g = gen(dev, 5)
    x = rand(g, 40, 96)
    x[1], x[2], x[3, 4], x[4, 5] = 7.0, 0.0, float("nan"), float("inf")
    x[6] = x[6] * 1e-3 + 1e4
    w, b = torch.ones(96, device=dev), torch.zeros(96, device=dev)
    y, mean, rstd = fused.layernorm_fwd(x, w, b, EPS)
    assert not y[1:3].any() and bool(y[3].isnan().all()) and not bool(y[4].isfinite().all())
    # steps of the values at 1e4 are 2^-10: the mean's error of CHAIN u 1e4 is what is left
    want = ln64(x[6].double(), None, None)[0]
    close(y[6], want, 1e4 * CHAIN * U * rstd[6].double() * (1 + want.abs()) + 1e-3, "far from zero")
    dx = fused.layernorm_bwd(torch.ones_like(x), x, mean, rstd, w, None, None)
    assert bool(dx[1:3].abs().max() < 1e-2) and bool(dx[3].isnan().all())
    assert bool(dx[7:].isfinite().all())
    y, mean, _ = fused.layernorm_fwd(x[:0], w, b, EPS)
    assert y.shape == (0, 96) and mean.shape == (0,)
    dw = torch.ones(96, device=dev)
    args = (x[:0], x[:0], mean, mean, w)
    assert fused.layernorm_bwd(*args, dw, None).shape == (0, 96) and bool((dw == 1.0).all())
    fused.layernorm_bwd(*args, dw, None, accumulate=False)
    assert not dw.any()
    assert fused.layernorm_fwd(x[:, :0], w[:0], b[:0], EPS)[0].shape == (40, 0)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("T", [1, 40, 1000])
def test_layernorm_statistics_without_columns(dev, T):
    """The mean of nothing is NaN, on both devices."""
    w = torch.ones(0, device=dev)
    old = [torch.full((T,), 7.0, device=dev) for _ in range(4)]  # (memory that the call may be given)
    del old
    y, mean, rstd = fused.layernorm_fwd(torch.ones(T, 0, device=dev), w, w, EPS)
    assert y.shape == (T, 0) and mean.shape == rstd.shape == (T,)
    assert bool(mean.isnan().all()) and bool(rstd.isnan().all())
    dw = torch.ones(0, device=dev)
    assert fused.layernorm_bwd(y, y, mean, rstd, w, dw, None, accumulate=False).shape == (T, 0)


# ---------------------------------------------------------------- distillation
def distill_case(dev, T, V, K, dtype, top_dtype=F32, tail=True, labels=True, tau=1.0, pad=0, skew=0,
                 ids64=False, seed=0):
    g = gen(dev, T + V + K + seed)
    c = {"logits": rand(g, T, V, dtype=dtype, scale=2.5, pad=pad, skew=skew), "temperature": tau}
    teacher = c["logits"].float() + rand(g, T, V, scale=0.7)
    top, ids = teacher.topk(K, dim=1)
    c["top_lse"] = (teacher.double() / tau).logsumexp(1).float() if tail else None
    # rows of other lists: short ones, an empty one, a token twice, a share of nothing
    if T > 2 and K > 2:
        ids[1, 1:], ids[2] = -1, -5
    if T > 5 and K > 3:
        ids[3, 2], top[4, 1], top[5, -1] = ids[3, 0], -math.inf, -80.0
    c["top_ids"] = ids if ids64 else ids.int()
    c["top_logits"] = top.to(top_dtype)
    c["labels"] = None
    if labels:
        lab = torch.randint(0, V, (T,), generator=g, device=dev)
        lab[::3] = c["top_ids"][::3, 0].long()  # (negative where the list is empty)
        lab[T // 2] = -100
        c["labels"] = lab
    return g, c


def distill64(c, z=None):
    """kd and ce from a dense distribution of the teacher, in 64 bits and differentiable in z."""
    z = c["logits"].double() if z is None else z
    T, V = z.shape
    ids, ok = c["top_ids"].long(), c["top_ids"] >= 0
    logq = torch.log_softmax(z / c["temperature"], 1)
    t = (c["top_logits"].double() / c["temperature"]).masked_fill(~ok, -math.inf)
    norm = t.logsumexp(1) if c["top_lse"] is None else c["top_lse"].double()
    p = torch.exp(t - norm.masked_fill(norm == -math.inf, 0.0)[:, None])
    named = (t - norm[:, None]).masked_fill(p == 0, 0.0)
    kd = (p * (named - torch.where(p > 0, logq.gather(1, ids.clamp(min=0)), named))).sum(1)
    if c["top_lse"] is not None:
        inside = torch.zeros(T, V + 1, dtype=torch.bool, device=z.device)
        inside = inside.scatter(1, ids.masked_fill(~ok, V), True)[:, :V]
        rest = logq.masked_fill(inside, -math.inf).logsumexp(1)
        left = (1 - p.sum(1)).clamp(min=0)
        kd = kd + torch.where((left > 0) & ~inside.all(1),
                              left * (left.clamp(min=1e-300).log() - rest), 0.0)
    if c["labels"] is None:
        return kd, None
    ce = -torch.log_softmax(z, 1).gather(1, c["labels"].clamp(min=0)[:, None])[:, 0]
    return kd, ce.masked_fill(c["labels"] < 0, 0.0)


def log_error(z, tau):
    """The error of a log of a sum of exponentials (fp32, the hardware's exponential): its argument is
    rounded (|x| up to the range of the row, where it counts up to 64 binary orders), 2^-22 of the
    exponential, a chain of 200 additions."""
    return 2.0 ** -22 + (64 + 200) * U + 3 * U * (z.double() / tau).abs().amax(1)


DISTILL = [
    (40, 64, 4, BF, F32, 1.0, 0, 0), (1, 33, 1, F32, F32, 1.0, 0, 0), (9, 1024, 8, BF, BF, 2.0, 0, 0),
    (30, 1000, 16, HF, F32, 0.7, 8, 0), (17, 5003, 33, BF, F32, 2.0, 0, 0),
    (12, 8193, 64, F32, F32, 1.5, 3, 2), (6, 40000, 100, BF, HF, 1.0, 5, 1),
    (3, 128256, 64, F32, F32, 2.0, 0, 0), (700, 300, 5, BF, F32, 1.0, 1, 1), (8, 7, 7, F32, F32, 1.0, 0, 0),
    (7, 1200, 1024, BF, F32, 0.7, 0, 0), (650, 9000, 40, HF, F32, 1.0, 0, 0),
]


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("T,V,K,dtype,top_dtype,tau,pad,skew", DISTILL)
@pytest.mark.parametrize("tail,labels,ids64", [(False, False, True), (True, True, False),
                                               (False, True, False), (True, False, True)])
def test_distill_fwd(dev, T, V, K, dtype, top_dtype, tau, pad, skew, tail, labels, ids64):
    _, c = distill_case(dev, T, V, K, dtype, top_dtype, tail, labels, tau, pad, skew, ids64)
    kd, ce, lse, stats = fused.distill_fwd(**c)
    want_kd, want_ce = distill64(c)
    z = c["logits"].double()
    err = log_error(z, tau)
    # the teacher's side is in 64 bits; the two logarithms and the list's logits times the temperature
    # carry their errors into sums whose weights add up to at most one
    close(kd, want_kd, 3 * err, "kd")
    want = torch.logsumexp(z / tau, 1)
    close(stats[:, 0], want, err, "lse at the temperature")
    if not tail:
        some = (c["top_ids"] >= 0).any(1)
        assert torch.equal(stats[:, 1], stats[:, 0]) and torch.equal(stats[:, 2] == 1.0, some)
    assert (ce is None) == (lse is None) == (not labels)
    if labels:
        close(lse, torch.logsumexp(z, 1), log_error(z, 1.0), "lse")
        close(ce, want_ce, 2 * log_error(z, 1.0), "ce")


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("T,V,K,dtype,top_dtype,tau,pad,skew", DISTILL)
@pytest.mark.parametrize("tail,labels,some,ids64", [
    (False, False, True, True), (True, True, False, False), (False, True, True, False),
    (True, False, False, True)])
def test_distill_bwd(dev, T, V, K, dtype, top_dtype, tau, pad, skew, tail, labels, some, ids64):
    g, c = distill_case(dev, T, V, K, dtype, top_dtype, tail, labels, tau, pad, skew, ids64)
    _, _, lse, stats = fused.distill_fwd(**c)
    R = (2 * T + 2) // 3 if some else T
    rows = kept(g, T, R) if some else None
    at = slice(None) if rows is None else rows.long()
    dkd = rand(g, R)
    dce = rand(g, R) if labels else None
    dkd[R // 2] = 0.0
    buf, o = empty(dev, R, V, dtype, pad, skew)
    args = {k: c[k] for k in ("logits", "top_ids", "top_logits", "temperature", "labels")}
    got = fused.distill_bwd(**args, stats=stats, lse=lse, dkd=dkd, dce=dce, rows=rows,
                            out=o if pad else None)
    assert got.dtype == dtype and got.shape == (R, V) and (not pad or got is o)
    z = c["logits"].double().requires_grad_()
    kd, ce = distill64(c, z)
    total = (kd[at] * dkd.double()).sum()
    soft = torch.zeros((), dtype=F64, device=dev)
    if labels:
        total = total + (ce[at] * dce.double()).sum()
        w = dce.double().masked_fill(c["labels"][at] < 0, 0.0).abs()[:, None]
        soft = torch.softmax(z.detach(), 1)[at] * w
    want = torch.autograd.grad(total, z)[0][at]
    # each term is a product with an exponential whose argument is off by the error of a logarithm
    # and its own rounding; `mass` is the sum of the terms' sizes
    zd = z.detach()[at]
    k = dkd.double().abs()[:, None] / tau
    q = torch.softmax(zd / tau, 1)
    named = torch.zeros(R, V + 1, dtype=F64, device=dev)
    ids = c["top_ids"].long()[at]
    t = c["top_logits"].double()[at] / tau
    p = torch.exp(t - stats[at, 3:4].double()).masked_fill(ids < 0, 0.0)
    p = p.masked_fill(p.isnan(), 0.0)
    named.scatter_add_(1, ids.masked_fill(ids < 0, V), p)
    inside = torch.zeros_like(named).scatter_(1, ids.masked_fill(ids < 0, V), 1.0)[:, :V].bool()
    rest = q.masked_fill(inside, 0.0).sum(1, keepdim=True)
    left = (1 - p.sum(1, keepdim=True)).clamp(min=0) if tail else torch.zeros_like(rest)
    share = (q / rest.clamp(min=1e-300)).masked_fill(inside, 0.0)
    mass = k * (q + named[:, :V] + share * (rest + left)) + 2 * soft
    err = (4 * log_error(zd, min(tau, 1.0)) + 2.0 ** -21)[:, None]
    norm = 2 * U * stats[at, 3:4].double().abs().masked_fill(stats[at, 3:4].isinf(), 0.0)
    close(got, want, (err + norm) * mass + 2 * U * (dce.double().abs()[:, None] if labels else 0.0),
          "dlogits")
    assert not pad or untouched(buf, V, skew)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_gradient_against_differences(dev, tail):
    g, c = distill_case(dev, 7, 50, 6, F32, tail=tail, tau=1.5, seed=3)
    kd, ce, lse, stats = fused.distill_fwd(**c)
    dkd, dce = rand(g, 7), rand(g, 7)
    args = {k: c[k] for k in ("logits", "top_ids", "top_logits", "temperature", "labels")}
    grad = fused.distill_bwd(**args, stats=stats, lse=lse, dkd=dkd, dce=dce)
    d, h = rand(g, 7, 50).double(), 2.0 ** -10
    z = c["logits"].double()

    def total(at):
        a, b = distill64(c, at)
        return float((a * dkd.double()).sum() + (b * dce.double()).sum())

    slope = (total(z + h * d) - total(z - h * d)) / (2 * h)
    assert abs(float((grad.double() * d).sum()) - slope) < 100 * h * h + 1e-4


@pytest.mark.parametrize("dev", CPU_GPU)
def test_distill_odd_rows(dev):
    """Masked logits, rows of which nothing is left, weights of zero, lists over the whole vocabulary."""
    g, c = distill_case(dev, 8, 96, 5, F32, tail=False, labels=True)
    z = c["logits"]
    c["top_ids"][6] = torch.arange(5, device=dev)
    z[6, 50:] = -math.inf  # masked, and nothing of the list
    c["labels"][:] = torch.arange(8, device=dev)
    z[7, c["top_ids"][7, 0].long()] = -math.inf  # a named token that the student rules out
    c["labels"][7] = int(c["top_ids"][7, 1])
    z[5] = -math.inf  # nothing is left
    z[4, 3] = float("nan")
    kd, ce, lse, stats = fused.distill_fwd(**c)
    assert bool(kd[6].isfinite()) and bool(kd[7] == math.inf) and bool(ce[:4].isfinite().all())
    assert not bool(kd[5].isfinite()) and bool(kd[4].isnan()) and bool(ce[4].isnan())
    dkd, dce = torch.ones(8, device=dev), torch.ones(8, device=dev)
    dkd[4:6] = dce[4:6] = 0.0  # weights of zero, whatever the rows hold
    args = {k: c[k] for k in ("logits", "top_ids", "top_logits", "temperature", "labels")}
    got = fused.distill_bwd(**args, stats=stats, lse=lse, dkd=dkd, dce=dce)
    assert bool(got.isfinite().all()) and not got[4:6].any() and not got[6, 50:].any()
    # the gradient of a softmax adds up to nothing, the infinite divergence's too
    assert float(got.double().sum(1).abs().max()) < 1e-5
    # a list over the whole vocabulary leaves nothing for the rest
    ids = torch.arange(96, device=dev, dtype=torch.int32).repeat(8, 1)
    z = rand(g, 8, 96)
    t = rand(g, 8, 96)
    kd, _, _, stats = fused.distill_fwd(z, ids, t, top_lse=t.double().logsumexp(1).float())
    p = torch.softmax(t.double(), 1)
    want = (p * (p.log() - torch.log_softmax(z.double(), 1))).sum(1)
    close(kd, want, 4 * log_error(z, 1.0) + 8 * U * t.double().abs().amax(1), "whole vocabulary")
    assert bool((stats[:, 1] == -math.inf).all()) and not stats[:, 2].any()
    got = fused.distill_bwd(z, ids, t, stats, torch.ones(8, device=dev))
    want = torch.softmax(z.double(), 1) - p
    close(got, want, 1e-5 * (want.abs() + 2 * p), "whole vocabulary's gradient")
    # without rows
    kd, ce, lse, stats = fused.distill_fwd(z[:0], ids[:0], t[:0], labels=c["labels"][:0])
    assert kd.shape == ce.shape == lse.shape == (0,) and stats.shape == (0, 4)
    rows = torch.empty(0, dtype=torch.int32, device=dev)
    full = fused.distill_fwd(z, ids, t)[3]
    assert fused.distill_bwd(z, ids, t, full, torch.empty(0, device=dev), rows=rows).shape == (0, 96)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("V,dtype", [(512, BF), (515, F32), (40000, BF)])
def test_distill_bwd_in_place(dev, V, dtype):
    g, c = distill_case(dev, 6, V, 9, dtype, tau=2.0)
    _, _, lse, stats = fused.distill_fwd(**c)
    args = {k: c[k] for k in ("logits", "top_ids", "top_logits", "temperature", "labels")}
    args.update(stats=stats, lse=lse, dkd=rand(g, 6), dce=rand(g, 6))
    want = fused.distill_bwd(**args)
    assert torch.equal(fused.distill_bwd(**args, out=c["logits"]), want)


def far_case(dev, T, V, K, dtype, gap, tau, labels, high="list"):
    """The listed tokens and the others `gap` apart in the student's logits; the teacher leaves the
    others 0.23.  Half of the labels are listed, some are ignored."""
    g = gen(dev, V + K + int(gap))
    z = rand(g, T, V)
    ids = torch.rand(T, V, generator=g, device=dev).argsort(1)[:, :K].int()
    z.scatter_add_(1, ids.long(), torch.full((T, K), gap if high == "list" else -gap, device=dev))
    z = z.to(dtype)
    p = torch.softmax(rand(g, T, K), 1) * 0.77
    c = {"logits": z, "top_ids": ids, "top_logits": p.log() * tau, "temperature": tau,
         "top_lse": torch.zeros(T, device=dev), "labels": None}
    if labels:
        lab = torch.randint(0, V, (T,), generator=g, device=dev)
        lab[::2] = ids[::2, -1].long()
        lab[T // 2] = -1
        c["labels"] = lab
    return g, c


def distill_far_check(g, c, err):
    """Both losses and their gradient against 64 bits, each exponential within `err` of its size."""
    T, V = c["logits"].shape
    tau, dev = c["temperature"], c["logits"].device
    kd, ce, lse, stats = fused.distill_fwd(**c)
    z = c["logits"].double().requires_grad_()
    want_kd, want_ce = distill64(c, z)
    close(kd, want_kd.detach(), 3 * log_error(c["logits"], tau), "kd")
    dkd = rand(g, T)
    args = {k: c[k] for k in ("logits", "top_ids", "top_logits", "temperature", "labels")}
    total, soft, dce = (want_kd * dkd.double()).sum(), 0.0, None
    if ce is not None:
        close(ce, want_ce.detach(), 2 * log_error(c["logits"], 1.0), "ce")
        dce = rand(g, T)
        total = total + (want_ce * dce.double()).sum()
        soft = dce.double().masked_fill(c["labels"] < 0, 0.0).abs()[:, None]
        soft = soft * (torch.softmax(z.detach(), 1) + 2 * U)
    got = fused.distill_bwd(**args, stats=stats, lse=lse, dkd=dkd, dce=dce)
    want = torch.autograd.grad(total, z)[0]
    x = z.detach() / tau
    inside = torch.zeros(T, V, dtype=torch.bool, device=dev).scatter_(1, c["top_ids"].long(), True)
    p = torch.exp(c["top_logits"].double() / tau)
    named = torch.zeros(T, V, dtype=F64, device=dev).scatter_add_(1, c["top_ids"].long(), p)
    q = torch.softmax(x, 1)
    share = torch.softmax(x.masked_fill(inside, -math.inf), 1)
    part = q.masked_fill(inside, 0.0).sum(1, keepdim=True)
    k = dkd.double().abs()[:, None] / tau
    mass = k * (q + named + share * (part + 0.23)) + 2 * soft
    # an exponential below 2^-126 counts as zero: the weights k (part - 0.23) and dce multiply one each
    weights = k if dce is None else k + dce.double().abs()[:, None]
    close(got, want, err * mass + 2.0 ** -126 * weights, "dlogits")


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("T,V,K,dtype,labels", [
    (5, 64, 2, F32, True), (9, 515, 7, BF, False), (4, 20000, 33, F32, False), (3, 40000, 5, BF, True),
    (1100, 300, 4, HF, True)])
@pytest.mark.parametrize("high", ["list", "rest"])
@pytest.mark.parametrize("gap,tau", [(60.0, 1.0), (90.0, 1.0), (200.0, 1.0), (9.5, 0.1), (60.0, 0.1),
                                     (200.0, 0.1), (150.0, 2.0)])
def test_distill_far_apart(dev, T, V, K, dtype, labels, high, gap, tau):
    """The student gives one side of the list next to nothing, less than fp32 holds: its logarithm
    is still there, and so is the gradient."""
    g, c = far_case(dev, T, V, K, dtype, gap, tau, labels, high)
    distill_far_check(g, c, (4 * log_error(c["logits"], min(tau, 1.0)) + 2.0 ** -21)[:, None])


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("T,V,K", [(5, 300, 3), (3, 20000, 33)])
@pytest.mark.parametrize("gap,tau", [(200.0, 0.1), (1e4, 1.0), (1e4, 2.0), (3e5, 0.7), (4e6, 1.0)])
@pytest.mark.parametrize("labels", [False, True])
def test_distill_gradient_of_a_far_rest(dev, T, V, K, gap, tau, labels):
    """The gradient of the tokens outside the list does not depend on how far they all lie below it,
    although an fp32 logarithm of their sum has ever fewer digits."""
    g, c = far_case(dev, T, V, K, F32, gap, tau, labels)
    c["logits"] -= gap  # the list near zero, the others far below
    _, _, lse, stats = fused.distill_fwd(**c)
    dkd, dce = rand(g, T), rand(g, T) if labels else None
    args = {k: c[k] for k in ("logits", "top_ids", "top_logits", "temperature", "labels")}
    got = fused.distill_bwd(**args, stats=stats, lse=lse, dkd=dkd, dce=dce)
    x = c["logits"].double() / tau
    out = torch.zeros(T, V, dtype=torch.bool, device=dev).scatter_(1, c["top_ids"].long(), True)
    left = (1 - torch.exp(c["top_logits"].double() / tau).sum(1, keepdim=True))
    share = torch.softmax(x.masked_fill(out, -math.inf), 1)
    want = -dkd.double()[:, None] / tau * left * share
    if labels:
        at = torch.arange(T, device=dev)[c["labels"] >= 0], c["labels"][c["labels"] >= 0]
        want[at] -= dce.double()[c["labels"] >= 0]
    # the sum (2^-22 of each exponential, a chain of 200 additions) and the exponential (the same, its
    # argument rounded at up to 150), the differences of the logits times the rounded temperature, five
    # roundings of factors
    spread = (x.masked_fill(out, -math.inf).amax(1) - x.masked_fill(out, math.inf).amin(1))[:, None]
    tol = (2.0 ** -21 + (64 + 200 + 150 + 5 + 3 * spread) * U) * want.abs() + 2.0 ** -126 * dkd.abs()[:, None]
    close(got.masked_fill(out, 0.0), want.masked_fill(out, 0.0), tol, "dlogits")


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("T,V,kept_cols", [
    (4, 1000, 992), (4, 1003, 1002), (3, 40000, 28000), (2, 64, 8), (1100, 300, 100)])
@pytest.mark.parametrize("tau,tail", [(1.0, True), (2.0, True), (0.7, True), (1.0, False), (0.5, False)])
def test_distill_logits_masked_by_the_lowest_value(dev, dtype, T, V, kept_cols, tau, tail):
    """A mask by the type's lowest value, whose product with the temperature may overflow, is one by
    -inf: in some columns, and where the list is all that is left of the vocabulary."""
    if dtype == HF:  # (-65504 is a logit like any other: the list may not be all that is left)
        kept_cols = max(kept_cols, 40)
    g = gen(dev, V + T)
    z = rand(g, T, V, dtype=dtype)
    K = min(kept_cols, 8)
    ids = torch.rand(T, kept_cols, generator=g, device=dev).argsort(1)[:, :K]
    lab = torch.randint(0, kept_cols, (T,), generator=g, device=dev)
    top = rand(g, T, K)
    lse = (top / tau).logsumexp(1) + 0.2 if tail else None
    dkd, dce = rand(g, T), rand(g, T)
    outs = []
    for low in (-math.inf, torch.finfo(dtype).min):
        z[:, kept_cols:] = low
        kd, ce, s, stats = fused.distill_fwd(z, ids, top, tau, top_lse=lse, labels=lab)
        outs.append((kd, ce, s, stats, fused.distill_bwd(z, ids, top, stats, dkd, tau, labels=lab,
                                                         lse=s, dce=dce)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert all(bool(t.isfinite().all()) for t in outs[0][:3] + outs[0][4:])
    c = {"logits": z[:, :kept_cols], "top_ids": ids, "top_logits": top, "temperature": tau,
         "top_lse": lse, "labels": lab}
    want_kd, want_ce = distill64(c)
    close(kd, want_kd, 3 * log_error(c["logits"], tau), "kd")
    close(ce, want_ce, 2 * log_error(c["logits"], 1.0), "ce")
    assert not outs[0][4][:, kept_cols:].any()


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("low", [None, -1e4, -1e9, -1e30])
@pytest.mark.parametrize("T,V,tau,tail", [(3, 200, 1.0, True), (2, 20000, 2.0, True), (5, 515, 0.7, False),
                                          (4, 1000, 0.5, True)])
def test_distill_rows_of_which_nothing_is_left(dev, dtype, low, T, V, tau, tail):
    """All logits at the value of a mask: what is left is a uniform distribution."""
    low = torch.finfo(dtype).min if low is None or dtype == HF else low
    g = gen(dev, V)
    z = torch.full((T, V), low, dtype=dtype, device=dev)
    ids, lab = torch.arange(6, device=dev).repeat(T, 1), torch.full((T,), 3, device=dev)
    top = rand(g, T, 6)
    lse = (top / tau).logsumexp(1) + 0.2 if tail else None
    kd, ce, s, stats = fused.distill_fwd(z, ids, top, tau, top_lse=lse, labels=lab)
    c = {"logits": z * 0, "top_ids": ids, "top_logits": top, "temperature": tau, "top_lse": lse,
         "labels": lab}
    want_kd, want_ce = distill64(c)
    close(kd, want_kd, 3 * log_error(c["logits"], tau), "kd")
    close(ce, want_ce, 2 * log_error(c["logits"], 1.0), "ce")
    assert bool(s.isfinite().all()) and bool(stats.isfinite().all())
    got = fused.distill_bwd(z, ids, top, stats, rand(g, T), tau, labels=lab, lse=s, dce=rand(g, T))
    assert bool(got.isfinite().all()) and bool(got.abs().max() < 20 / tau)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("T,V,K", [(4, 64, 2), (5, 1003, 1), (3, 40000, 33), (1100, 300, 6)])
@pytest.mark.parametrize("tau,labels", [(1.0, False), (1.0, True), (2.0, True), (0.7, False)])
def test_distill_lists_without_a_share(dev, T, V, K, tau, labels):
    """A list of nothing but -inf is an empty one: no divergence, and no gradient but the labels'."""
    g = gen(dev, V)
    z, ids = rand(g, T, V), torch.rand(T, V, generator=g, device=dev).argsort(1)[:, :K]
    top = torch.full((T, K), -math.inf, device=dev)
    top[0] = rand(g, K)
    lab = ids[:, -1].clone() if labels else None
    if labels:
        lab[::2] = (ids[::2, 0] + 1) % V
    dkd, dce = rand(g, T), rand(g, T) if labels else None
    grads = []
    for where in (ids, torch.where(top > -math.inf, ids, torch.full_like(ids, -1))):
        kd, _, lse, stats = fused.distill_fwd(z, where, top, tau, labels=lab)
        assert not kd[1:].any() and bool(kd[0] > 0)
        grads.append(fused.distill_bwd(z, where, top, stats, dkd, tau, labels=lab, lse=lse, dce=dce))
    # (of a listed label the exponential is formed in 64 bits)
    close(grads[0], grads[1].double(), 2.0 ** -20 * grads[1].double().abs(), "as without entries")
    alone = fused.distill_bwd(z, ids, top, stats, torch.zeros_like(dkd), tau, labels=lab, lse=lse, dce=dce)
    assert torch.equal(grads[0][1:], alone[1:]) and bool(grads[0][0].any())
    top[1, 0] = math.nan
    kd, _, lse, stats = fused.distill_fwd(z, ids, top, tau, labels=lab)
    got = fused.distill_bwd(z, ids, top, stats, dkd, tau, labels=lab, lse=lse, dce=dce)
    assert bool(kd[1].isnan()) and bool(got[1].isnan().any())


def test_distill_definition_against_torch():
    """Without the teacher's tail the gradient is that of torch's divergence to a dense teacher."""
    g, c = distill_case("cpu", 5, 40, 40, F32, tail=False, labels=False, tau=2.0, seed=1)
    c["top_ids"] = torch.stack([torch.randperm(40, generator=g) for _ in range(5)]).int()
    dense = torch.zeros(5, 40).scatter_(1, c["top_ids"].long(), c["top_logits"].float())
    z = c["logits"].double().requires_grad_()
    want = torch.nn.functional.kl_div(torch.log_softmax(z / 2, 1),
                                      torch.log_softmax(dense.double() / 2, 1), log_target=True,
                                      reduction="none").nan_to_num(0.0).sum(1)
    kd, _, _, stats = ref.distill(c["logits"], c["top_ids"], c["top_logits"], 2.0)
    assert torch.allclose(kd, want, rtol=1e-12, atol=1e-12)
    got = ref.distill_bwd(c["logits"], c["top_ids"], c["top_logits"], stats, torch.ones(5), 2.0)
    assert torch.allclose(got, torch.autograd.grad(want.sum(), z)[0], rtol=1e-10, atol=1e-12)


# ---------------------------------------------------------------- refusals and bad indices
def status():
    from centrifuge_b200.ops._ext import status_block
    s = status_block(0)
    s[0] = 0
    return s


def test_bad_indices_raise_on_the_cpu():
    x, w = torch.ones(4, 8, dtype=BF), torch.ones(8, 16, dtype=BF)
    z = torch.ones(3, 16, dtype=BF)
    for bad in (-1, 3):
        rows = torch.tensor([0, 1, bad, 2], dtype=torch.int32)
        with pytest.raises(IndexError):
            gemm.linear_act_dgrad(x, w, z, "gelu", z_rows=rows)
        dw = torch.ones(8)
        with pytest.raises(IndexError):
            fused.layernorm_bwd(x, z[:, :8], torch.zeros(3), torch.ones(3), None, dw, None, rows=rows)
        assert bool((dw == 1.0).all())
    logits, ids, top = torch.zeros(3, 10), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    stats = fused.distill_fwd(logits, ids, top)[3]
    for bad in (-1, 3):
        with pytest.raises(IndexError):
            fused.distill_bwd(logits, ids, top, stats, torch.ones(1),
                              rows=torch.tensor([bad], dtype=torch.int32))
    ids[1, 1] = 10
    with pytest.raises(IndexError):
        fused.distill_fwd(logits, ids, top)
    ids[1, 1] = 0
    with pytest.raises(IndexError):
        fused.distill_fwd(logits, ids, top, labels=torch.tensor([0, 10, -1]))


@pytest.mark.gpu
@pytest.mark.parametrize("N", [16, 300, 33])
def test_linear_dgrad_reports_bad_rows(N):
    g = gen("cuda", N)
    dy, w, z = rand(g, 6, 64, dtype=BF), rand(g, 64, N, dtype=BF), rand(g, 5, N, dtype=BF)
    rows = torch.tensor([0, 4, 5, 2, -1, 1], dtype=torch.int32, device="cuda")
    s = status()
    got = gemm.linear_act_dgrad(dy, w, z, "gelu", z_rows=rows)
    assert int(s[0]) == 128
    s[0] = 0
    good = torch.tensor([0, 1, 3, 5], device="cuda")
    want = gemm.linear_act_dgrad(dy[good], w, z, "gelu", z_rows=rows[good])
    assert torch.equal(got[good], want) and not got[2].any() and not got[4].any()
    assert int(s[0]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("H,dtype", [(64, BF), (512, BF), (1000, HF), (250, BF), (33, F32), (2048, BF),
                                     (4096, F32), (16384, BF)])
def test_layernorm_bwd_reports_bad_rows(H, dtype):
    g = gen("cuda", H)
    x, dy, w = rand(g, 9, H, dtype=dtype), rand(g, 5, H, dtype=dtype), rand(g, H, dtype=dtype)
    _, mean, rstd = fused.layernorm_fwd(x, w, None, EPS)
    dres = rand(g, 5, H, dtype=dtype)
    rows = torch.tensor([8, 9, 0, -7, 3], dtype=torch.int32, device="cuda")
    dw, db = torch.empty(H, device="cuda"), torch.empty(H, device="cuda")
    s = status()
    dx = fused.layernorm_bwd(dy, x, mean, rstd, w, dw, db, rows=rows, dres=dres, accumulate=False)
    assert int(s[0]) == 128
    s[0] = 0
    good = torch.tensor([0, 2, 4], device="cuda")
    gw, gb = torch.empty(H, device="cuda"), torch.empty(H, device="cuda")
    want = fused.layernorm_bwd(dy[good], x, mean, rstd, w, gw, gb, rows=rows[good], dres=dres[good],
                               accumulate=False)
    assert int(s[0]) == 0 and torch.equal(dx[good], want) and not dx[1].any() and not dx[3].any()
    # the rows may be summed in another order: three of them, and the additions of zeros
    assert torch.allclose(dw, gw, rtol=0, atol=float(8 * U * gw.abs().max() + 8 * U * dy.abs().sum()))
    assert torch.allclose(db, gb, rtol=0, atol=float(8 * U * dy.float().abs().sum(0).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [64, 9001])
def test_distill_reports_bad_indices(V):
    g, c = distill_case("cuda", 6, V, 4, BF, tail=True, labels=True)
    c["labels"] = torch.arange(6, device="cuda")
    fine = {**c, "top_ids": c["top_ids"].clone(), "labels": c["labels"].clone()}
    c["top_ids"][0, 2], c["labels"][3] = V, V + 7
    fine["top_ids"][0, 2], fine["labels"][3] = -1, -1
    s = status()
    got = fused.distill_fwd(**c)
    assert int(s[0]) == 128
    s[0] = 0
    want = fused.distill_fwd(**fine)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    dkd, dce = rand(g, 3), rand(g, 3)
    rows = torch.tensor([0, 6, 3], dtype=torch.int32, device="cuda")
    args = [{k: t[k] for k in ("logits", "top_ids", "top_logits", "temperature", "labels")}
            for t in (c, fine)]
    kw = dict(stats=want[3], lse=want[2])
    a = fused.distill_bwd(**args[0], **kw, dkd=dkd, dce=dce, rows=rows)
    assert int(s[0]) == 128
    s[0] = 0
    at = torch.tensor([0, 2], device="cuda")
    b = fused.distill_bwd(**args[1], **kw, dkd=dkd[at], dce=dce[at], rows=rows[at])
    assert int(s[0]) == 0 and torch.equal(a[at], b) and not a[1].any()


def linear_refusals(dev):
    def t(*shape, dtype=BF):
        return torch.zeros(*shape, dtype=dtype, device=dev)

    x, w, z = t(8, 16), t(24, 16), t(8, 24)
    buf = t(8, 64)
    i32 = torch.zeros(8, dtype=torch.int32, device=dev)
    fwd, dgrad, wgrad = gemm.linear_act_fwd, gemm.linear_act_dgrad, gemm.linear_bias_wgrad
    return [
        lambda: fwd(x, w, act="tanh"), lambda: fwd(x.long(), w), lambda: fwd(x, w.half()),
        lambda: fwd(x, t(24, 15)), lambda: fwd(x.view(-1), w), lambda: fwd(x, w, bias=t(23)),
        lambda: fwd(x, w, bias=t(24, dtype=F32)), lambda: fwd(x, w, bias=t(48)[::2]),
        lambda: fwd(x, w, resid=t(8, 23)), lambda: fwd(x, w, out=t(7, 24)),
        lambda: fwd(x, w, out=t(8, 24, dtype=F32)), lambda: fwd(x, w, z=t(8, 24, dtype=HF)),
        lambda: fwd(x[:, :0], w[:, :0]), lambda: fwd(x.t(), t(24, 8)),
        lambda: fwd(x, w, out=z, z=z), lambda: fwd(buf[:, :16], w, out=buf[:, 8:32]),
        lambda: fwd(x, w, resid=buf[:, :24], out=buf[:, 8:32]),
        lambda: fwd(x, w, resid=z, z=z),
        lambda: dgrad(z, w, x, "swish"), lambda: dgrad(z, w, t(7, 16), "gelu"),
        lambda: dgrad(z, w, x, "gelu", z_rows=i32[:7]), lambda: dgrad(z, w, x, "gelu", z_rows=i32.long()),
        lambda: dgrad(z, w, x.half(), "gelu"), lambda: dgrad(z, w, x, "gelu", z_rows=i32, out=x),
        lambda: dgrad(z, w, x, "gelu", out=t(8, 24)), lambda: dgrad(z, t(23, 16), x, "gelu"),
        lambda: dgrad(z, w, t(8, 17), "gelu"),
        lambda: dgrad(buf[:, :24], w, x, "gelu", out=buf[:, 8:24]),
        lambda: wgrad(z, x, t(24, 16)), lambda: wgrad(z, x, t(16, 24, dtype=F32)),
        lambda: wgrad(z, t(7, 16), t(24, 16, dtype=F32)),
        lambda: wgrad(z, x, t(24, 16, dtype=F32), t(16, dtype=F32)),
        lambda: wgrad(z, x, t(24, 16, dtype=F32), t(24)),
        lambda: (lambda d: wgrad(z, x, d, d.view(-1)[:24]))(t(24, 16, dtype=F32)),
        lambda: (lambda d: wgrad(d.view(BF)[:8, :24], x, d))(t(24, 16, dtype=F32)),
    ]


def layernorm_refusals(dev):
    def t(*shape, dtype=F32):
        return torch.zeros(*shape, dtype=dtype, device=dev)

    x, w, s = t(6, 32, dtype=BF), t(32, dtype=BF), t(6)
    dw = t(32)
    i32 = torch.zeros(6, dtype=torch.int32, device=dev)
    fwd, bwd = fused.layernorm_fwd, fused.layernorm_bwd
    return [
        lambda: fwd(x.view(-1), w, None, EPS), lambda: fwd(x, t(31, dtype=BF), None, EPS),
        lambda: fwd(x, w, t(32), EPS), lambda: fwd(x, t(32), None, EPS), lambda: fwd(x.long(), None, None, EPS),
        lambda: fwd(x, w, None, EPS, out=x), lambda: fwd(x, w, None, EPS, out=t(6, 32)),
        lambda: fwd(x.t(), t(6, dtype=BF), None, EPS), lambda: fwd(t(2, 16385), None, None, EPS),
        lambda: fwd(x, w, None, EPS, out=t(5, 32, dtype=BF)), lambda: fwd(x, t(64, dtype=BF)[::2], None, EPS),
        lambda: bwd(x[:5], x, s, s, w, dw, None), lambda: bwd(x, x.half(), s, s, w, dw, None),
        lambda: bwd(x, x, s[:5], s, w, dw, None), lambda: bwd(x, x, s, s.double(), w, dw, None),
        lambda: bwd(x, x, s, s, t(32), dw, None), lambda: bwd(x, x, s, s, w, t(33), None),
        lambda: bwd(x, x, s, s, w, w, None), lambda: bwd(x, x, s, s, w, dw, dw),
        lambda: bwd(x, x, s, s, w, dw, None, dres=t(6, 32)),
        lambda: bwd(x, x, s, s, w, dw, None, rows=i32[:5]),
        lambda: bwd(x, x, s, s, w, dw, None, rows=i32.long()),
        lambda: (lambda d: bwd(x, x, d[:6], s, w, d, None))(t(32)),
        lambda: (lambda d: bwd(x, d, s, s, w, d[0], None))(t(6, 32)),
    ]


def distill_refusals(dev):
    def t(*shape, dtype=F32):
        return torch.zeros(*shape, dtype=dtype, device=dev)

    z, ids, top, lab = t(6, 40), t(6, 4, dtype=torch.int32), t(6, 4), t(6, dtype=torch.long)
    st, one = t(6, 4), t(6)
    i32 = t(6, dtype=torch.int32)
    fwd, bwd = fused.distill_fwd, fused.distill_bwd
    return [
        lambda: fwd(z.view(-1), ids, top), lambda: fwd(z.double(), ids, top), lambda: fwd(z, top, top),
        lambda: fwd(z, ids[:5], top), lambda: fwd(z, ids, top[:, :3]), lambda: fwd(z, ids, top, 0.0),
        lambda: fwd(z, ids, top, -1.0), lambda: fwd(z, ids, top, math.inf), lambda: fwd(z, ids, top, math.nan),
        lambda: fwd(z, ids, top, top_lse=one[:5]), lambda: fwd(z, ids, top, top_lse=one.double()),
        lambda: fwd(z, ids, top, labels=i32), lambda: fwd(z, ids, top, labels=lab[:5]),
        lambda: fwd(z, ids[:, :0], top[:, :0]), lambda: fwd(z[:, :0], ids, top),
        lambda: fwd(z, t(6, 1025, dtype=torch.int32), t(6, 1025)), lambda: fwd(z, ids, lab.view(6, 1)),
        lambda: fwd(t(1, (1 << 20) + 1, dtype=BF), ids[:1], top[:1]),
        lambda: fwd(z, ids.t().contiguous().t(), top),
        lambda: bwd(z, ids, top, st[:5], one), lambda: bwd(z, ids, top, st, one[:5]),
        lambda: bwd(z, ids, top, st, one.half()), lambda: bwd(z, ids, top, st, one, labels=lab),
        lambda: bwd(z, ids, top, st, one, labels=lab, lse=one), lambda: bwd(z, ids, top, st, one, dce=one),
        lambda: bwd(z, ids, top, st, one, labels=lab, lse=one, dce=one[:5]),
        lambda: bwd(z, ids, top, st, one, rows=i32[:5]), lambda: bwd(z, ids, top, st, one, rows=lab),
        lambda: bwd(z, ids, top, st, one, rows=i32, out=z), lambda: bwd(z, ids, top, st, one, out=t(6, 39)),
        lambda: bwd(z, ids, top, st, one, out=t(6, 40, dtype=BF)),
        lambda: (lambda b: bwd(b[:, :40], ids, top, st, one, out=b[:, 8:48]))(t(6, 64)),
    ]


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("calls", [linear_refusals, layernorm_refusals, distill_refusals])
def test_refusals(dev, calls):
    for i, call in enumerate(calls(dev)):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("dev", CPU_GPU)
def test_temperatures_beyond_fp32(dev):
    """One whose reciprocal fp32 does not hold gave NaN on the GPU; large ones make a softmax uniform."""
    z, ids, top = torch.zeros(3, 40, device=dev), torch.arange(4, device=dev).repeat(3, 1), torch.zeros(3, 4, device=dev)
    z[:, 30:] = -math.inf
    z[1, :20], z[2] = 2.0, z[2] - 3.0
    kd, _, _, stats = fused.distill_fwd(z, ids, top, 2.0 ** 100)
    close(kd, torch.full((3,), math.log(30 / 4), dtype=F64, device=dev), 1e-6, "kd")
    args = (z, ids, top, stats, kd)
    assert bool(fused.distill_bwd(*args, temperature=2.0 ** 100).isfinite().all())
    for tau in (1e-46, 1e-39, 2.0 ** -101, 2.0 ** 101, 1e39, 1e46, 1e300):
        with pytest.raises(ValueError):
            fused.distill_fwd(z, ids, top, tau)
        with pytest.raises(ValueError):
            fused.distill_bwd(*args, temperature=tau)


@pytest.mark.gpu
def test_another_device_is_refused():
    x, w = torch.zeros(4, 16, dtype=BF, device="cuda"), torch.zeros(8, 16, dtype=BF)
    with pytest.raises(ValueError):
        gemm.linear_act_fwd(x, w)
    with pytest.raises(ValueError):
        gemm.linear_bias_wgrad(x, x, torch.zeros(16, 16))
    with pytest.raises(ValueError):
        fused.layernorm_fwd(x, w[0], None, EPS)
    with pytest.raises(ValueError):
        fused.distill_fwd(x, torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("R,N,K", [(20000, 256, 256), (16384, 300, 130), (9000, 5632, 1024),
                                   (33000, 128, 128)])
def test_wgrad_over_many_rows_keeps_fp32_accuracy(R, N, K):
    """The products' own additions end after 1024 rows (2 * 1024 u of a segment's mass at most, for
    more than 16384 rows to a block in proportion), the segments' sums are fp32."""
    g = gen("cuda", R)
    dy, x = rand(g, R, N, dtype=BF, shift=0.25), rand(g, R, K, dtype=BF, shift=0.25)
    dw, db = torch.empty(N, K, device="cuda"), torch.empty(N, device="cuda")
    runs = []
    for _ in range(2):
        gemm.linear_bias_wgrad(dy, x, dw, db, accumulate=False)
        runs.append((dw.clone(), db.clone()))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    mass = dy.double().abs().t() @ x.double().abs()
    close(dw, dy.double().t() @ x.double(), (2 * 1024 + R // 1024 + 2) * U * mass, "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("R,N,K", [
    (16384, 1280, 1280), (16385, 1500, 1500), (65536, 1500, 1500), (131072, 1280, 1280), (100000, 256, 250),
    (9217, 128, 64), (5000, 200, 1200), (4096, 1500, 1500), (65536, 640, 512), (40000, 5632, 1024)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_wgrad_error_does_not_grow_with_the_rows(R, N, K, dtype):
    """Products of one sign, whose errors add up: an instruction adds those of 16 rows to a sum of at
    most 1024 rows and may drop a step (2 u) of it, the sums of 1024 rows are added in fp32."""
    g = gen("cuda", R + N)
    dy, x = rand(g, R, N, dtype=dtype).abs(), rand(g, R, K, dtype=dtype).abs()
    dw = rand(g, N, K).abs()
    before = dw.clone()
    gemm.linear_bias_wgrad(dy, x, dw)
    cols = torch.randperm(N, generator=g, device="cuda")[:96]
    want = torch.zeros(len(cols), K, dtype=F64, device="cuda")
    for i in range(0, R, 1 << 14):
        want += dy[i:i + (1 << 14), cols].double().t() @ x[i:i + (1 << 14)].double()
    close(dw[cols], want + before[cols].double(), (2 * 64 + R // 1024 + 4) * U * (want + before[cols]), "dw")
    again = before.clone()
    gemm.linear_bias_wgrad(dy, x, again)
    assert torch.equal(dw, again)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_distill_lists_with_strides(dev):
    g, c = distill_case(dev, 20, 333, 6, BF, tail=True, tau=2.0)
    want = fused.distill_fwd(**c)
    wide = {}
    for k in ("top_ids", "top_logits"):
        buf = torch.full((20, 17), 5, dtype=c[k].dtype, device=dev)
        buf[:, 3:9] = c[k]
        wide[k] = buf[:, 3:9]
    got = fused.distill_fwd(**{**c, **wide})
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    kw = dict(stats=want[3], lse=want[2], dkd=rand(g, 20), dce=rand(g, 20), labels=c["labels"],
              temperature=2.0)
    a = fused.distill_bwd(c["logits"], c["top_ids"], c["top_logits"], **kw)
    assert torch.equal(fused.distill_bwd(c["logits"], wide["top_ids"], wide["top_logits"], **kw), a)


# ---------------------------------------------------------------- together
def student_step(s, rows):
    """A block with layer norms and a biased MLP, its head, both losses, and the gradients over the
    kept rows, as a training step calls them."""
    kept_of = lambda t: fused.gather_rows(t, rows)  # noqa: E731
    n1, m1, r1 = fused.layernorm_fwd(s["x"], s["g1"], s["b1"], EPS)
    z = torch.empty(n1.shape[0], s["w1"].shape[0], dtype=n1.dtype, device=n1.device)
    h = gemm.linear_act_fwd(n1, s["w1"], s["c1"], act="gelu_tanh", z=z)
    y = gemm.linear_act_fwd(h, s["w2"], s["c2"], resid=s["x"])
    n2, m2, r2 = fused.layernorm_fwd(y, s["g2"], s["b2"], EPS)
    logits = gemm.linear_act_fwd(n2, s["head"])
    kd, ce, lse, stats = fused.distill_fwd(logits, s["ids"], s["top"], 2.0, top_lse=s["top_lse"],
                                           labels=s["labels"])
    f32 = dict(dtype=F32, device=logits.device)
    acc = {k: torch.zeros(s[k].shape, **f32) for k in ("head", "w1", "w2", "c1", "c2", "g1", "b1",
                                                       "g2", "b2")}
    dlogits = fused.distill_bwd(logits, s["ids"], s["top"], stats, s["dkd"], 2.0, labels=s["labels"],
                                lse=lse, dce=s["dce"], rows=rows)
    gemm.linear_bias_wgrad(dlogits, kept_of(n2), acc["head"])
    dn2 = gemm.linear_dgrad(dlogits, s["head"])
    dy = fused.layernorm_bwd(dn2, y, m2, r2, s["g2"], acc["g2"], acc["b2"], rows=rows)
    gemm.linear_bias_wgrad(dy, kept_of(h), acc["w2"], acc["c2"])
    dz = gemm.linear_act_dgrad(dy, s["w2"], z, "gelu_tanh", z_rows=rows)
    gemm.linear_bias_wgrad(dz, kept_of(n1), acc["w1"], acc["c1"])
    dn1 = gemm.linear_dgrad(dz, s["w1"])
    dx = fused.layernorm_bwd(dn1, s["x"], m1, r1, s["g1"], acc["g1"], acc["b1"], rows=rows, dres=dy)
    return {"kd": kd, "ce": ce, "dx": dx, **acc}


def student_case(dev, T=96, R=50, H=64, F=128, V=160, K=8, seed=7):
    g = gen(dev, seed)
    w = lambda *shape, scale, shift=0.0: rand(g, *shape, dtype=BF, scale=scale, shift=shift)  # noqa: E731
    s = {"x": w(T, H, scale=1.0), "w1": w(F, H, scale=H ** -0.5), "w2": w(H, F, scale=F ** -0.5),
         "c1": w(F, scale=0.3), "c2": w(H, scale=0.3), "g1": w(H, scale=0.2, shift=1.0),
         "g2": w(H, scale=0.2, shift=1.0), "b1": w(H, scale=0.2), "b2": w(H, scale=0.2),
         "head": w(V, H, scale=2.0 * H ** -0.5)}
    t = rand(g, T, V, scale=2.0)
    s["top"], s["ids"] = t.topk(K, dim=1)
    s["top_lse"] = (t.double() / 2.0).logsumexp(1).float()
    s["labels"] = torch.randint(-1, V, (T,), generator=g, device=dev)
    s["dkd"] = torch.rand(R, generator=g, device=dev)
    s["dce"] = torch.rand(R, generator=g, device=dev)
    return g, s, kept(g, T, R)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_step_of_a_student(dev):
    """Twelve roundings of half a bf16 step lie on the longest way through the block, its head and
    back, each of which moves a gradient by at most 2^-8 of its norm."""
    _, s, rows = student_case(dev)
    got = student_step(s, rows)
    again = student_step(s, rows)
    assert all(torch.equal(got[k], again[k]) for k in got)
    leaf = {k: s[k].double().requires_grad_() for k in ("x", "w1", "w2", "c1", "c2", "g1", "b1", "g2",
                                                        "b2", "head")}
    n1 = ln64(leaf["x"], leaf["g1"], leaf["b1"])[0]
    h = act64(n1 @ leaf["w1"].t() + leaf["c1"], "gelu_tanh")
    y = h @ leaf["w2"].t() + leaf["c2"] + leaf["x"]
    z = ln64(y, leaf["g2"], leaf["b2"])[0] @ leaf["head"].t()
    kd, ce = distill64({"logits": z, "top_ids": s["ids"], "top_logits": s["top"], "temperature": 2.0,
                        "top_lse": s["top_lse"], "labels": s["labels"]}, z)
    at = rows.long()
    # the gradient of what the kept rows' own losses say
    ((kd[at] * s["dkd"].double()).sum() + (ce[at] * s["dce"].double()).sum()).backward()
    want = {k: v.grad for k, v in leaf.items()}
    want["dx"] = want.pop("x")[at]
    for k, v in want.items():
        err = float((got[k].double() - v).norm() / v.norm())
        assert err < 12 * 2.0 ** -8, (k, err)
    for k, v in (("kd", kd), ("ce", ce)):
        assert float((got[k].double() - v.detach()).norm() / v.detach().norm()) < 5 * 2.0 ** -8


@pytest.mark.gpu
def test_student_captured_and_replayed_with_other_inputs():
    cases = [student_case("cuda", seed=s, **k) for s, k in
             ((1, {}), (2, dict(T=700, R=333, H=256, F=1024, V=2048, K=40)))]
    for _, s, rows in cases:
        student_step(s, rows)
    torch.cuda.synchronize()
    graphs = []
    for _, s, rows in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = student_step(s, rows)
        graphs.append((graph, res))
    for turn in range(3):
        for graph, _ in graphs:
            graph.replay()
        for (_, res), (_, s, rows) in zip(graphs, cases):
            want = student_step(s, rows)
            assert all(torch.equal(res[k], want[k]) for k in want)
        for g, s, rows in cases:  # new values in the same places
            for k in ("x", "w1", "c2", "g2", "head", "top"):
                s[k].copy_(rand(g, *s[k].shape, scale=0.3 * (turn + 1)))
            s["labels"].copy_(torch.randint(-1, 160, s["labels"].shape, generator=g, device="cuda"))


@pytest.mark.gpu
def test_student_on_two_streams_at_once():
    cases = [student_case("cuda", seed=s, T=500, R=222, H=128, F=512, V=1056, K=33) for s in (3, 4)]
    want = [student_step(s, rows) for _, s, rows in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for st, (_, s, rows) in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append(student_step(s, rows))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(a[k], b[k]) for k in b)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["logits", "norm", "linear"])
def test_offsets_past_32_bits(kind):
    """More than 2^31 elements: the last rows against the same rows alone."""
    g = gen("cuda", 9)
    if kind == "logits":
        T, V = 17000, 128256
        z = torch.empty(T, V, dtype=BF, device="cuda")
        z[-40:] = rand(g, 40, V, dtype=BF, scale=2.0)
        z[:-40] = 0.0
        t, ids = z[-40:].float().topk(6, dim=1)
        top, all_ids = torch.zeros(T, 6, device="cuda"), torch.zeros(T, 6, dtype=torch.int32, device="cuda")
        top[-40:], all_ids[-40:] = t, ids.int()
        kd, _, _, stats = fused.distill_fwd(z, all_ids, top, 2.0)
        want = fused.distill_fwd(z[-40:], ids.int(), t, 2.0)
        # rows alone may be split over blocks, whose sums are joined in another order
        assert torch.allclose(kd[-40:], want[0], rtol=1e-5, atol=1e-5)
        d = torch.ones(T, device="cuda")
        got = fused.distill_bwd(z, all_ids, top, stats, d, 2.0, out=z.clone())
        alone = fused.distill_bwd(z[-40:], ids.int(), t, stats[-40:].contiguous(), d[:40], 2.0)
        assert torch.equal(got[-40:], alone)
    elif kind == "norm":
        T, H = 530000, 4096
        x = torch.zeros(T, H, dtype=BF, device="cuda")
        x[-9:] = rand(g, 9, H, dtype=BF)
        w = rand(g, H, dtype=BF)
        y, mean, rstd = fused.layernorm_fwd(x, w, w, EPS)
        assert torch.equal(y[-9:], fused.layernorm_fwd(x[-9:], w, w, EPS)[0])
        rows = torch.arange(T - 9, T, dtype=torch.int32, device="cuda")
        dy = rand(g, 9, H, dtype=BF)
        dx = fused.layernorm_bwd(dy, x, mean, rstd, w, None, None, rows=rows)
        assert torch.equal(dx, fused.layernorm_bwd(dy, x[-9:], mean[-9:], rstd[-9:], w, None, None))
    else:
        M, N, K = 70000, 32768, 64
        x, w = rand(g, M, K, dtype=BF), rand(g, N, K, dtype=BF)
        z = torch.empty(M, N, dtype=BF, device="cuda")
        y = gemm.linear_act_fwd(x, w, act="relu", z=z)
        want = x[-50:].double() @ w.double().t()
        tol = 2 * (K + 2) * U * (x[-50:].double().abs() @ w.double().abs().t())
        close(z[-50:], want, tol, "z")
        close(y[-50:], want.clamp(min=0), tol, "y")
        rows = torch.arange(M - 300, M, dtype=torch.int32, device="cuda")
        dy, w2 = rand(g, 300, K, dtype=BF), rand(g, K, N, dtype=BF)
        dz = gemm.linear_act_dgrad(dy, w2, z, "relu", z_rows=rows)
        assert torch.equal(dz, gemm.linear_act_dgrad(dy, w2, z[-300:], "relu"))
