"""The row operators around the blocks: scaled embedding and its gradient, the norms after and before
a block, and clipping of a gradient list, against their formulas in 64 bits.

Tolerances are bounds on the rounding errors of the arithmetic, element by element: u = 2^-24 for an
fp32 operation, k u sum|x| for a sum whose longest chain has k additions, and half a step of the
output's type for its one rounding.
"""
import math

import pytest
import torch

from centrifuge_b200.ops import fused

U = 2.0 ** -24
EPS = 1e-5
CPU_GPU = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def half_step(t):
    """Half a step of type t relative to the value, and its smallest absolute half step."""
    return torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def close(got, want, tol, what):
    """|got - want| <= tol everywhere, after the rounding to got's type."""
    rel, tiny = half_step(got.dtype)
    bound = tol + rel * (want.abs() + tol) + tiny
    bad = ~((got.double() - want).abs() <= bound)
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


# ---------------------------------------------------------------- scaled embedding
@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("V,H,R,dtype,out,ids32,pad", [
    (50, 256, 300, BF, BF, False, 0), (50, 8, 1, HF, HF, True, 0), (7, 1, 33, F32, F32, False, 0),
    (1, 250, 5, BF, F32, True, 0), (300, 1000, 77, HF, F32, False, 8), (90, 255, 40, BF, BF, True, 3),
    (33, 2048, 64, F32, BF, False, 0), (20, 4104, 9, BF, HF, False, 8), (20, 64, 0, BF, BF, False, 0),
])
def test_scaled_embedding_fwd(dev, V, H, R, dtype, out, ids32, pad):
    g = gen(dev, V + H)
    table = rand(g, V, H, dtype=dtype, pad=pad)
    ids = torch.randint(0, V, (R,), generator=g, device=dev)
    ids = ids.int() if ids32 else ids
    o = None if out == dtype and not pad else torch.empty(R, H + pad, dtype=out, device=dev)[:, :H]
    got = fused.scaled_embedding_fwd(table, ids, math.sqrt(H), out=o)
    assert got.dtype == out and got.shape == (R, H) and (o is None or got is o)
    want = table[ids.long()].double() * math.sqrt(H)
    close(got, want, 2 * U * want.abs(), "out")  # the scale and the product are rounded to fp32


def grad_of_table(dy, tok, V, scale):
    """The gradient and the bound of an fp32 sum of each token's rows, in 64 bits."""
    z = torch.zeros(V, dy.shape[1], dtype=torch.float64, device=dy.device)
    count = torch.bincount(tok, minlength=V).double().unsqueeze(1)
    mass = z.clone().index_add_(0, tok, dy.double().abs()) * scale
    return z.clone().index_add_(0, tok, dy.double()) * scale, (count + 3) * U * mass


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("V,H,T,R,dtype,ids32,kind", [
    (1024, 256, 256, 128, BF, False, "uniform"), (1024, 256, 1, 1, BF, True, "uniform"),
    (5, 8, 400, 400, HF, False, "uniform"), (1, 64, 333, 200, F32, False, "uniform"),
    (3000, 1000, 3000, 3000, BF, False, "text"), (3000, 250, 1000, 999, BF, True, "text"),
    (70000, 64, 5000, 4097, BF, False, "text"), (200000, 8, 700, 700, F32, False, "uniform"),
    (2000, 2056, 900, 900, HF, False, "one"), (500, 96, 4000, 3333, BF, False, "half"),
    (32, 33, 64, 64, F32, False, "runs"), (32, 7, 33, 32, BF, True, "runs"),
    (40, 2048, 70, 65, F32, False, "text"), (40, 2500, 70, 65, BF, False, "text"),
    (64, 16, 100, 0, BF, False, "uniform"), (50, 1030, 200, 192, BF, False, "one"),
    (50, 1032, 200, 193, BF, False, "half"), (50, 1032, 300, 256, F32, False, "one"),
    (50, 1031, 300, 256, HF, False, "half"), (50, 1032, 300, 257, BF, False, "one"),
    (50, 1031, 300, 257, F32, False, "half"), (50, 2048, 512, 511, BF, False, "half"),
    (900, 300, 513, 513, HF, True, "text"), (7, 520, 600, 129, F32, False, "one"),
    (300, 1033, 500, 130, BF, False, "text"),
])
@pytest.mark.parametrize("accumulate,pad", [(True, None), (False, 3), (False, None)])
def test_scaled_embedding_bwd(dev, V, H, T, R, dtype, ids32, kind, accumulate, pad):
    g = gen(dev, V + H + T)
    if kind == "uniform":
        ids = torch.randint(0, V, (T,), generator=g, device=dev)
    elif kind == "text":
        u = torch.rand(T, generator=g, device=dev, dtype=torch.float64)
        ids = (torch.exp(u * math.log(V)) - 1).long().clamp(0, V - 1)
    elif kind == "one":
        ids = torch.full((T,), V - 1, device=dev)
    elif kind == "half":
        ids = torch.randint(0, V, (T,), generator=g, device=dev)
        ids[torch.rand(T, generator=g, device=dev) < 0.5] = 3
    else:  # sorted runs whose borders fall on and beside multiples of 32
        ids = (torch.arange(T, device=dev) + 1) // 31 % V
    ids = ids.int() if ids32 else ids
    rows = None
    if R != T:
        rows = torch.randperm(T, generator=g, device=dev)[:R].sort().values.int()
    dy = rand(g, R, H, dtype=dtype)
    before = rand(g, V, H)
    got = before.clone()
    res = fused.scaled_embedding_bwd(dy, ids, got, 1.7, id_rows=rows, padding_idx=pad,
                                     accumulate=accumulate)
    assert res is got
    tok = (ids if rows is None else ids[rows.long()]).long()
    keep = tok != (-1 if pad is None else pad)
    want, tol = grad_of_table(dy[keep], tok[keep], V, 1.7)
    if accumulate:
        want = want + before.double()
        tol = tol + 2 * U * want.abs()
    close(got, want, tol, "dtable")
    if not accumulate:  # nothing of what the table held is left
        assert not got[torch.bincount(tok[keep], minlength=V) == 0].any()


@pytest.mark.gpu
def test_scaled_embedding_bwd_is_repeatable_and_takes_strides():
    g = gen("cuda", 5)
    ids = torch.randint(0, 300, (2, 3000), generator=g, device="cuda")
    ids[:, ::3] = 17
    dy = rand(g, 6000, 512, dtype=BF, pad=24)
    base = torch.zeros(300, 520, device="cuda")
    for a in (base[:, :512], torch.empty(300, 512, device="cuda")):
        runs = []
        for _ in range(3):
            a.zero_()
            runs.append(fused.scaled_embedding_bwd(dy, ids, a, 0.5).clone())
        assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
        want, tol = grad_of_table(dy, ids.reshape(-1), 300, 0.5)
        close(runs[0], want, tol, "dtable")
    assert not base[:, 512:].any()  # behind the rows nothing is written
    base.fill_(7.0)
    fused.scaled_embedding_bwd(dy, ids, base[:, :512], 0.5, accumulate=False)
    assert torch.equal(base[:, :512], runs[0]) and bool((base[:, 512:] == 7.0).all())
    # rows that begin off the vector borders
    off = torch.zeros(300, 515, device="cuda")[:, 1:514]
    fused.scaled_embedding_bwd(rand(g, 6000, 513, dtype=BF, skew=3), ids, off)
    assert bool(off.any())


@pytest.mark.gpu
def test_scaled_embedding_reports_bad_indices():
    from centrifuge_b200.ops._ext import kernels
    status = kernels().status_block(0)
    status.zero_()
    g = gen("cuda", 6)
    table = rand(g, 64, 128, dtype=BF)
    ids = torch.tensor([3, 64, 5, -1, 1 << 40], device="cuda")
    out = fused.scaled_embedding_fwd(table, ids, 2.0)
    assert int(status[0]) == 128 and not out[[1, 3, 4]].any()
    assert torch.equal(out[[0, 2]], table[[3, 5]] * 2)
    status.zero_()
    dy = rand(g, 3, 128, dtype=BF)
    for rows in ([0, 1, 2], [0, 3, 9], [0, 4, -5]):
        dt = torch.zeros(64, 128, device="cuda")
        rid = torch.tensor(rows, dtype=torch.int32, device="cuda")
        fused.scaled_embedding_bwd(dy, ids, dt, id_rows=rid)
        assert int(status[0]) == 128
        status.zero_()
        assert torch.equal(dt[3], dy[0].float())
        used = [3] + ([5] if rows[2] == 2 else [])
        dt[used] = 0
        assert not dt.any()


@pytest.mark.gpu
@pytest.mark.parametrize("ids32", [False, True])
@pytest.mark.parametrize("V,T,R", [(500, 300, 257), (500, 3000, 2900), (200000, 3000, 2900),
                                   (500, 50000, 40000)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_table_gradient_of_many_rows_reports_bad_indices(ids32, V, T, R, accumulate):
    """Tokens and row ids out of range among rows that are sorted: recorded, and nothing else moves."""
    from centrifuge_b200.ops._ext import kernels
    status = kernels().status_block(0)
    g = gen("cuda", V + R)
    good_ids = torch.randint(0, V, (T,), generator=g, device="cuda")
    good_rows = torch.randperm(T, generator=g, device="cuda")[:R]
    bad_tokens = [-1, V, -V, (1 << 31) - 1, -(1 << 31)] + ([] if ids32 else [1 << 31, 1 << 32, 1 << 40])
    bad_rows = [-1, T, (1 << 31) - 1, -(1 << 31)]
    dy = rand(g, R, 24, dtype=BF)
    before = rand(g, V, 24)

    def check(ids, rows, keep, code):
        status.zero_()
        got = before.clone()
        fused.scaled_embedding_bwd(dy, ids.int() if ids32 else ids, got, 0.5, id_rows=rows.int(),
                                   accumulate=accumulate)
        assert int(status[0]) == code
        status.zero_()
        want, tol = grad_of_table(dy[keep], good_ids[good_rows[keep]], V, 0.5)
        if accumulate:
            want = want + before.double()
            tol = tol + 2 * U * want.abs()
        close(got, want, tol, "dtable")

    check(good_ids, good_rows, torch.ones(R, dtype=torch.bool, device="cuda"), 0)
    some = torch.arange(0, R, 7, device="cuda")  # the rows that are made bad
    some = some[: len(some) // len(bad_tokens) * len(bad_tokens)]
    ids = good_ids.clone()
    ids[good_rows[some]] = torch.tensor(bad_tokens, device="cuda").repeat(len(some) // len(bad_tokens))
    keep = torch.ones(R, dtype=torch.bool, device="cuda")
    keep[some] = False
    check(ids, good_rows, keep, 128)
    rows = good_rows.clone()
    rows[some] = torch.tensor(bad_rows, device="cuda").repeat(len(some))[:len(some)]
    check(good_ids, rows, keep, 128)
    one = good_ids.clone()  # a single one, in the last row
    one[good_rows[-1]] = V
    keep[:] = True
    keep[-1] = False
    check(one, good_rows, keep, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("V,H,R,share", [(32000, 64, 40000, 0.3), (300, 65, 40000, 0.5),
                                         (140000, 32, 66000, 0.9), (32000, 40, 20000, 0.95)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_table_gradient_of_a_large_batch(V, H, R, share, accumulate):
    """Text and one frequent token, over and under the rows whose keys the sort holds."""
    g = gen("cuda", R + H)
    u = torch.rand(R, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(V)) - 1).long().clamp(0, V - 1)
    ids[torch.rand(R, generator=g, device="cuda") < share] = V // 2
    dy = rand(g, R, H, dtype=BF)
    before = rand(g, V, H)
    got = before.clone()
    fused.scaled_embedding_bwd(dy, ids, got, 1.5, accumulate=accumulate)
    want, tol = grad_of_table(dy, ids, V, 1.5)
    if accumulate:
        want = want + before.double()
        tol = tol + 2 * U * want.abs()
    close(got, want, tol, "dtable")


@pytest.mark.gpu
@pytest.mark.parametrize("run", [16, 17, 143, 144, 145, 160, 4095, 4096, 4097, 4112, 4113, 4128, 8192,
                                 8208, 8209, 9000])
@pytest.mark.parametrize("H", [16, 9])
def test_table_gradient_of_one_run(run, H):
    """The first token in `run` of 9000 rows: chunks of 16 rows, the join's share of one warp (eight
    more chunks) and its steps of 256 chunks begin and end there."""
    g = gen("cuda", run)
    ids = torch.arange(9000, device="cuda") % 77 + 1
    ids[:run] = 0
    ids = ids[torch.randperm(9000, generator=g, device="cuda")]
    dy = rand(g, 9000, H, dtype=HF)
    got = torch.full((100, H), 5.0, device="cuda")
    fused.scaled_embedding_bwd(dy, ids, got, accumulate=False)
    close(got, *grad_of_table(dy, ids, 100, 1.0), "dtable")


@pytest.mark.gpu
@pytest.mark.parametrize("R,H", [(6000, 513), (6000, 512), (200, 513), (200, 512), (6000, 3)])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("accumulate", [False, True])
def test_table_gradient_off_the_vector_borders(R, H, dtype, accumulate):
    """Rows that begin anywhere, by value; nothing beside the table's columns is written."""
    g = gen("cuda", R + H)
    ids = torch.randint(0, 290, (R,), generator=g, device="cuda")
    ids[::5] = 7
    dy = rand(g, R, H, dtype=dtype, skew=3)
    base = rand(g, 300, H + 4)
    keep = base.clone()
    got = base[:, 1:H + 1]
    fused.scaled_embedding_bwd(dy, ids, got, 0.5, accumulate=accumulate)
    want, tol = grad_of_table(dy, ids, 300, 0.5)
    if accumulate:
        want = want + keep[:, 1:H + 1].double()
        tol = tol + 2 * U * want.abs()
    close(got, want, tol, "dtable")
    assert torch.equal(base[:, 0], keep[:, 0]) and torch.equal(base[:, H + 1:], keep[:, H + 1:])


@pytest.mark.parametrize("dev", CPU_GPU)
def test_scaled_embedding_refuses_the_too_large(dev):
    """Widths whose slabs no grid has, before anything of the table is written, and padding tokens
    that the sort cannot compare."""
    ids = torch.zeros(300, dtype=torch.long, device=dev)
    dt = torch.ones(1, 65535 * 128 + 1, device=dev)
    dy = torch.ones(1, dt.shape[1], dtype=BF, device=dev)
    for call in (lambda: fused.scaled_embedding_bwd(dy, ids[:1], dt),
                 lambda: fused.scaled_embedding_fwd(dy, ids)):
        with pytest.raises(ValueError, match="over 8388480"):
            call()
    assert bool((dt == 1.0).all())
    if dev == "cuda":
        from centrifuge_b200.ops._ext import kernels
        kernels().status_block(0).zero_()
    for rows in (3, 300):  # the largest padding token is no error, whatever the number of rows
        small = torch.zeros(4, 8, device=dev)
        pads = torch.full((rows,), (1 << 31) - 1, device=dev)
        one = torch.ones(rows, 8, device=dev)
        fused.scaled_embedding_bwd(one, pads, small, padding_idx=(1 << 31) - 1)
        assert not small.any()
        with pytest.raises(ValueError, match="over 31 bits"):
            fused.scaled_embedding_bwd(one, pads, small, padding_idx=1 << 31)
    if dev == "cuda":
        assert int(kernels().status_block(0)[0]) == 0


@pytest.mark.parametrize("bad", [-1, 8, 1 << 40])
def test_bad_indices_raise_on_the_cpu(bad):
    """The CPU path refuses ids and row ids outside their range; nothing counts from the end."""
    table, dy, dt = torch.ones(8, 16), torch.ones(3, 16), torch.zeros(8, 16)
    ids = torch.tensor([1, bad, 2])
    with pytest.raises(IndexError):
        fused.scaled_embedding_fwd(table, ids)
    with pytest.raises(IndexError):
        fused.scaled_embedding_bwd(dy, ids, dt, accumulate=False, padding_idx=1)
    h = torch.ones(8, 16)
    r, w = torch.ones(8), torch.ones(16)
    if bad < 1 << 31:
        rows = ids.int()
        with pytest.raises(IndexError):
            fused.scaled_embedding_bwd(dy, torch.arange(8), dt, id_rows=rows)
        with pytest.raises(IndexError):
            fused.block_norms_bwd(dy, dy, h, h, r, r, w, w, dt[0], dt[1], rows=rows)
    assert not dt.any()
    # a padding token adds nothing, wherever it lies
    fused.scaled_embedding_bwd(dy, torch.tensor([1, 9, 2]), dt, padding_idx=9)
    assert bool((dt[1:3] == 1.0).all()) and not dt[3:].any()


@pytest.mark.parametrize("dev", CPU_GPU)
def test_scaled_embedding_refuses_what_is_read_and_written(dev):
    """An output over an input of the same call; columns of one buffer's rows are apart."""
    buf = torch.zeros(8, 48, device=dev)
    ids = torch.zeros(8, dtype=torch.long, device=dev)
    a, b = buf[:, :16], buf[:, 16:32]
    a.fill_(3.0)
    for out in (a, buf[:, 8:24], buf.view(-1)[48:176].view(8, 16)):
        with pytest.raises(ValueError, match="overlap"):
            fused.scaled_embedding_fwd(a, ids, out=out)
        with pytest.raises(ValueError, match="overlap"):
            fused.scaled_embedding_bwd(a, ids, out)
    over_ids = torch.zeros(8 * 16, device=dev).view(8, 16)
    with pytest.raises(ValueError, match="overlap"):
        fused.scaled_embedding_fwd(a, over_ids.view(torch.long).view(-1)[8:16], out=over_ids)
    with pytest.raises(ValueError, match="overlap"):
        fused.scaled_embedding_bwd(a, over_ids.view(torch.long).view(-1)[8:16], over_ids)
    with pytest.raises(ValueError, match="overlap"):
        fused.scaled_embedding_bwd(a, ids, over_ids,
                                   id_rows=over_ids.view(torch.int32).view(-1)[:8])
    fused.scaled_embedding_fwd(a, ids, 2.0, out=b)
    assert bool((b == 6.0).all()) and not buf[:, 32:].any()
    fused.scaled_embedding_bwd(b, ids, a, 0.5)
    assert bool((a[0] == 27.0).all()) and bool((a[1:] == 3.0).all())
    fused.scaled_embedding_bwd(buf[7:, 32:], ids[:1], a, accumulate=False)  # one row in the gaps
    assert not a.any() and bool((b == 6.0).all())


# ---------------------------------------------------------------- norms around a block
def norms_case(dev, T, H, dtype, resid, gate, pre, pad=0, skew=0, seed=0):
    g = gen(dev, 1000 * T + H + seed)
    c = {"h": rand(g, T, H, dtype=dtype, pad=pad, skew=skew),
         "x": rand(g, T, H, dtype=resid, scale=2.0, pad=pad, skew=skew),
         "w_post": rand(g, H, dtype=dtype, scale=0.1, shift=1.0),
         "w_pre": rand(g, H, dtype=dtype, scale=0.1, shift=1.0) if pre else None}
    c["gate"] = {"none": lambda: None,
                 "channel": lambda: rand(g, H, dtype=dtype, scale=0.3, shift=0.5),
                 "token": lambda: rand(g, T, 1, pad=pad),
                 "element": lambda: rand(g, T, H, dtype=dtype, pad=pad, skew=skew)}[gate]()
    return g, c


def norms_formula(c, a, b):
    """Forward in 64 bits from fp64 leaves."""
    h = c["h"]
    rp = (h.square().mean(-1, keepdim=True) + EPS).rsqrt()
    br = b * h * rp * c["w_post"]
    if c["gate"] is not None:
        br = br * c["gate"]
    y = a * c["x"] + br
    if c["w_pre"] is None:
        return y, None, rp, None, br
    rq = (y.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return y, y * rq * c["w_pre"], rp, rq, br


def doubles(c):
    return {k: None if v is None else v.double() for k, v in c.items()}


NORM_CASES = [
    (256, 256, BF, BF, "none", True), (1, 8, BF, BF, "channel", True), (3, 1, F32, F32, "token", True),
    (17, 33, HF, HF, "element", True), (300, 250, BF, F32, "channel", True),
    (200, 1000, HF, HF, "none", False), (65, 512, BF, F32, "token", True),
    (129, 768, F32, F32, "element", True), (77, 2048, BF, BF, "channel", True),
    (300, 2048, BF, BF, "token", False), (40, 2049, BF, BF, "element", True),
    (33, 4096, BF, F32, "element", True), (19, 5632, HF, F32, "channel", False),
    (12, 8192, BF, BF, "token", True), (9, 8200, BF, BF, "channel", True),
    (5, 16384, F32, F32, "element", True), (4, 16383, BF, BF, "channel", True),
    (2500, 64, BF, BF, "channel", True), (2, 24, BF, BF, "channel", True),
]


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("T,H,dtype,resid,gate,pre", NORM_CASES)
@pytest.mark.parametrize("pad,skew", [(0, 0), (8, 0), (5, 1)])
def test_block_norms_fwd(dev, T, H, dtype, resid, gate, pre, pad, skew):
    _, c = norms_case(dev, T, H, dtype, resid, gate, pre, pad, skew)
    a, b = 0.75, 0.5  # exact in fp32
    y, n, rp, rq = fused.block_norms_fwd(c["h"], c["x"], c["w_post"], c["w_pre"], EPS,
                                         gate=c["gate"], block_scale=b, resid_scale=a)
    assert y.dtype == resid and rp.dtype == F32 and (n is None) == (rq is None) == (not pre)
    wy, wn, wp, wq, br = norms_formula(doubles(c), a, b)
    # a mean of squares: a chain of at most 128 additions and 10 exchanges, half of it in the root,
    # whose own error is at most two steps
    dr = 70 * U + 4 * U
    close(rp, wp.squeeze(1), dr * wp.squeeze(1), "rstd_post")
    dy = (dr + 6 * U) * br.abs() + 3 * U * (a * c["x"].double()).abs()
    close(y, wy, dy, "y")
    if pre:
        assert n.dtype == dtype
        moved = dy.norm(dim=1, keepdim=True) * wq / math.sqrt(H)  # what dy does to the root
        close(rq, wq.squeeze(1), ((dr + moved) * wq).squeeze(1), "rstd_pre")
        close(n, wn, (wq * c["w_pre"].double()).abs() * dy + wn.abs() * (dr + moved + 3 * U), "n")


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("T,H,dtype,resid,gate,pre", NORM_CASES)
@pytest.mark.parametrize("kept,accumulate,with_dy,pad,skew", [
    (False, False, True, 0, 0), (True, True, True, 8, 0), (True, False, False, 5, 1)])
def test_block_norms_bwd(dev, T, H, dtype, resid, gate, pre, kept, accumulate, with_dy, pad, skew):
    g, c = norms_case(dev, T, H, dtype, resid, gate, pre, pad, skew, seed=7)
    a, b = 0.75, 0.5
    y, _, rp, rq = fused.block_norms_fwd(c["h"], c["x"], c["w_post"], c["w_pre"], EPS,
                                         gate=c["gate"], block_scale=b, resid_scale=a)
    with_dy = with_dy or not pre
    R = max(1, T // 2) if kept else T
    rows = torch.randperm(T, generator=g, device=dev)[:R].sort().values.int() if kept else None
    at = torch.arange(T, device=dev) if rows is None else rows.long()
    dn = rand(g, R, H, dtype=dtype, pad=pad, skew=skew) if pre else None
    dy = rand(g, R, H, dtype=resid, pad=pad, skew=skew) if with_dy else None
    base = rand(g, 3, H)
    acc = base.clone()
    learned = c["gate"] is not None and c["gate"].dim() == 1
    dx, dh, dg = fused.block_norms_bwd(
        dy, dn, c["h"], y if pre else None, rp, rq, c["w_post"], c["w_pre"], acc[0],
        acc[1] if pre else None, gate=c["gate"], dgate=acc[2] if learned else None, block_scale=b,
        resid_scale=a, rows=rows, accumulate=accumulate)
    assert dx.dtype == resid and dh.dtype == dtype and dx.shape == dh.shape == (R, H)

    # the formulas at the saved statistics, in 64 bits, and the bounds
    d = doubles(c)
    h, r1, w1 = d["h"][at], rp[at].double().unsqueeze(1), d["w_post"]
    gt = torch.ones(1, 1, dtype=torch.float64, device=dev)
    if c["gate"] is not None:
        gt = d["gate"] if learned else d["gate"][at]
    up = torch.zeros(R, H, dtype=torch.float64, device=dev) if dy is None else dy.double()
    t_up = 4 * U * up.abs()
    K = 48 * U  # a chain of at most 16 products and 10 exchanges, and their roundings, twice over
    if pre:
        yy, r2 = y[at].double(), rq[at].double().unsqueeze(1)
        q = dn.double() * d["w_pre"]
        dot, mass = (q * yy).sum(1, keepdim=True), (q * yy).abs().sum(1, keepdim=True)
        part = yy * r2 ** 3 / H
        up = up + r2 * q - part * dot
        t_up = t_up + 4 * U * r2 * q.abs() + part.abs() * K * mass + 8 * U * (part * dot).abs()
        t_up = t_up + 2 * U * up.abs()
        s = dn.double() * yy * r2
        want = s.sum(0)
        tol = (R + 24) * U * s.abs().sum(0)
        if accumulate:
            want, tol = want + base[1].double(), tol + 2 * U * (want + base[1].double()).abs()
        close(acc[1], want, tol, "dw_pre")
    close(dx, a * up, a * t_up + 2 * U * up.abs(), "dx")
    v = b * up * gt * w1
    t_v = (b * gt * w1).abs() * t_up + 4 * U * v.abs()
    dot, mass = (v * h).sum(1, keepdim=True), (v * h).abs().sum(1, keepdim=True)
    t_dot = (t_v * h.abs()).sum(1, keepdim=True) + K * mass
    part = h * r1 ** 3 / H
    close(dh, r1 * v - part * dot,
          r1 * t_v + part.abs() * t_dot + 8 * U * (r1 * v.abs() + (part * dot).abs()), "dh")
    per = b * up * h * r1  # the gradient of gate times weight
    t_per = (b * h * r1).abs() * t_up + 4 * U * per.abs()

    def summed(got, want, tol, old, what):
        if accumulate:
            want, tol = want + old, tol + 2 * U * (want + old).abs()
        close(got, want, tol, what)

    summed(acc[0], (per * gt).sum(0),
           ((t_per * gt.abs()).sum(0) + (R + 24) * U * (per * gt).abs().sum(0)), base[0].double(),
           "dw_post")
    if learned:
        assert dg.data_ptr() == acc[2].data_ptr()
        summed(acc[2], (per * w1).sum(0),
               (t_per * w1.abs()).sum(0) + (R + 24) * U * (per * w1).abs().sum(0), base[2].double(),
               "dgate")
    elif c["gate"] is None:
        assert dg is None
    elif gate == "token" or H == 1 and dtype == F32:
        close(dg, (per * w1).sum(1, keepdim=True),
              (t_per * w1.abs()).sum(1, keepdim=True) + K * (per * w1).abs().sum(1, keepdim=True),
              "dgate")
    else:
        close(dg, per * w1, t_per * w1.abs() + 2 * U * (per * w1).abs(), "dgate")


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("gate", ["none", "channel", "token", "element"])
@pytest.mark.parametrize("T,H,dtype,resid,pre", [
    (61, 2400, BF, BF, True), (43, 3400, HF, HF, True), (29, 4800, BF, F32, True),
    (75, 1536, BF, F32, False), (31, 2401, BF, BF, False), (90, 96, HF, HF, False)])
def test_block_norms_at_widths_of_other_teams(dev, T, H, dtype, resid, gate, pre):
    """Every gate at the widths between the powers of two, and without the norm before a block."""
    test_block_norms_fwd(dev, T, H, dtype, resid, gate, pre, 0, 0)
    test_block_norms_bwd(dev, T, H, dtype, resid, gate, pre, True, True, True, 0, 0)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("gate", ["none", "channel", "token", "element"])
def test_block_norms_gradient_against_differences(dev, gate):
    """Central differences of the 64-bit formula along random directions."""
    g, c = norms_case(dev, 6, 40, F32, F32, gate, True, seed=3)
    a, b = 0.75, 0.5
    y, _, rp, rq = fused.block_norms_fwd(c["h"], c["x"], c["w_post"], c["w_pre"], EPS,
                                         gate=c["gate"], block_scale=b, resid_scale=a)
    dy, dn = rand(g, 6, 40), rand(g, 6, 40)
    acc = torch.zeros(3, 40, device=dev)
    dx, dh, dg = fused.block_norms_bwd(dy, dn, c["h"], y, rp, rq, c["w_post"], c["w_pre"], acc[0],
                                       acc[1], gate=c["gate"],
                                       dgate=acc[2] if gate == "channel" else None, block_scale=b,
                                       resid_scale=a)
    grads = {"h": dh, "x": dx, "w_post": acc[0], "w_pre": acc[1], "gate": dg}
    d = doubles(c)

    def loss(k, step):
        p = dict(d)
        p[k] = p[k] + step
        y_, n_, _, _, _ = norms_formula(p, a, b)
        return float((y_ * dy).sum() + (n_ * dn).sum())

    for k, grad in grads.items():
        if d[k] is None:
            continue
        way = torch.randn(d[k].shape, generator=g, device=dev, dtype=torch.float64)
        e = 1e-5
        diff = (loss(k, e * way) - loss(k, -e * way)) / (2 * e)
        # differences: e^2 of the third derivative and 1e-16 / e of the loss; the gradient: fp32
        mass = float((grad.double() * way).abs().sum())
        assert abs(float((grad.double() * way).sum()) - diff) < 1e-5 * (mass + 1), k


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("accumulate", [True, False])
@pytest.mark.parametrize("which", [(0, 0, 1), (0, 1, 0), (0, 1, 1), (0, 0, 0)])
@pytest.mark.parametrize("T,H,dtype", [(300, 2048, BF), (40, 2049, F32), (0, 64, HF)])
def test_block_norms_bwd_of_a_shared_parameter(dev, accumulate, which, T, H, dtype):
    """One buffer for two or all of dw_post, dw_pre and dgate gets the sum of their gradients."""
    g, c = norms_case(dev, T, H, dtype, dtype, "channel", True, seed=9)
    y, _, rp, rq = fused.block_norms_fwd(c["h"], c["x"], c["w_post"], c["w_pre"], EPS, c["gate"])
    dy, dn = rand(g, T, H, dtype=dtype), rand(g, T, H, dtype=dtype)

    def grads(a, b, d, accumulate):
        fused.block_norms_bwd(dy, dn, c["h"], y, rp, rq, c["w_post"], c["w_pre"], a, b,
                              gate=c["gate"], dgate=d, accumulate=accumulate)

    alone = torch.empty(3, H, device=dev)
    grads(*alone, False)
    base = rand(g, 2, H)
    for _ in range(3):
        acc = base.clone()
        grads(*(acc[i] for i in which), accumulate)
        for i in range(max(which) + 1):
            parts = [alone[k].double() for k in range(3) if which[k] == i]
            if accumulate:
                parts.append(base[i].double())
            # each gradient is rounded once alone (its product with the gate or the weight, where the
            # sum may fuse it) and once in the sum, which has at most four terms
            close(acc[i], sum(parts), 4 * U * sum(p.abs() for p in parts), f"buffer {i}")
    buf = torch.zeros(2 * H, device=dev)
    for a, b, d in ((buf[:H], buf[1:H + 1], alone[2]), (alone[0], buf[:H], buf[H - 1:2 * H - 1])):
        with pytest.raises(ValueError, match="overlap in part"):
            grads(a, b, d, accumulate)
    if dtype == F32:
        for over in ("w_post", "w_pre", "gate"):
            with pytest.raises(ValueError, match="overlaps a weight or the gate"):
                grads(alone[0], alone[1], c[over], accumulate)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_block_norms_odd_values(dev):
    """Rows of zeros stay finite; what is no number in one row stays in its row; no rows at all."""
    _, c = norms_case(dev, 5, 64, BF, BF, "channel", True)
    c["h"][1] = 0
    c["x"][1] = 0
    c["h"][3, 5] = float("nan")
    c["x"][4, 6] = float("inf")
    y, n, rp, rq = fused.block_norms_fwd(c["h"], c["x"], c["w_post"], c["w_pre"], EPS, c["gate"])
    assert not y[1].any() and not n[1].any()
    for t in (y, n):
        assert bool(torch.isfinite(t[:3]).all()) and bool(t[3].isnan().any())
    assert bool(y[4].isinf().any()) and bool(torch.isfinite(rp[[0, 1, 2, 4]]).all())
    acc = torch.ones(3, 64, device=dev)
    d = torch.zeros(0, 64, dtype=BF, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    for accumulate in (True, False):
        dx, dh, _ = fused.block_norms_bwd(d, d, c["h"], y, rp, rq, c["w_post"], c["w_pre"], acc[0],
                                          acc[1], c["gate"], acc[2], rows=none,
                                          accumulate=accumulate)
        assert dx.shape == dh.shape == (0, 64)
        assert bool((acc == (1.0 if accumulate else 0.0)).all())
    y, n, _, _ = fused.block_norms_fwd(d, d, c["w_post"], c["w_pre"], EPS)
    assert y.shape == n.shape == (0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "token", "element"])
@pytest.mark.parametrize("pre", [True, False])
def test_block_norms_bwd_reports_bad_rows(gate, pre):
    from centrifuge_b200.ops._ext import kernels
    status = kernels().status_block(0)
    status.zero_()
    g, c = norms_case("cuda", 2000, 512, BF, BF, gate, pre)
    y, _, rp, rq = fused.block_norms_fwd(c["h"], c["x"], c["w_post"], c["w_pre"], EPS, c["gate"])
    rows = torch.arange(2000, dtype=torch.int32, device="cuda")
    good = rows % 3 != 0
    bad = torch.where(good, rows, torch.where(rows % 2 == 0, -1 - rows, 2000 + rows))
    dy = rand(g, 2000, 512, dtype=BF)
    res = []
    for ids, w in ((bad, 1.0), (rows, good.unsqueeze(1).to(BF))):
        acc = torch.zeros(2, 512, device="cuda")
        d = dy * w
        dx, dh, dg = fused.block_norms_bwd(d, d if pre else None, c["h"], y if pre else None, rp, rq,
                                           c["w_post"], c["w_pre"], acc[0], acc[1] if pre else None,
                                           gate=c["gate"], rows=ids)
        res.append((dx, dh, acc, *([] if dg is None else [dg])))
        assert int(status[0]) == (128 if ids is bad else 0)
        status.zero_()
    for p, q in zip(*res):
        assert torch.equal(p, q)  # the bad rows add nothing and come back as zeros


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,dtype,resid", [(1000, 513, BF, BF), (1000, 250, HF, F32),
                                             (700, 2048, F32, F32), (400, 8200, BF, BF),
                                             (400, 8192, BF, F32), (300, 2050, BF, BF),
                                             (900, 256, BF, BF), (300, 4096, BF, F32)])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "element"])
@pytest.mark.parametrize("pre", [True, False])
def test_block_norms_bwd_reports_bad_rows_at_other_widths(T, H, dtype, resid, gate, pre):
    """The kernels beside the ring, and its other teams: a row id out of range is recorded, gives zero
    rows and adds nothing."""
    from centrifuge_b200.ops._ext import kernels
    status = kernels().status_block(0)
    status.zero_()
    g, c = norms_case("cuda", T, H, dtype, resid, gate, pre)
    y, _, rp, rq = fused.block_norms_fwd(c["h"], c["x"], c["w_post"], c["w_pre"], EPS, c["gate"])
    rows = torch.arange(T, dtype=torch.int32, device="cuda")
    good = rows % 3 != 0
    out = torch.where(rows % 2 == 0, -1 - rows, T + rows)
    bad = torch.where(good, rows, torch.where(rows % 9 == 0, (1 << 31) - 1 - rows, out))
    dy, dn = rand(g, T, H, dtype=resid), rand(g, T, H, dtype=dtype)
    res = []
    for ids, w in ((bad, good.new_ones(T, 1)), (rows, good.unsqueeze(1))):
        acc = torch.zeros(3, H, device="cuda")
        dx, dh, dg = fused.block_norms_bwd(
            dy * w, dn * w if pre else None, c["h"], y if pre else None, rp, rq, c["w_post"],
            c["w_pre"], acc[0], acc[1] if pre else None, gate=c["gate"],
            dgate=acc[2] if gate == "channel" else None, rows=ids)
        res.append((dx, dh, acc, *([] if dg is None else [dg])))
        assert int(status[0]) == (128 if ids is bad else 0)
        status.zero_()
    for p, q in zip(*res):
        assert bool(p.any()) and torch.equal(p, q)


# ---------------------------------------------------------------- gradient lists
def grad_list(dev, sizes, types, seed=0, skew=0):
    g = gen(dev, seed)
    got = []
    for i, n in enumerate(sizes):
        t = rand(g, n + skew, dtype=types[i % len(types)], scale=0.01)
        got.append(t[skew:])
    return got


LISTS = {
    "one": [1], "tiny": [1, 2, 3, 0, 7, 8, 9], "borders": [32767, 32768, 32769, 65536, 65537, 1],
    "mixed": [100000, 17, 0, 70001, 5, 256, 33000], "many": [13] * 300, "groups": [3, 40] * 700,
    "large": [5_000_001, 12],
}


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("types", [(F32,), (BF,), (F32, BF, HF)])
@pytest.mark.parametrize("out_type", [None, F32, BF])
@pytest.mark.parametrize("over,skew", [(3.0, 0), (3.0, 1), (0.5, 0)])
def test_grad_list_clip(dev, name, types, out_type, over, skew):
    grads = grad_list(dev, LISTS[name], types, seed=len(name), skew=skew)
    want = [g.double() for g in grads]
    norm = math.sqrt(sum(float(g.square().sum()) for g in want)) * 0.25
    max_norm = norm / over
    outs = None if out_type is None else [torch.empty(g.numel() + skew, dtype=out_type, device=dev)[skew:]
                                          for g in grads]
    got_norm = fused.grad_list_clip_(grads, max_norm, extra_scale=0.25, out=outs)
    # squares: a thread's chain of 128 additions in fp32, half of it in the root; the partial sums
    # and the norm are rounded once each
    dn = (70 + 4) * U
    assert got_norm.shape == (1,) and abs(float(got_norm) - norm) <= dn * norm
    k = 0.25 * min(1.0, max_norm / (norm + 1e-6))
    for i, (g, w) in enumerate(zip(grads if outs is None else outs, want)):
        close(g, w * k, (w * k).abs() * (dn + 4 * U), f"tensor {i}")


@pytest.mark.parametrize("dev", CPU_GPU)
def test_grad_list_in_place_and_dense_layouts(dev):
    grads = [torch.randn(30, 50, device=dev).t(), torch.randn(2, 3, 4, 5, device=dev).permute(0, 2, 3, 1),
             torch.randn((), device=dev)]
    keep = [g.clone() for g in grads]
    ptrs = [g.data_ptr() for g in grads]
    big = float(sum(g.double().square().sum() for g in keep).sqrt()) * 2
    fused.grad_list_clip_(grads, big)  # under the limit: not a bit changes
    assert all(torch.equal(g, k) for g, k in zip(grads, keep))
    n1 = fused.grad_list_clip_(grads, 1.0)
    n2 = fused.grad_list_clip_(grads, 0.0)  # no limit
    assert [g.data_ptr() for g in grads] == ptrs
    assert abs(float(n2) - 1.0) < 1e-5 and float(n1) == pytest.approx(big / 2, rel=1e-5)
    for g, k in zip(grads, keep):
        assert torch.allclose(g, k / float(n1), rtol=1e-5, atol=0)
    # one output is its gradient, the other another tensor
    other = torch.empty_like(grads[1])
    fused.grad_list_clip_([grads[0], grads[1]], 0.5, out=[grads[0], other])
    assert float(sum(t.double().square().sum() for t in (grads[0], other)).sqrt()) == pytest.approx(
        0.5, rel=1e-4)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_grad_list_norm_of_odd_values(dev):
    for bad in (float("inf"), float("nan")):
        grads = [torch.ones(100, device=dev), torch.ones(5, device=dev)]
        grads[1][2] = bad
        norm = fused.grad_list_clip_(grads, 1.0)
        if math.isinf(bad):  # a limit of zero: what was finite is zero, infinity is no number
            assert math.isinf(float(norm)) and not grads[0].any() and bool(grads[1][2].isnan())
        else:
            assert math.isnan(float(norm)) and bool(grads[0].isnan().all())
    zeros = [torch.zeros(10, device=dev)]
    assert float(fused.grad_list_clip_(zeros, 1.0)) == 0.0 and not zeros[0].any()
    empty = [torch.empty(0, device=dev)]
    assert float(fused.grad_list_clip_(empty, 1.0)) == 0.0
    assert float(fused.grad_list_clip_([], 1.0)) == 0.0


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("value,n", [(1.7e18, 100), (1.5e19, 1), (1.1e-19, 70000), (3e-18, 5)])
def test_grad_list_norm_of_large_and_small_values(dev, value, n):
    """Sums of squares up to 3.4e38, and squares down to 1.2e-38, keep the bound of the norm."""
    g = torch.full((n,), value, device=dev)
    norm = fused.grad_list_clip_([g], 0.0)
    want = float(g[0].double()) * math.sqrt(n)
    assert abs(float(norm) - want) <= (70 + 4) * U * want
    assert float(fused.grad_list_sumsq([g]).double().sum()) == pytest.approx(want * want, rel=1e-5)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_grad_list_over_ranks_and_coef(dev):
    """Two lists whose sums of squares are added, as ranks with different parameters do it."""
    a, b = grad_list(dev, [1000, 77], (F32,), 1), grad_list(dev, [500], (BF,), 2)
    want = [g.double() for g in a + b]
    norm = math.sqrt(sum(float(g.square().sum()) for g in want))
    total = fused.grad_list_sumsq(a).sum() + fused.grad_list_sumsq(b).sum()
    for part in (a, b):
        n = fused.grad_list_clip_(part, norm / 2, extra_sumsq=total.view(1))
        assert float(n) == pytest.approx(norm, rel=1e-5)
    for g, w in zip(a + b, want):
        k = (norm / 2) / (norm + 1e-6)
        close(g, w * k, (w * k).abs() * 80 * U, "clipped")
    c = grad_list(dev, [1000, 77], (F32, BF), 1)
    ref = math.sqrt(sum(float(g.double().square().sum()) for g in c))
    coef, nrm = torch.empty(1, device=dev), torch.empty(1, device=dev)
    fused.grad_list_clip_coef(c, ref / 4, 0.5, coef, nrm)
    assert float(nrm) == pytest.approx(ref / 2, rel=1e-5)
    assert float(coef) == pytest.approx(0.25, rel=1e-4)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_grad_list_of_a_rank_without_parameters(dev):
    """The norm comes from the other ranks' sums; an output without a gradient is refused."""
    sums = torch.tensor([3.0, 6.0], device=dev)
    n = fused.grad_list_clip_([], 1.0, 0.5, extra_sumsq=sums)
    assert n.device == sums.device and n.shape == (1,) and float(n) == 1.5
    norm = torch.empty(1, device=dev)
    assert fused.grad_list_clip_([], 1.0, norm=norm, extra_sumsq=sums) is norm or dev == "cuda"
    assert float(norm) == 3.0 and float(fused.grad_list_clip_([], 1.0, norm=norm)) == 0.0
    with pytest.raises(ValueError):
        fused.grad_list_clip_([], 1.0, out=[norm])
    with pytest.raises(ValueError):
        fused.grad_list_clip_([], 1.0, norm=sums[:1], extra_sumsq=sums)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_grad_list_clip_refuses_a_norm_or_sums_in_the_list(dev):
    """What is written while other blocks read it, or read while others write it."""
    buf = torch.ones(300, device=dev)
    keep = buf.clone()
    g, o, sums, norm = buf[:100], buf[100:200], buf[200:208], buf[299:]
    for kw in (dict(norm=g[3:4]), dict(norm=g[99:]), dict(out=[o], norm=o[:1]),
               dict(out=[o], norm=g[:1]),  # o only: g is read
               dict(extra_sumsq=g[4:8]), dict(out=[o], extra_sumsq=buf[196:204]),
               dict(norm=sums[3:4], extra_sumsq=sums), dict(norm=sums[:1], extra_sumsq=sums)):
        with pytest.raises(ValueError, match="overlap"):
            fused.grad_list_clip_([g], 1.0, **kw)
        assert torch.equal(buf, keep)
    # sums in a gradient that is only read, and neighbours, are fine
    n = fused.grad_list_clip_([g], 1.0, out=[o], norm=norm, extra_sumsq=g[:16])
    assert n.data_ptr() == norm.data_ptr() and float(n) == 4.0
    assert torch.equal(g, keep[:100]) and torch.equal(sums, keep[200:208])
    close(o, torch.full((100,), 0.25 / (1 + 2.5e-7), dtype=torch.float64, device=dev),
          torch.full((100,), 4 * U, dtype=torch.float64, device=dev), "out")


@pytest.mark.parametrize("dev", CPU_GPU)
def test_grad_list_clip_checks_norm_and_sums(dev):
    """The CPU and the GPU take the same buffers: one fp32 element, and contiguous fp32 sums."""
    g = torch.full((4,), 2.0, device=dev)
    two = torch.zeros(2, device=dev)
    for kw in (dict(norm=two), dict(norm=two[:1].double()), dict(norm=two[:0]),
               dict(extra_sumsq=two.double()), dict(extra_sumsq=two.new_ones(6)[::2]),
               dict(extra_sumsq=two[:0])):
        with pytest.raises(ValueError):
            fused.grad_list_clip_([g], 1.0, **kw)
        assert bool((g == 2.0).all()) and not two.any()
    norm = torch.zeros((), device=dev)
    assert float(fused.grad_list_clip_([g], 8.0, norm=norm)) == 4.0 and float(norm) == 4.0


@pytest.mark.parametrize("dev", CPU_GPU)
def test_grad_list_clip_coef_checks_its_buffers(dev):
    """What the kernel writes is on its device; a list of bf16 tensors, its first one empty."""
    g = [torch.empty(0, dtype=BF, device=dev), torch.full((2, 8), 0.5, dtype=BF, device=dev)]
    one = torch.zeros(1, device=dev)
    bad = [one.double(), torch.zeros(2, device=dev), one[:0], one.int()]
    if dev == "cuda":
        bad.append(torch.zeros(1))
    for t in bad:
        for kw in (dict(coef=t, norm=one), dict(coef=one, norm=t)):
            with pytest.raises(ValueError):
                fused.grad_list_clip_coef(g, 1.0, 1.0, **kw)
    with pytest.raises(ValueError, match="empty list"):
        fused.grad_list_clip_coef([], 1.0, 1.0, one, one.clone())
    norm = one.clone()
    fused.grad_list_clip_coef(iter(g), 1.0, 1.0, one, norm)
    assert float(norm) == 2.0 and float(one) == pytest.approx(0.5, rel=1e-6)


# ---------------------------------------------------------------- launch counter
def test_launch_counter_adds_what_the_module_counts(monkeypatch):
    from centrifuge_b200.ops import _ext

    class Module:
        made = 5

        def row_launches(self):
            return self.made

    mod = Module()
    monkeypatch.setattr(_ext, "_mod", mod)
    counter = _ext.LaunchCounter()
    assert counter.reset() == 5 and counter.count == 0
    mod.made, counter.calls = 8, 2
    assert counter.count == 5 and counter.reset() == 5 and counter.reset() == 0


@pytest.mark.gpu
def test_launch_counter_of_the_row_operators():
    """As many as a call makes: they depend on rows, tensors and chunks."""
    from centrifuge_b200.ops._ext import counter
    g = gen("cuda", 3)

    def made(f):
        counter.reset()
        f()
        return counter.reset()

    ids = torch.randint(0, 40, (300,), generator=g, device="cuda")
    dy, dt = rand(g, 300, 64), torch.zeros(40, 64, device="cuda")
    assert made(lambda: fused.scaled_embedding_fwd(dt, ids)) == 1
    for rows, accumulate, n in ((0, True, 0), (0, False, 1), (1, True, 1), (256, False, 1),
                                (257, True, 3), (300, False, 3)):
        assert made(lambda: fused.scaled_embedding_bwd(dy[:rows], ids[:rows], dt,
                                                       accumulate=accumulate)) == n, rows
    h, w, acc = rand(g, 30, 64), torch.ones(64, device="cuda"), torch.zeros(2, 64, device="cuda")
    res = []
    assert made(lambda: res.extend(fused.block_norms_fwd(h, h, w, w, EPS))) == 1
    y, _, rp, rq = res
    for a, b, n in ((0, 1, 2), (1, 1, 3)):
        assert made(lambda: fused.block_norms_bwd(h, h, h, y, rp, rq, w, w, acc[a], acc[b])) == n
    part = rand(g, 40_000_000, scale=1e-3)
    sums = torch.ones(3, device="cuda")
    for grads, kw, n in (([h], {}, 2), ([h], dict(extra_sumsq=sums), 1), ([], dict(extra_sumsq=sums), 1),
                         ([part], {}, 3), (list(part[:1500].split(1)), {}, 5)):
        assert made(lambda: fused.grad_list_clip_(grads, 1.0, **kw)) == n, len(grads)
    assert made(lambda: fused.grad_list_sumsq([h, part])) == 1


# ---------------------------------------------------------------- refusals
@pytest.mark.parametrize("dev", CPU_GPU)
def test_refusals(dev):
    def t(*shape, dtype=F32):
        return torch.zeros(*shape, dtype=dtype, device=dev)

    def no(f, *args, **kw):
        with pytest.raises((ValueError, RuntimeError)):
            f(*args, **kw)

    ids = torch.zeros(4, dtype=torch.long, device=dev)
    no(fused.scaled_embedding_fwd, t(8, 16, dtype=torch.float64), ids)
    no(fused.scaled_embedding_fwd, t(16, 8).t(), ids)
    no(fused.scaled_embedding_fwd, t(8, 16), ids.float())
    no(fused.scaled_embedding_fwd, t(8, 16), ids, out=t(3, 16))
    no(fused.scaled_embedding_fwd, t(8, 16), ids, out=t(1, 16).expand(4, 16))
    dy, dt = t(4, 16), t(8, 16)
    no(fused.scaled_embedding_bwd, dy, ids[:3], dt)
    no(fused.scaled_embedding_bwd, dy, ids, t(8, 16, dtype=BF))
    no(fused.scaled_embedding_bwd, dy, ids, t(8, 15))
    no(fused.scaled_embedding_bwd, dy, ids, t(1, 16).expand(8, 16))
    no(fused.scaled_embedding_bwd, dy, ids, t(0, 16))
    no(fused.scaled_embedding_bwd, dy, ids, dt, padding_idx=-1)
    no(fused.scaled_embedding_bwd, dy, ids, dt, id_rows=ids)
    no(fused.scaled_embedding_bwd, dy, ids, dt, id_rows=ids[:3].int())

    h, x, w, r, z = t(4, 16, dtype=BF), t(4, 16, dtype=BF), t(16, dtype=BF), t(4), t(16)
    ok = dict(eps=EPS)
    no(fused.block_norms_fwd, h, t(4, 16, dtype=HF), w, w, **ok)
    no(fused.block_norms_fwd, h, t(3, 16, dtype=BF), w, w, **ok)
    no(fused.block_norms_fwd, h, x, t(15, dtype=BF), w, **ok)
    no(fused.block_norms_fwd, h, x, w.float(), w, **ok)
    no(fused.block_norms_fwd, h[0], x, w, w, **ok)
    no(fused.block_norms_fwd, h, x, w, w, gate=t(4, 1, dtype=BF), **ok)
    no(fused.block_norms_fwd, h, x, w, w, gate=t(3, 1), **ok)
    no(fused.block_norms_fwd, h, x, w, w, gate=t(1, 16, dtype=BF), **ok)
    big = t(1, 16392, dtype=BF)
    no(fused.block_norms_fwd, big, big, big[0], big[0], **ok)
    bwd = dict(dy=x, dn=h, h=h, y=x, rstd_post=r, rstd_pre=r, w_post=w, w_pre=w, dw_post=z.clone(),
               dw_pre=z.clone())
    fused.block_norms_bwd(**bwd)
    for change in (dict(dn=None), dict(w_pre=None), dict(y=None), dict(dw_pre=None),
                   dict(dy=x.float()), dict(dn=h.float()), dict(rstd_post=r[:3]),
                   dict(dw_post=w), dict(dgate=z), dict(gate=w), dict(gate=w, dgate=w),
                   dict(gate=t(4, 1), dgate=z), dict(rows=torch.zeros(4, device=dev)),
                   dict(rows=torch.zeros(3, dtype=torch.int32, device=dev)), dict(dy=x[:3])):
        no(fused.block_norms_bwd, **{**bwd, **change})
    no(fused.block_norms_bwd, **{**bwd, "dy": None, "dn": None, "w_pre": None, "y": None,
                                 "rstd_pre": None, "dw_pre": None})

    g = t(100)
    no(fused.grad_list_clip_, [g.double()], 1.0)
    no(fused.grad_list_clip_, [g], 1.0, extra_scale=0.0)
    no(fused.grad_list_clip_, [g], 1.0, out=[])
    no(fused.grad_list_clip_, [g], 1.0, out=[t(99)])
    no(fused.grad_list_sumsq, [])
    no(fused.grad_list_clip_, [g], 1.0, norm=z[:1], extra_sumsq=z[:1])
    no(fused.grad_list_clip_, [g], 1.0, norm=t(0))
    no(fused.grad_list_clip_, [g, g], 1.0)  # the same tensor twice
    no(fused.grad_list_clip_, [g[:60], g[50:]], 1.0)
    no(fused.grad_list_clip_, [t(100), t(100)], 1.0, out=[g[:], g[:]])
    no(fused.grad_list_clip_, [g[:50], t(50)], 1.0, out=[t(50), g[25:75]])
    no(fused.grad_list_clip_, [g[::2]], 1.0)
    no(fused.grad_list_clip_, [t(1).expand(10)], 1.0)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("dtype,tol", [
    (F32, 2e-5),  # some hundred roundings of 2^-24
    # about 13 roundings of half a bf16 step on the longest way through three blocks and back,
    # each of which moves a gradient by at most 2^-8 of its norm
    (BF, 13 * 2.0 ** -8)])
def test_step_of_a_model_with_norms_on_both_sides(dev, dtype, tol):
    """Scaled embedding, three linear blocks with the norms after and before them, the gradient on
    the kept rows only, and clipping of all gradients, against autograd in 64 bits."""
    g = gen(dev, 11)
    V, H, T, R, L = 60, 48, 90, 41, 3
    scale, a, b = 4.0, 0.75, 0.5
    table = rand(g, V, H, dtype=dtype, scale=0.25)
    ids = torch.randint(0, V // 4, (2, T // 2), generator=g, device=dev)
    rows = torch.randperm(T, generator=g, device=dev)[:R].sort().values.int()
    W = [rand(g, H, H, dtype=dtype, scale=H ** -0.5) for _ in range(L)]
    post = [rand(g, H, dtype=dtype, scale=0.1, shift=1.0) for _ in range(L)]
    pre = [rand(g, H, dtype=dtype, scale=0.1, shift=1.0) for _ in range(L)]
    gates = [torch.rand(T, 1, generator=g, device=dev), rand(g, H, dtype=dtype, shift=1.0),
             rand(g, T, H, dtype=dtype, shift=1.0)]
    c = rand(g, R, H, dtype=dtype)

    def one_step():
        x = n = fused.scaled_embedding_fwd(table, ids, scale)
        saved = []
        for i in range(L):
            h = n @ W[i]
            y, n_next, rp, rq = fused.block_norms_fwd(h, x, post[i], pre[i], EPS, gates[i], b, a)
            saved.append((n, h, y, rp, rq))
            x, n = y, n_next
        f32 = dict(dtype=F32, device=dev)
        dw = torch.zeros(L, 3, H, **f32)
        dW = torch.zeros(L, H, H, **f32)
        dE = torch.full((V, H), 7.0, **f32)
        dgate = [None] * L
        dy, dn = None, c
        for i in reversed(range(L)):
            n, h, y, rp, rq = saved[i]
            dy, dh, dgate[i] = fused.block_norms_bwd(
                dy, dn, h, y, rp, rq, post[i], pre[i], dw[i, 0], dw[i, 1], gate=gates[i],
                dgate=dw[i, 2] if i == 1 else None, block_scale=b, resid_scale=a, rows=rows)
            dW[i] = n[rows.long()].float().t() @ dh.float()
            dn = dh @ W[i].t()
        fused.scaled_embedding_bwd((dy.float() + dn.float()).to(dtype), ids, dE, scale,
                                   id_rows=rows, accumulate=False)
        grads = [dE, dW, dw]
        norm = fused.grad_list_clip_(grads, 0.5)
        return [*grads, dgate[0], dgate[2], norm]

    got = one_step()
    again = one_step()
    assert all(torch.equal(p, q) for p, q in zip(got, again))  # the same bits

    # the same in 64 bits, with the loss on the kept rows
    leaf = [t.double().requires_grad_() for t in (table, *W, *post, *pre, *gates)]
    E, w64, post64, pre64, g64 = (leaf[0], leaf[1:1 + L], leaf[1 + L:1 + 2 * L],
                                  leaf[1 + 2 * L:1 + 3 * L], leaf[1 + 3 * L:])
    x = n = E[ids.reshape(-1)] * scale
    for i in range(L):
        x, n, _, _, _ = norms_formula({"h": n @ w64[i], "x": x, "w_post": post64[i],
                                       "w_pre": pre64[i], "gate": g64[i]}, a, b)
    at = rows.long()
    (n[at] * c.double()).sum().backward()
    dw = torch.stack([torch.stack([post64[i].grad, pre64[i].grad,
                                   g64[1].grad if i == 1 else torch.zeros_like(post64[i])])
                      for i in range(L)])
    want = [E.grad, torch.stack([w.grad for w in w64]), dw]
    norm = math.sqrt(sum(float(t.square().sum()) for t in want))
    assert norm > 1.0
    want = [t * (0.5 / (norm + 1e-6)) for t in want] + [g64[0].grad[at], g64[2].grad[at],
                                                        torch.tensor([norm])]
    for p, q, what in zip(got, want, ("dE", "dW", "dw", "dgate token", "dgate element", "norm")):
        q = q.to(p.device)
        err = float((p.double() - q).norm() / q.norm())
        assert err < tol, (what, err)


# ---------------------------------------------------------------- streams, graphs, long offsets
def _all_operators(g, k=1.0):
    """Inputs on the GPU, and a call of every operator on them that returns what it writes."""
    T, R, H, V = 300, 200, 256, 500
    s = {"table": rand(g, V, H, dtype=BF, scale=k), "ids": torch.randint(0, V, (T,), generator=g, device="cuda"),
         "rows": torch.randperm(T, generator=g, device="cuda")[:R].sort().values.int(),
         "h": rand(g, T, H, dtype=BF), "x": rand(g, T, H, dtype=BF, scale=k),
         "w": rand(g, 2, H, dtype=BF, shift=1.0), "gate": rand(g, H, dtype=BF),
         "dy": rand(g, R, H, dtype=BF), "dn": rand(g, R, H, dtype=BF, scale=k),
         "grads": rand(g, 3, 40000, scale=k)}

    def call(s):
        e = fused.scaled_embedding_fwd(s["table"], s["ids"], 2.0)
        y, n, rp, rq = fused.block_norms_fwd(s["h"], s["x"], s["w"][0], s["w"][1], EPS, s["gate"])
        acc = torch.empty(3, H, device="cuda")
        dx, dh, _ = fused.block_norms_bwd(s["dy"], s["dn"], s["h"], y, rp, rq, s["w"][0], s["w"][1],
                                          acc[0], acc[1], s["gate"], acc[2], rows=s["rows"],
                                          accumulate=False)
        dE = torch.empty(V, H, device="cuda")
        fused.scaled_embedding_bwd(dx, s["ids"], dE, 2.0, id_rows=s["rows"], accumulate=False)
        few = torch.ones(V, H, device="cuda")
        fused.scaled_embedding_bwd(dx[:50], s["ids"], few, 2.0, id_rows=s["rows"][:50])
        out = torch.empty(3, 40000, dtype=BF, device="cuda")
        norm = fused.grad_list_clip_(list(s["grads"]), 1.0, out=list(out))
        return [e, y, n, rp, rq, dx, dh, acc, dE, few, out, norm]

    return s, call


@pytest.mark.gpu
def test_captured_and_replayed_with_other_inputs():
    """Two graphs of the same calls, replayed in turn and with new inputs in place of the old."""
    g = gen("cuda", 21)
    sets = [_all_operators(g, k) for k in (1.0, 3.0)]
    for s, call in sets:
        call(s)
    torch.cuda.synchronize()
    graphs = []
    for s, call in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = call(s)
        graphs.append((graph, res))
    for turn in range(3):
        for (graph, res), (s, call) in zip(graphs, sets):
            graph.replay()
        for (graph, res), (s, call) in zip(graphs, sets):
            want = call(s)
            assert all(torch.equal(p, q) for p, q in zip(res, want))
        for s, _ in sets:  # new values in the same places
            for k in ("h", "x", "dy", "dn", "grads", "table"):
                s[k].copy_(rand(g, *s[k].shape, scale=turn + 0.5))
            s["ids"].copy_(torch.randint(0, 500, (300,), generator=g, device="cuda"))


@pytest.mark.gpu
def test_shared_buffers_and_other_ranks_sums_captured():
    """A shared parameter's gradient and a rank without parameters, in a graph that is replayed."""
    g, c = norms_case("cuda", 200, 264, BF, BF, "channel", True)
    y, _, rp, rq = fused.block_norms_fwd(c["h"], c["x"], c["w_post"], c["w_pre"], EPS, c["gate"])
    dy, dn = rand(g, 200, 264, dtype=BF), rand(g, 200, 264, dtype=BF)
    acc, sums = torch.zeros(2, 264, device="cuda"), torch.tensor([9.0, 16.0], device="cuda")

    def call():
        for which, accumulate in (((0, 0, 0), False), ((0, 1, 0), True), ((1, 1, 0), True)):
            fused.block_norms_bwd(dy, dn, c["h"], y, rp, rq, c["w_post"], c["w_pre"], acc[which[0]],
                                  acc[which[1]], c["gate"], acc[which[2]], accumulate=accumulate)
        return fused.grad_list_clip_([], 1.0, extra_sumsq=sums)

    call()
    acc.zero_()
    call()
    want = acc.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = call()
    for k in (1.0, 2.0):
        acc.zero_()
        sums.mul_(k * k)
        graph.replay()
        assert torch.equal(acc, want) and float(norm) == 5.0 * k


@pytest.mark.gpu
def test_on_two_streams_at_once():
    g = gen("cuda", 22)
    sets = [_all_operators(g, k) for k in (1.0, 2.0)]
    want = [call(s) for s, call in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for st, (s, call) in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(call(s))
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(p, q))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [200, 257, 3000])
@pytest.mark.parametrize("H", [256, 515])
def test_table_gradient_captured_and_on_two_streams(rows, H):
    """The sorted gradient's launches in graphs that share a pool, and beside each other."""
    g = gen("cuda", 24)
    sets = []
    for k in range(2):
        ids = torch.randint(0, 700, (rows,), generator=g, device="cuda")
        ids[::3] = 11 + k
        sets.append((rand(g, rows, H, dtype=BF), ids, torch.empty(700, H, device="cuda")))

    def call(s):
        fused.scaled_embedding_bwd(*s, 0.5, accumulate=False)
        return fused.scaled_embedding_bwd(*s, 2.0)

    want = [call(s).clone() for s in sets]
    for (dy, ids, _), w in zip(sets, want):
        close(w, *grad_of_table(dy, ids, 700, 2.5), "dtable")
    torch.cuda.synchronize()
    graphs = []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=graphs[0].pool() if len(graphs) > 1 else None):
            call(s)
    for _ in range(3):
        for (_, _, table), graph in zip(sets, graphs):
            table.fill_(float("nan"))
            graph.replay()
        assert all(torch.equal(s[2], w) for s, w in zip(sets, want))
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        torch.cuda.synchronize()
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                call(s)
        torch.cuda.synchronize()
        assert all(torch.equal(s[2], w) for s, w in zip(sets, want))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows that begin behind element 2^31 of their tensors."""
    g = gen("cuda", 23)
    H, T = 4096, 530_000
    h = torch.zeros(T, H, dtype=BF, device="cuda")
    x = torch.zeros(T, H, dtype=BF, device="cuda")
    some = torch.tensor([0, 1, T - 3, T - 1], device="cuda")
    h[some], x[some] = rand(g, 4, H, dtype=BF), rand(g, 4, H, dtype=BF)
    w = torch.ones(H, dtype=BF, device="cuda")
    y, n, rp, rq = fused.block_norms_fwd(h, x, w, w, EPS)
    parts = fused.block_norms_fwd(h[some], x[some], w, w, EPS)
    for p, q in zip((y, n, rp, rq), parts):
        assert torch.equal(p[some], q)
    assert not y[T // 2].any()
    dn = rand(g, 4, H, dtype=BF)
    acc = torch.zeros(4, H, device="cuda")
    one = fused.block_norms_bwd(None, dn, h, y, rp, rq, w, w, acc[0], acc[1], rows=some.int())
    two = fused.block_norms_bwd(None, dn, h[some], y[some], rp[some], rq[some], w, w, acc[2], acc[3])
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    assert torch.equal(acc[:2], acc[2:])
    del y, n, x
    # gradient rows and table rows past 2^31 elements
    ids = torch.zeros(T, dtype=torch.long, device="cuda")
    ids[some] = torch.tensor([5, T - 1, T - 1, 7], device="cuda")
    dt = torch.empty(T, H, device="cuda")
    fused.scaled_embedding_bwd(h, ids, dt, padding_idx=0, accumulate=False)
    assert torch.equal(dt[5], h[0].float()) and torch.equal(dt[7], h[T - 1].float())
    assert torch.equal(dt[T - 1], h[1].float() + h[T - 3].float())
    assert int(dt.any(1).sum()) == 3
    back = fused.scaled_embedding_fwd(dt, torch.tensor([T - 1, 0], device="cuda"))
    assert torch.equal(back[0], dt[T - 1]) and not back[1].any()
    norm = fused.grad_list_clip_([dt], 1.0)
    assert float(norm) == pytest.approx(float(dt[[5, 7, T - 1]].double().norm()) * float(norm), rel=1e-4)
