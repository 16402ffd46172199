"""The embedding-head operators (hessboost_b200/head.py) against plain 64-bit formulas.

Tolerances. u is the unit roundoff of the output's type (f32 2^-24, f16 2^-11, bf16 2^-8) and U = 2^-24 that of the f32
sums. A sum of n terms formed in f32 in any order is off by at most n U sum|term| (first order), and the output's one
rounding by u |value|: `close` checks every element against those, with the terms' sum computed in 64 bits, and the
2-norm of the error against u + (32 + n / 4) U times the norm (roundings of many elements are not all at their worst at
once, but those of one value added again and again are alike).
Where the operator rounds a factor of its products to the inputs' type (the cross entropy's G in bf16), each term carries
another u, and the norm's bound is 2 u.
"""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0**-24
UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def head():
    from hessboost_b200 import head as h

    return h


def close(got, want, terms, n, rounded=0.0, norm=None):
    """got (any type) against want (64 bits): n terms of the sums `terms` of magnitudes, each rounded by `rounded`."""
    u = UNIT[got.dtype]
    got = got.double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    bound = u * (1 + 2 * rounded) * want.abs() + (rounded + (n + 4) * U) * terms + TINY[F32] * (n + 1) + 2 * TINY[
        {v: k for k, v in UNIT.items()}[u]]
    bad = (got - want).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / bound).max()):.3g} of the bound"
    if want.numel() >= 64 and u > TINY[F16] and want.norm() > 0 and (u != UNIT[F16] or want.abs().max() > 1e-3) and (
            want.norm() > 1e-3 * terms.norm()):  # not where the terms cancel
        rel = float((got - want).norm() / want.norm())
        assert rel <= (norm if norm is not None else u + 32 * U) + n / 4 * U, rel


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32, by=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * by).to(dtype)


# ------------------------------------------------------------- embedding
def embed64(tok, table, rows, row_of, scale):
    """(out, sum of magnitudes) in 64 bits."""
    v = table.shape[0]
    there = (tok >= 0) & (tok < v)
    t = table.double()[tok[there].long()] * scale
    z = torch.zeros(rows, table.shape[1], dtype=torch.float64, device="cuda")
    return z.index_add(0, row_of[there], t), z.index_add(0, row_of[there], t.abs())


def embed64_grad(grad, tok, v, row_of, scale):
    there = (tok >= 0) & (tok < v)
    t = grad.double()[row_of[there]] * scale
    z = torch.zeros(v, grad.shape[1], dtype=torch.float64, device="cuda")
    return z.index_add(0, tok[there].long(), t), z.index_add(0, tok[there].long(), t.abs())


def check_embed(head, tok, ptr, table, grad, scale):
    v, d = table.shape
    flat = tok.reshape(-1)
    if ptr is None:
        rows = tok.shape[0]
        per = flat.numel() // rows if rows else 0
        row_of = torch.arange(rows, device="cuda").repeat_interleave(per) if rows else torch.zeros(0, dtype=torch.long, device="cuda")
        most = per
    else:
        rows = ptr.numel() - 1
        count = ptr[1:] - ptr[:-1]
        row_of = torch.repeat_interleave(torch.arange(rows, device="cuda"), count)
        most = int(count.max()) if rows else 0
        flat = flat[int(ptr[0]):int(ptr[-1])]
    out = head.embed_forward(tok, table, row_ptr=ptr, scale=scale)
    assert out.dtype == table.dtype and out.shape == (rows, d) and out.is_contiguous()
    want, mag = embed64(flat, table, rows, row_of, scale)
    close(out, want, mag, most)
    again = head.embed_forward(tok, table, row_ptr=ptr, scale=scale)
    assert torch.equal(out, again)
    dt = head.embed_backward(grad, tok, v, row_ptr=ptr, scale=scale)
    assert dt.dtype == grad.dtype and dt.shape == (v, d)
    want, mag = embed64_grad(grad, flat, v, row_of, scale)
    often = int(torch.bincount(flat[(flat >= 0) & (flat < v)].long(), minlength=1).max()) if flat.numel() else 0
    close(dt, want, mag, often)
    assert torch.equal(dt, head.embed_backward(grad, tok, v, row_ptr=ptr, scale=scale))
    seen = torch.zeros(v, dtype=torch.bool, device="cuda")
    seen[flat[(flat >= 0) & (flat < v)].long()] = True
    assert (dt[~seen] == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,per_row,v,d", [
    (1, 28, 7168, 64), (1, 1, 1, 1), (3, 5, 2, 7), (257, 28, 7168, 64), (1000, 100, 300, 20), (33, 1, 50, 1000),
    (5000, 3, 17, 8), (2049, 28, 70000, 129), (4100, 2, 1, 96), (70, 9, 513, 2051),
])
def test_embed_bags(head, dtype, rows, per_row, v, d):
    g = gen(rows + d)
    tok = torch.randint(-1, v + 1, (rows, per_row), generator=g, device="cuda", dtype=torch.int32)
    check_embed(head, tok, None, rand(g, v, d, dtype=dtype), rand(g, rows, d, dtype=dtype), 0.37)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,mean,v,d,ints", [
    (1, 4, 10, 16, torch.int32), (100, 0, 10, 16, torch.int32), (500, 40, 1280, 128, torch.int64),
    (3001, 7, 128000, 33, torch.int32), (40, 900, 5, 24, torch.int32), (20000, 40, 4096, 16, torch.int32),
])
def test_embed_ragged(head, dtype, rows, mean, v, d, ints):
    g = gen(rows + v)
    count = torch.poisson(torch.full((rows,), float(mean), device="cuda"), generator=g).long()
    count[torch.rand(rows, generator=g, device="cuda") < 0.2] = 0
    count[0] = 0
    count[-1] = 0 if rows > 1 else count[-1]
    ptr = torch.cat([count.new_zeros(1), count.cumsum(0)])
    tok = torch.randint(-2, v + 2, (int(ptr[-1]),), generator=g, device="cuda").to(ints)
    check_embed(head, tok, ptr, rand(g, v, d, dtype=dtype), rand(g, rows, d, dtype=dtype), 1.0)


@pytest.mark.parametrize("n,v,d", [(1, 5, 8), (16384, 300, 72), (9000, 131072, 40), (70001, 3, 16)])
def test_embed_lookup_frequent_ids(head, n, v, d):
    g = gen(n)
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    tok = (torch.exp(u * math.log(v + 1)) - 1).long().clamp_(0, v - 1)
    check_embed(head, tok, None, rand(g, v, d, dtype=BF16), rand(g, n, d, dtype=BF16), 2.0)
    # one id alone, over more cells than any tile of the sort or of the sums
    check_embed(head, torch.full_like(tok, v - 1), None, rand(g, v, d), rand(g, n, d), 1.0)


def test_embed_absent_and_extreme_ids(head):
    g = gen(3)
    table, grad = rand(g, 6, 10), rand(g, 8, 10)
    table[0], grad[7] = float("nan"), float("inf")  # met by no cell
    ids = [-1, 6, 2**31, 2**32, 2**32 + 1, 2**40, -(2**40), -(2**63)]
    tok = torch.tensor([[i, 1 + k % 5] for k, i in enumerate(ids)], device="cuda")
    tok[7] = -1
    out = head.embed_forward(tok, table)
    assert torch.equal(out[:7], table[[1 + k % 5 for k in range(7)]]) and (out[7] == 0).all()
    dt = head.embed_backward(grad, tok, 6)
    assert torch.isfinite(dt).all() and (dt[0] == 0).all()


def test_embed_no_rows_no_cells(head):
    table = torch.ones(4, 3, device="cuda")
    for tok, ptr, rows in ((torch.zeros(0, 5, dtype=torch.int32, device="cuda"), None, 0),
                           (torch.zeros(6, 0, dtype=torch.int32, device="cuda"), None, 6),
                           (torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda"), 3)):
        out = head.embed_forward(tok, table, row_ptr=ptr)
        assert out.shape == (rows, 3) and (out == 0).all()
        dt = head.embed_backward(torch.ones(rows, 3, device="cuda"), tok, 4, row_ptr=ptr)
        assert dt.shape == (4, 3) and (dt == 0).all()


def test_embed_row_ptr_out_of_range_is_clamped(head):
    # offsets past the cells, or falling: cells inside the tensor alone are read
    table, tok = torch.eye(4, device="cuda"), torch.tensor([0, 1, 2, 3], device="cuda")
    ptr = torch.tensor([-5, 2, 1, 900], device="cuda")
    out = head.embed_forward(tok, table, row_ptr=ptr)
    assert out.tolist() == [[1, 1, 0, 0], [0, 0, 0, 0], [0, 1, 1, 1]]
    assert torch.isfinite(head.embed_backward(torch.ones(3, 4, device="cuda"), tok, 4, row_ptr=ptr)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embed_strides_and_offsets(head, dtype):
    g = gen(5)
    wide = rand(g, 200, 70, dtype=dtype)
    tok = torch.randint(200, (90, 6), generator=g, device="cuda", dtype=torch.int32)
    for table in (wide[:, 3:67], wide[:, :64], wide.T.contiguous().T[:, :9], wide[::2, 1:2]):
        grad = rand(g, 90, table.shape[1] + 5, dtype=dtype)[:, 2:2 + table.shape[1]]
        check_embed(head, tok % table.shape[0], None, table, grad, 0.5)
    one = rand(g, 1, 64, dtype=dtype).expand(90, 64)  # a broadcast gradient
    check_embed(head, tok, None, wide[:, :64], one, 0.5)


def test_embed_past_32_bits(head):
    free, _ = torch.cuda.mem_get_info()
    v, d = 2**25 + 3, 128  # 4.3e9 elements
    if free < 5 * v * d:
        pytest.skip("needs 22 GB")
    table = torch.zeros(v, d, dtype=BF16, device="cuda")
    table[-1], table[-2], table[1] = 3, 5, 7
    tok = torch.tensor([[v - 1, v - 2], [1, v], [1, v - 1]], device="cuda")
    assert head.embed_forward(tok, table)[:, -1].tolist() == [8, 7, 10]
    dt = head.embed_backward(torch.tensor([[1.0], [2], [4]], device="cuda").expand(3, d).to(BF16), tok, v)
    assert dt[-1, -1] == 5 and dt[-2, 0] == 1 and dt[1, 5] == 6
    assert int((dt != 0).any(1).sum()) == 3


# ------------------------------------------------------------ layer norm
def norm64(x, w, b, dy, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    xh = (x - mean) * rstd
    w = torch.ones_like(x[0]) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    dy = dy.double()
    g = dy * w
    a, c = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    return dict(mean=mean[:, 0], rstd=rstd[:, 0], xh=xh, y=xh * w + b, dx=rstd * (g - a - xh * c), dw=(dy * xh).sum(0),
                db=dy.sum(0), w=w, b=b, g=g)


def check_norm(head, x, w, b, dy, eps=1e-5):
    n, d = x.shape
    r = norm64(x, w, b, dy, eps)
    y, mean, rstd = head.layer_norm_forward(x, w, b, eps=eps)
    assert y.dtype == x.dtype and mean.dtype == rstd.dtype == F32
    x64 = x.double()
    # mean: a sum of d terms. A centred value is then off by e = that + its own rounding, the variance by 2 |c| e and
    # d U, rstd by half of the variance's share; one more d for slack in the sums of squares
    mag = x64.abs().mean(1)
    close(mean, r["mean"], mag, d)
    e = ((d + 4) * U * mag + 2 * U * x64.abs().max(1).values)
    c = x64 - r["mean"][:, None]
    dvar = (2 * c.abs().mean(1) * e + e * e + (2 * d + 8) * U * c.square().mean(1)) * r["rstd"] ** 2
    drel = 0.5 * dvar + 4 * U
    assert ((rstd.double() - r["rstd"]).abs() <= r["rstd"] * (drel + drel**2) + U * r["rstd"]).all()
    dxh = (e * r["rstd"])[:, None] + r["xh"].abs() * (drel[:, None] + 4 * U)
    close(y, r["y"], r["w"].abs() * dxh / (4 * U) + (r["xh"] * r["w"]).abs() + r["b"].abs(), 0,
          norm=UNIT[y.dtype] + 32 * U + float((r["w"] * dxh).norm() / max(float(r["y"].norm()), 1e-30)))
    for params in (True, False):
        dx, dw, db = head.layer_norm_backward(dy, x, w, mean, rstd, params=params)
        assert dx.dtype == x.dtype
        ga, gx = r["g"].abs(), (r["g"] * r["xh"]).abs()
        da = (d + 4) * U * ga.mean(1, keepdim=True)
        dc = (d + 8) * U * gx.mean(1, keepdim=True) + (ga * dxh).mean(1, keepdim=True)
        c1 = (r["g"] * r["xh"]).mean(1, keepdim=True).abs()
        slack = r["rstd"][:, None] * (da + dc * r["xh"].abs() + c1 * dxh + drel[:, None] * (
            ga + ga.mean(1, keepdim=True) + c1 * r["xh"].abs()))
        mags = r["rstd"][:, None] * (ga + ga.mean(1, keepdim=True) + c1 * r["xh"].abs())
        close(dx, r["dx"], slack / (4 * U) + 2 * mags, 0,
              norm=UNIT[dx.dtype] + 32 * U + float(slack.norm() / max(float(r["dx"].norm()), 1e-30)))
        if not params:
            assert dw is None and db is None
            continue
        assert dw.dtype == db.dtype == (x.dtype if w is None else w.dtype)
        off = (dy.double().abs() * dxh).sum(0)
        close(dw, r["dw"], (dy.double() * r["xh"]).abs().sum(0) + off / ((n + 8) * U), n + 4,
              norm=UNIT[dw.dtype] + 32 * U + float(off.norm() / max(float(r["dw"].norm()), 1e-30)))
        close(db, r["db"], dy.double().abs().sum(0), n)
        d2 = head.layer_norm_backward(dy, x, w, mean, rstd)
        assert torch.equal(dx, d2[0]) and torch.equal(dw, d2[1]) and torch.equal(db, d2[2])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,d", [(1, 64), (1, 1), (5, 3), (130, 64), (1027, 128), (300, 257), (64, 1000), (33, 4097),
                                 (7, 8192), (2, 20011), (3000, 8), (5001, 33)])
def test_norm(head, dtype, n, d):
    g = gen(n * d)
    x = rand(g, n, d, dtype=dtype, by=2.0) + rand(g, n, 1, dtype=dtype)
    check_norm(head, x, 1 + rand(g, d, dtype=dtype, by=0.2), rand(g, d, dtype=dtype, by=0.1), rand(g, n, d, dtype=dtype))


@pytest.mark.parametrize("d", [16, 96, 1500])
def test_norm_parameter_types_and_none(head, d):
    g = gen(d)
    x, dy = rand(g, 70, d, dtype=BF16), rand(g, 70, d, dtype=BF16)
    w, b = 1 + rand(g, d, by=0.2), rand(g, d)
    check_norm(head, x, w, b, dy)
    check_norm(head, x, w, None, dy)
    check_norm(head, x, None, w, dy)
    check_norm(head, x, None, None, dy)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_strides_offsets_shapes(head, dtype):
    g = gen(11)
    wide, grad = rand(g, 65, 300, dtype=dtype), rand(g, 65, 300, dtype=dtype)
    w, b = rand(g, 301, dtype=dtype)[1:], rand(g, 300, dtype=dtype)
    check_norm(head, wide[:, 1:257], w[:256], b[:256], grad[:, 3:259])
    check_norm(head, wide[:, :256], w[:256], b[44:], grad[:, :256])
    check_norm(head, wide[::3], w[:300], b, grad[::3])
    check_norm(head, wide.T.contiguous().T, w[:300], b, grad)
    check_norm(head, wide[:1].expand(65, 300), w[:300], b, grad[:1].expand(65, 300))
    y, mean, rstd = head.layer_norm_forward(wide.reshape(5, 13, 300), b, b)
    y2 = head.layer_norm_forward(wide, b, b)[0]
    assert y.shape == (5, 13, 300) and torch.equal(y.reshape(65, 300), y2) and mean.shape == (65,)


def test_norm_constant_rows_offsets_and_no_rows(head):
    g = gen(12)
    # constant rows: variance 0, rstd 1 / sqrt(eps), y = bias
    x = torch.full((4, 100), 3.0, device="cuda")
    w, b = rand(g, 100), rand(g, 100)
    y, mean, rstd = head.layer_norm_forward(x, w, b, eps=1e-4)
    assert torch.equal(y, b.expand(4, 100)) and (mean == 3).all()
    assert torch.allclose(rstd, torch.full((4,), 100.0, device="cuda"), rtol=4 * U, atol=0)
    # rows far from 0 beside their spread
    check_norm(head, 1000 + rand(g, 50, 640), w.repeat(7)[:640], b.repeat(7)[:640], rand(g, 50, 640))
    # no rows: dweight and dbias are sums of nothing
    x = torch.empty(0, 100, device="cuda")
    y, mean, rstd = head.layer_norm_forward(x, w, b)
    dx, dw, db = head.layer_norm_backward(x, x, w, mean, rstd)
    assert y.shape == dx.shape == (0, 100) and (dw == 0).all() and (db == 0).all()
    # a row with an infinity or a NaN is NaN, and the others are not touched
    x = rand(g, 6, 200)
    x[2, 5], x[4, 7] = float("inf"), float("nan")
    y = head.layer_norm_forward(x)[0]
    assert torch.isnan(y[[2, 4]]).all() and torch.isfinite(y[[0, 1, 3, 5]]).all()


def test_norm_gradient_against_differences(head):
    g = gen(13)
    x, w, b, dy, by = rand(g, 9, 50), 1 + rand(g, 50, by=0.2), rand(g, 50), rand(g, 9, 50), rand(g, 9, 50)
    _, mean, rstd = head.layer_norm_forward(x, w, b)
    dx, dw, db = head.layer_norm_backward(dy, x, w, mean, rstd)
    f = lambda x, w, b: float((head.layer_norm_forward(x, w, b)[0].double() * dy.double()).sum())  # noqa: E731
    h = 2.0**-7
    # central differences: the third derivative's share is h^2 times terms of order 1 to 10 per element, the
    # rounding's 450 elements * U * 4 / h
    tol = 20 * h * h * math.sqrt(450) + 450 * U * 4 / h
    assert abs((f(x + h * by, w, b) - f(x - h * by, w, b)) / (2 * h) - float((dx.double() * by.double()).sum())) <= tol
    assert abs((f(x, w + h * by[0], b) - f(x, w - h * by[0], b)) / (2 * h) - float((dw * by[0]).sum())) <= tol
    assert abs((f(x, w, b + h * by[0]) - f(x, w, b - h * by[0])) / (2 * h) - float((db * by[0]).sum())) <= tol


# --------------------------------------- softmax cross entropy of a layer
def xent64(x, w, labels, dloss):
    x, w = x.double(), w.double()
    z = x @ w.T
    lse = torch.logsumexp(z, 1)
    there = (labels >= 0) & (labels < w.shape[0])
    at = labels.clamp(0, w.shape[0] - 1).long()
    loss = torch.where(there, lse - z.gather(1, at[:, None])[:, 0], 0.0)
    p = torch.exp(z - lse[:, None])
    g = p.clone()
    g.scatter_add_(1, at[:, None], -torch.ones_like(at, dtype=torch.float64)[:, None])
    g *= torch.where(there, dloss.double(), 0.0)[:, None]
    return dict(z=z, lse=lse, loss=loss, g=g, p=p, dx=g @ w, dw=g.T @ x, there=there)


def check_xent(head, x, w, labels, dloss):
    n, d = x.shape
    v = w.shape[0]
    r = xent64(x, w, labels, dloss)
    loss, lse = head.linear_xent_forward(x, w, labels)
    assert loss.dtype == lse.dtype == F32 and loss.shape == (n,)
    # a logit is a sum of d products; lse moves by no more than the worst logit, and its own log and sum of v terms
    # by (v / 32 + 32) U (each of at least 32 partial sums is formed apart)
    dz = (d + 4) * U * (x.double().abs() @ w.double().abs().T)
    worst = dz.max(1).values if n else dz.new_zeros(0)
    dl = worst + (v / 32 + 32) * U + 4 * U * (r["lse"].abs() + r["z"].abs().max(1).values if n else 0)
    assert ((lse.double() - r["lse"]).abs() <= dl).all()
    assert ((loss.double() - r["loss"]).abs() <= torch.where(r["there"], 2 * dl + 4 * U * r["z"].abs().max(1).values, 0.0)).all()
    dx, dw = head.linear_xent_backward(dloss, x, w, labels, lse)
    assert dx.dtype == dw.dtype == x.dtype and dx.shape == x.shape and dw.shape == w.shape
    # G's elements: exp(z - lse) relative to dz + dl, and G's rounding to the inputs' type where that is bf16
    each = torch.where(r["there"], dloss.double(), 0.0).abs()[:, None]
    dg = each * (r["p"] * (dz + dl[:, None] + 8 * U) + 2 * U)
    u = UNIT[x.dtype] if x.dtype == BF16 else 4 * U
    extra = dg @ w.double().abs()
    close(dx, r["dx"], r["g"].abs() @ w.double().abs() + extra / u, v if x.dtype == F32 else v, rounded=u,
          norm=None if n * d < 64 else 2 * UNIT[x.dtype] + 64 * U + float(extra.norm() / max(float(r["dx"].norm()), 1e-30)))
    extra = dg.T @ x.double().abs()
    close(dw, r["dw"], r["g"].T.abs() @ x.double().abs() + extra / u, n, rounded=u,
          norm=None if v * d < 64 else 2 * UNIT[x.dtype] + 64 * U + float(extra.norm() / max(float(r["dw"].norm()), 1e-30)))
    assert (dx[~r["there"]] == 0).all()
    l2, e2 = head.linear_xent_forward(x, w, labels)
    assert torch.equal(loss, l2) and torch.equal(lse, e2)
    d2 = head.linear_xent_backward(dloss, x, w, labels, lse)
    assert torch.equal(dx, d2[0]) and torch.equal(dw, d2[1])


def xent_inputs(g, n, d, v, dtype, spread=1.0):
    x, w = rand(g, n, d, dtype=dtype), rand(g, v, d, dtype=dtype, by=spread * d**-0.5)
    labels = torch.randint(-1, v + 1, (n,), generator=g, device="cuda")
    return x, w, labels, (0.5 + torch.rand(n, generator=g, device="cuda")) / max(n, 1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,d,v", [
    (1, 64, 1000), (1, 1, 2), (2, 3, 1), (16, 128, 1000), (100, 100, 10), (513, 100, 10), (65, 33, 65), (128, 64, 256),
    (129, 72, 257), (300, 257, 2049), (1000, 40, 3), (17, 1030, 700), (2000, 16, 127), (1, 256, 20011), (260, 520, 4000),
    (3000, 8, 64), (700, 200, 33),
])
def test_xent(head, dtype, n, d, v):
    check_xent(head, *xent_inputs(gen(n + d + v), n, d, v, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,d,v", [(2500, 136, 2600), (4999, 520, 1300), (3000, 257, 9000), (60000, 24, 1000), (20000, 160, 6000),
                                   (9000, 72, 5000)])
def test_xent_pieces_and_chunks(head, dtype, n, d, v):
    # several pieces of the classes, chunks of the rows, both; tiles of one CTA and of two
    check_xent(head, *xent_inputs(gen(n + d + v), n, d, v, dtype))


@pytest.mark.parametrize("n,d,v", [(1, 1233, 4), (40, 2048, 30), (300, 1030, 700), (3000, 600, 2600), (130, 4100, 200)])
def test_xent_wide_f32(head, n, d, v):
    # long sums in f32: no further off than 32 U of the gradients' norms, wherever they are formed
    x, w, labels, dl = xent_inputs(gen(n + d), n, d, v, F32)
    labels = labels.clamp(0, v - 1)
    check_xent(head, x, w, labels, dl)
    loss, lse = head.linear_xent_forward(x, w, labels)
    dx, dw = head.linear_xent_backward(dl, x, w, labels, lse)
    r = xent64(x, w, labels, dl)
    assert float((loss.double() - r["loss"]).norm() / r["loss"].norm()) <= 16 * U
    assert float((dx.double() - r["dx"]).norm() / r["dx"].norm()) <= 64 * U
    assert float((dw.double() - r["dw"]).norm() / r["dw"].norm()) <= 64 * U


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_xent_one_factor_for_all_rows(head, dtype):
    # a mean's factor, whose rounding to the inputs' type would be the same for every row: 1 / 1000 is 2.2e-3 off in bf16
    x, w, labels, _ = xent_inputs(gen(25), 1000, 64, 500, dtype)
    labels[0] = 3
    dl = torch.full((1000,), 1e-3, device="cuda")
    _, lse = head.linear_xent_forward(x, w, labels)
    dx, dw = head.linear_xent_backward(dl, x, w, labels, lse)
    r = xent64(x, w, labels, dl)
    # one rounding of the output, and one of random size of each element of G
    assert float((dx.double() - r["dx"]).norm() / r["dx"].norm()) <= 0.75 * UNIT[dtype] + 64 * U
    assert float((dw.double() - r["dw"]).norm() / r["dw"].norm()) <= 0.75 * UNIT[dtype] + 64 * U


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,d,v", [(40, 64, 12), (200, 96, 3000)])
def test_xent_large_logits(head, dtype, n, d, v):
    # logits of hundreds: peaked rows, where exp of the plain logit overflows
    check_xent(head, *xent_inputs(gen(v), n, d, v, dtype, spread=100.0))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [7, 900])
def test_xent_strides_offsets_types(head, dtype, v):
    g = gen(21)
    x, w, labels, dl = xent_inputs(g, 90, 75, v, dtype)
    check_xent(head, x[:, 3:67], w[:, 1:65], labels.int(), dl)
    check_xent(head, x[:, :64], w[:, 8:72], labels, dl[:1].expand(90))
    check_xent(head, x[::2], w, labels[::2], dl[::2])
    check_xent(head, x.T.contiguous().T, w.T.contiguous().T, labels, dl)
    check_xent(head, x[:1].expand(90, 75), w[:1].expand(v, 75), labels, dl)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [5, 600])
def test_xent_rows_without_labels(head, dtype, v):
    g = gen(22)
    x, w, labels, dl = xent_inputs(g, 70, 40, v, dtype)
    check_xent(head, x, w, torch.full_like(labels, -1), dl)
    labels[:] = torch.tensor([-1, v, 2**40, -(2**62), 0, v - 1, 1] * 10, device="cuda")
    # a factor of an unlabelled row plays no part, whatever it is
    dl = dl.clone()
    dl[0], dl[1] = float("nan"), float("inf")
    loss, lse = head.linear_xent_forward(x, w, labels)
    dx, dw = head.linear_xent_backward(dl, x, w, labels, lse)
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all() and (dx[:4] == 0).all() and (loss[:4] == 0).all()
    dl[0] = dl[1] = 1.0
    check_xent(head, x, w, labels, dl)


def test_xent_no_rows(head):
    w = torch.ones(30, 8, device="cuda")
    x, labels = torch.empty(0, 8, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")
    loss, lse = head.linear_xent_forward(x, w, labels)
    dx, dw = head.linear_xent_backward(loss, x, w, labels, lse)
    assert loss.shape == (0,) and dx.shape == (0, 8) and (dw == 0).all()


def test_xent_nonfinite_rows_stay_apart(head):
    g = gen(23)
    for v in (6, 700):
        x, w, labels, dl = xent_inputs(g, 20, 32, v, F32)
        labels = labels.clamp(0, v - 1)
        x[3, 4] = float("nan")
        loss, lse = head.linear_xent_forward(x, w, labels)
        assert torch.isnan(loss[3]) and torch.isfinite(loss[torch.arange(20, device="cuda") != 3]).all()


@pytest.mark.parametrize("n,d,v", [(30, 24, 9), (50, 64, 800)])
def test_xent_gradient_against_differences(head, n, d, v):
    g = gen(24)
    x, w, labels, _ = xent_inputs(g, n, d, v, F32)
    dl = 0.5 + torch.rand(n, generator=g, device="cuda")
    _, lse = head.linear_xent_forward(x, w, labels)
    dx, dw = head.linear_xent_backward(dl, x, w, labels, lse)
    f = lambda x, w: float((head.linear_xent_forward(x, w, labels)[0].double() * dl.double()).sum())  # noqa: E731
    for step, grad, at in ((rand(g, n, d), dx, 0), (rand(g, v, d), dw, 1)):
        h = 2.0**-6 / float(step.norm())
        move = [(x + s * h * step, w) if at == 0 else (x, w + s * h * step) for s in (1, -1)]
        got = (f(*move[0]) - f(*move[1])) / (2 * h)
        # third derivative of a row's loss along a direction of norm |q| is at most |q|^3 (|w| or |x|)^3 / 6; the
        # losses, n values near log v, are each off by (d + v / 32 + 40) U times their magnitudes
        other = w if at == 0 else x
        tol = n * 2 * (h * float(other.norm(dim=1).max()) * float(step.norm())) ** 2 * float(other.norm(dim=1).max()) * float(
            step.norm()) / 6 + n * 1.5 * (d + v / 32 + 40) * U * (2 + math.log(v)) / h
        want = float((grad.double() * step.double()).sum())
        assert abs(got - want) <= tol, (got, want, tol)


# -------------------------------------------------------------- clipping
def check_clip(head, tensors, max_norm, outs=None):
    want = math.sqrt(sum(float(t.double().square().sum()) for t in tensors))
    n = sum(t.numel() for t in tensors)
    before = [t.clone() for t in tensors]
    norm = head.grad_norm(tensors)
    # squares and sums of f32, at most 2^16 to one f32 sum; sqrt halves the share
    tol = (2**16 + 8) * U * want
    assert norm.dtype == F32 and norm.dim() == 0 and abs(float(norm) - want) <= tol
    if n >= 64:
        assert abs(float(norm) - want) <= 32 * U * want
    got = head.clip_grad_norm(tensors, max_norm, out=outs)
    assert torch.equal(got, norm)
    q = max_norm / (float(norm) + 1e-6)
    for t, o, b in zip(tensors, outs if outs is not None else tensors, before):
        if outs is not None:
            assert torch.equal(t, b)
        if o.numel():
            w = b.double().reshape(-1) * min(1.0, q)
            close(o.reshape(-1), w, w.abs(), 4)
        if q > 1.001:
            assert torch.equal(o.reshape(-1), b.reshape(-1))


@pytest.mark.parametrize("sizes", [[1], [5, 0, 64], [65536], [65537, 3, 70001], [1000] * 20, [0, 0, 7], [7] * 1300,
                                   [3_000_001, 17, 250_000]])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_clip_sizes(head, sizes, dtype):
    g = gen(len(sizes))
    tensors = [rand(g, s, dtype=dtype, by=10.0 ** -(i % 4)) for i, s in enumerate(sizes)]
    check_clip(head, tensors, 1.0, [torch.empty_like(t) for t in tensors])
    check_clip(head, [t.clone() for t in tensors], 1e9)
    check_clip(head, [t.clone() for t in tensors], 0.25)


def test_clip_mixed_types_offsets(head):
    g = gen(31)
    base = [rand(g, 5000, dtype=t) for t in (F32, F16, BF16)]
    tensors = [b[o:o + s] for b, (o, s) in zip(base * 2, [(1, 4097), (3, 4000), (5, 100), (4500, 400), (4100, 7), (1000, 3000)])]
    flat = [torch.zeros(5001, dtype=t.dtype, device="cuda") for t in tensors]
    check_clip(head, tensors, 2.0, [f[1:1 + t.numel()] for f, t in zip(flat, tensors)])
    assert all(f[0] == 0 and (f[1 + t.numel():] == 0).all() for f, t in zip(flat, tensors))
    check_clip(head, [rand(g, 30, 40), rand(g, 3, 4, 5)], 0.5)


def test_clip_zero_and_nonfinite(head):
    z = [torch.zeros(100, device="cuda"), torch.zeros(3, device="cuda")]
    assert float(head.clip_grad_norm(z, 1.0)) == 0 and (z[0] == 0).all()
    a = [torch.ones(70000, device="cuda"), torch.ones(4, device="cuda")]
    a[0][69999] = float("inf")
    assert float(head.clip_grad_norm(a, 1.0)) == math.inf
    assert (a[1] == 0).all() and torch.isnan(a[0][69999])
    a = [torch.ones(100, device="cuda"), torch.full((4,), float("nan"), device="cuda")]
    assert math.isnan(float(head.clip_grad_norm(a, 1.0))) and torch.isnan(a[0]).all()
    b = [torch.ones(4, device="cuda")]
    head.clip_grad_norm(b, 0.0)
    assert (b[0] == 0).all()


# ---------------------------------------------------------------- streams
def test_other_streams(head):
    g = gen(41)
    x, w, labels, dl = xent_inputs(g, 600, 64, 900, BF16)
    tok = torch.randint(900, (600, 7), generator=g, device="cuda")
    want = None
    for s in (torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()):
        s.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(s):
            a = torch.empty(1 << 26, device="cuda").fill_(1.0)  # work ahead of the calls on this stream
            xs = x * a[:1].to(BF16)
            y, mean, rstd = head.layer_norm_forward(xs)
            dx, dw, db = head.layer_norm_backward(xs, xs, None, mean, rstd)
            loss, lse = head.linear_xent_forward(y, w, labels)
            gx, gw = head.linear_xent_backward(dl, y, w, labels, lse)
            e, de = head.embed_forward(tok, w), head.embed_backward(gx, tok, 900)
            t = [gw, de]
            norm = head.clip_grad_norm(t, 1.0)
            got = [y, dx, dw, db, loss, gx, gw, e, de, norm]
        s.synchronize()
        want = want or got
        assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_autograd(head):
    g = gen(42)
    tok = torch.randint(-1, 50, (40, 6), generator=g, device="cuda")
    labels = torch.randint(30, (40,), generator=g, device="cuda")
    p = [rand(g, 50, 32), 1 + rand(g, 32, by=0.1), rand(g, 32, by=0.1), rand(g, 30, 32)]

    def step(p, emb, norm, xent):
        p = [t.clone().requires_grad_() for t in p]
        loss = xent(norm(emb(tok, p[0]), p[1], p[2]), p[3], labels).mean()
        loss.backward()
        return [loss.detach()] + [t.grad for t in p]

    fn = torch.nn.functional
    there = (tok >= 0)[..., None]
    want = step([t.double() for t in p], lambda k, t: (t[k.clamp(0)] * there).sum(1) * 0.5,
                lambda x, w, b: fn.layer_norm(x, (32,), w, b), lambda x, w, l: fn.cross_entropy(x @ w.T, l, reduction="none"))
    got = step(p, lambda k, t: head.embed(k, t, scale=0.5), head.layer_norm, head.linear_xent)
    for a, b in zip(got, want):
        assert float((a.double() - b).norm() / b.norm()) <= 64 * U
