"""The embedding-head operators (hessboost_b200/head.py) where their sums cancel, run long or leave a type's range,
against plain 64-bit formulas. u is the unit roundoff of a type (f32 2^-24, bf16 2^-8) and U = 2^-24 that of f32 sums."""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0**-24
F32, BF16 = torch.float32, torch.bfloat16
UNIT = {F32: 2.0**-24, BF16: 2.0**-8}


@pytest.fixture(scope="module")
def head():
    from hessboost_b200 import head as h

    return h


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32, by=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * by).to(dtype)


def xent64(x, w, labels, dloss):
    """loss, |G|, dx and dw in 64 bits; every label is a class."""
    x, w = x.double(), w.double()
    z = x @ w.T
    at = labels.long()[:, None]
    zl = z.gather(1, at)[:, 0]
    # log sum exp(z - z_label): no cancellation where the label's logit is all there is
    rest = (z - zl[:, None]).scatter(1, at, -math.inf)
    loss = torch.logaddexp(torch.zeros_like(zl), torch.logsumexp(rest, 1))
    g = torch.softmax(z, 1)
    g.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    g *= dloss.double()[:, None]
    return dict(z=z, loss=loss, g=g, dx=g @ w, dw=g.T @ x)


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("n,d,v", [(600, 64, 3000), (257, 72, 500), (5000, 128, 700)])
def test_xent_gradient_of_weights_with_a_common_offset(head, n, d, v):
    # a row of G sums to 0, so what all the classes' weights share cancels in dx = G w
    g = gen(n + v)
    x, w = rand(g, n, d, by=0.125), (8 + rand(g, v, d, by=0.25)).to(BF16)
    x = (x - x.mean(1, keepdim=True)).to(BF16)
    labels = torch.randint(v, (n,), generator=g, device="cuda")
    dl = (0.5 + torch.rand(n, generator=g, device="cuda")) / n
    _, lse = head.linear_xent_forward(x, w, labels)
    dx, dw = head.linear_xent_backward(dl, x, w, labels, lse)
    r = xent64(x, w, labels, dl)
    u = UNIT[BF16]
    # the output's rounding (0.6 u of the norm: elements at their worst are u / sqrt 3); two roundings of G's elements (u
    # each of what the first leaves), which do not cancel; and p's error, that of logits added up 16 products at a time
    # (2 U of at most the sum of magnitudes each) and of lse
    z_off = (d / 16 + 2) * 2 * U * float((x.double().abs() @ w.double().abs().T).max())
    assert off(dx, r["dx"]) <= 0.6 * u + (u * u + z_off) * float((r["g"].abs() @ w.double().abs()).norm() / r["dx"].norm())
    assert off(dw, r["dw"]) <= 0.6 * u + (u * u + z_off) * float((r["g"].T.abs() @ x.double().abs()).norm() / r["dw"].norm())


@pytest.mark.parametrize("first", [0.0, 1e-3, 1.0])
def test_xent_one_factor_for_all_rows_but_the_first(head, first):
    # a mean over the rows that count: 1 / 1000 rounded to bf16 once would be 2.2e-3 off in every element of G alike
    g = gen(25)
    x, w = rand(g, 1000, 64, dtype=BF16), rand(g, 500, 64, dtype=BF16, by=0.125)
    labels = torch.randint(500, (1000,), generator=g, device="cuda")
    dl = torch.full((1000,), 1e-3, device="cuda")
    dl[0] = first
    _, lse = head.linear_xent_forward(x, w, labels)
    dx, dw = head.linear_xent_backward(dl, x, w, labels, lse)
    r = xent64(x, w, labels, dl)
    assert off(dx, r["dx"]) <= 0.75 * UNIT[BF16] + 64 * U
    assert off(dw, r["dw"]) <= 0.75 * UNIT[BF16] + 64 * U


@pytest.mark.parametrize("one_sign", [False, True])
@pytest.mark.parametrize("n,d,v", [(4096, 600, 64), (300000, 1024, 40), (600000, 600, 20)])
def test_xent_long_sums_in_f32(head, n, d, v, one_sign):
    # dw sums over the rows, which the tensor cores would round towards zero at every step. A part of 1,024 has 64 steps
    # of 16, each off by 2 U of what is summed so far at most, 64 U of a sum of terms of one sign; the logits, of about 1
    # and in parts of 512, have 32, and so has p its relative error of 64 U at most
    g = gen(n)
    x = torch.rand(n, d, generator=g, device="cuda") + 0.5 if one_sign else rand(g, n, d)
    w = rand(g, v, d, by=d**-0.5)
    labels = torch.zeros(n, dtype=torch.int64, device="cuda") if one_sign else torch.randint(v, (n,), generator=g, device="cuda")
    dl = torch.full((n,), 1.0 / n, device="cuda")
    _, lse = head.linear_xent_forward(x, w, labels)
    dw = head.linear_xent_backward(dl, x, w, labels, lse)[1]
    assert off(dw, xent64(x, w, labels, dl)["dw"]) <= 128 * U


@pytest.mark.parametrize("n,d,v", [(33, 1970, 16918), (300000, 1024, 40), (600000, 600, 20), (9000, 72, 5000)])
def test_xent_f32_gradients_are_as_near_as_f32_sums(head, n, d, v):
    # a part of 512 has 32 steps, each off by half a unit in the last place of what is summed so far: 0.72 U on average
    # over its mantissas. Of terms of either sign, what is summed after i steps is about sqrt(i / 32) of the part:
    # 0.72 U x 21.6 = 15.5 U, always towards zero, so of the whole sum too. 2.5 U for p and the output's rounding
    g = gen(n + 1)
    x, w = rand(g, n, d), rand(g, v, d, by=d**-0.5)
    labels = torch.randint(v, (n,), generator=g, device="cuda")
    dl = (0.5 + torch.rand(n, generator=g, device="cuda")) / n
    _, lse = head.linear_xent_forward(x, w, labels)
    dx, dw = head.linear_xent_backward(dl, x, w, labels, lse)
    r = xent64(x, w, labels, dl)
    assert off(dx, r["dx"]) <= 18 * U
    assert off(dw, r["dw"]) <= 18 * U


@pytest.mark.parametrize("n,d,v", [(130, 2056, 700), (512, 4096, 3000), (300, 16384, 1000), (3000, 4100, 2600)])
def test_xent_logits_of_wide_bf16_rows(head, n, d, v):
    # the loss is f32: logits of about 1 in parts of 2,048, 128 steps of 16 each off by 2 U of what is summed so far (half
    # of the part's sum on average): 128 U of a logit at most, 16 U of a loss of log v
    g = gen(d)
    x, w = rand(g, n, d, dtype=BF16), rand(g, v, d, dtype=BF16, by=d**-0.5)
    labels = torch.randint(v, (n,), generator=g, device="cuda")
    dl = (0.5 + torch.rand(n, generator=g, device="cuda")) / n
    loss, lse = head.linear_xent_forward(x, w, labels)
    r = xent64(x, w, labels, dl)
    assert off(loss, r["loss"]) <= 16 * U
    assert off(lse, torch.logsumexp(r["z"], 1)) <= 16 * U
    dx, dw = head.linear_xent_backward(dl, x, w, labels, lse)
    assert off(dx, r["dx"]) <= 0.75 * UNIT[BF16] + 128 * U and off(dw, r["dw"]) <= 0.75 * UNIT[BF16] + 128 * U


def test_embed_cells_near_32_bits(head):
    # rows of one warp go on together: a short row beside a long one, both within the long one's length of 2^32 cells
    cells = 2**32 - 5000
    if torch.cuda.mem_get_info()[0] < 6 * cells:
        pytest.skip("needs 26 GB")
    tok = torch.full((cells,), -1, dtype=torch.int32, device="cuda")
    tok[:200000] = 1  # of no row
    at = [cells - 110000, cells - 10000, cells - 9990, cells - 9990, cells - 9000, cells]
    tok[at[0]:] = 0
    tok[at[1]:at[2]] = 2
    # so many rows that a warp takes several; the others are empty, before and after
    ptr = torch.tensor([at[0]] * 8 + at + [cells] * 40000, device="cuda")
    out = head.embed_forward(tok, torch.eye(3, device="cuda"), row_ptr=ptr)
    assert out[8:13].tolist() == [[100000, 0, 0], [0, 0, 10], [0, 0, 0], [990, 0, 0], [9000, 0, 0]]
    assert (out[:8] == 0).all() and (out[13:] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d,v", [(64, 12), (64, 3000), (200, 500)])
@pytest.mark.parametrize("near", [0.0, 0.9])
def test_xent_loss_of_certain_rows(head, dtype, d, v, near):
    # logits of 20 to 200, the label's far above the rest, or a little above one other: the loss is what the rest add to
    # 1, and never below 0
    g = gen(v)
    w = rand(g, v, d, dtype=dtype)
    labels = torch.randint(v, (4000,), generator=g, device="cuda")
    by = (20 + 180 * torch.rand(4000, 1, generator=g, device="cuda")) / d
    x = ((w[labels].float() + near * w[labels - 1].float()) * by).to(dtype)
    loss, lse = head.linear_xent_forward(x, w, labels)
    r = xent64(x, w, labels, torch.ones(4000, device="cuda"))
    assert float(loss.min()) >= 0, (int((loss < 0).sum()), float(loss.min()))
    # each of the rest's terms is off by the logits' own error (d products); their sum and log by (v / 32 + 32) U, and
    # their terms' exponents by one rounding
    dz = (d + 4) * U * (x.double().abs() @ w.double().abs().T).max(1).values
    assert ((loss.double() - r["loss"]).abs() <= (r["loss"] + 32 * U) * torch.expm1(2 * dz) + (v / 32 + 32) * U + 2 * U * r["loss"]).all()


def masked_by_the_lowest_value(head, dtype, v, kept):
    # a column of ones makes the weights' last column a bias; the type's lowest value there masks a class, here whole
    # tiles of them: the others' loss and gradients are those of a layer without it
    g = gen(v)
    n, d = 300, 64
    x, w = rand(g, n, d, dtype=dtype), rand(g, v, d, dtype=dtype, by=0.125)
    x[:, -1] = 1
    keep = torch.arange(v, device="cuda") < kept
    w[~keep, -1] = torch.finfo(dtype).min
    labels = torch.randint(kept, (n,), generator=g, device="cuda")
    dl = (0.5 + torch.rand(n, generator=g, device="cuda")) / n
    loss, lse = head.linear_xent_forward(x, w, labels)
    dx, dw = head.linear_xent_backward(dl, x, w, labels, lse)
    r = xent64(x, w[keep], labels, dl)
    tol = 0.75 * UNIT[dtype] + 64 * U
    assert off(loss, r["loss"]) <= 64 * U
    assert off(dx, r["dx"]) <= tol and off(dw[keep], r["dw"]) <= tol
    assert (dw[~keep] == 0).all()


@pytest.mark.parametrize("v,kept", [(20, 7), (2049, 200), (5000, 2700)])
def test_xent_classes_masked_by_the_lowest_value_bf16(head, v, kept):
    masked_by_the_lowest_value(head, BF16, v, kept)


@pytest.mark.parametrize("v,kept", [(20, 7), (2049, 200), (5000, 2700)])
def test_xent_classes_masked_by_the_lowest_value_f32(head, v, kept):
    masked_by_the_lowest_value(head, F32, v, kept)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [1e25, 3e30, 1e-25, 1e-30, 1e-37])
def test_clip_squares_past_the_range_of_f32(head, dtype, size):
    g = gen(6)
    for sizes, common in (([5, 70001], size), ([200003, 3], 1e-3 * size), ([7] * 40, 0.0)):
        t = [rand(g, s, dtype=dtype, by=common) for s in sizes]
        t[0][3] = t[-1][1] = size
        before = [a.clone() for a in t]
        want = math.sqrt(sum(float(a.double().square().sum()) for a in t))
        assert abs(float(head.grad_norm(t)) - want) <= 32 * U * want
        max_norm = 0.5 * want
        norm = head.clip_grad_norm(t, max_norm)
        assert abs(float(norm) - want) <= 32 * U * want
        by = min(1.0, max_norm / (want + 1e-6))
        for a, b in zip(t, before):
            w = b.double() * by
            # the factor's own error, the output's rounding, and the smallest steps of either
            bound = w.abs() * (UNIT[dtype] + 64 * U) + 2.0**-133 + b.double().abs() * 2.0**-148
            assert ((a.double() - w).abs() <= bound).all()


def test_clip_in_place_is_noticed_by_autograd(head):
    # a tensor that a graph has saved changes under it: the graph says so instead of using the new values
    a = torch.ones(50, device="cuda", requires_grad=True)
    t = a * 3.0
    y = (t * t).sum()
    head.clip_grad_norm([t.detach()], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    t = a * 3.0
    y = (t * t).sum()
    head.clip_grad_norm([torch.ones(50, device="cuda")], 1.0, out=[t.detach()])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    # what is only read stays usable
    t = a * 3.0
    y = (t * t).sum()
    head.grad_norm([t.detach()])
    head.clip_grad_norm([t.detach()], 1.0, out=[torch.empty(50, device="cuda")])
    y.backward()
    assert (a.grad == 18).all()
    with torch.inference_mode():
        head.clip_grad_norm([torch.ones(3, device="cuda")], 1.0)
