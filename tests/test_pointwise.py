"""Matrix product with bias, residual and activation against its definition in 64 bits."""
import math

import pytest
import torch

from fast_autoaugment_amd.ops.pointwise import conv1x1_act, linear_act

DEV = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
GPU = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
ACTS = ["none", "relu", "swish", "sigmoid"]


def oracle(x, w, b, r, act, dy):
    """Values in 64 bits from the definition, and what their rounding errors are made of."""
    x, w, dy0 = x.double(), w.double(), dy.double()
    z = x @ w.t()
    size = x.abs() @ w.abs().t()
    for t in (b, r):
        if t is not None:
            z, size = z + t.double(), size + t.double().abs()
    sig = torch.sigmoid(z)
    y, slope, bend = {
        "none": (z, torch.ones_like(z), 0.0), "relu": (z.clamp_min(0), (z > 0).double(), 0.0),
        "swish": (z * sig, sig * (1 + z * (1 - sig)), 0.5), "sigmoid": (sig, sig * (1 - sig), 0.1)}[act]
    # a value at relu's border may fall to either side: it is given no gradient
    dy0 = torch.where((z.abs() < 2.0 ** -12 * size + 1e-3) & torch.tensor(act == "relu"), 0.0, dy0)
    dz = dy0 * slope
    return dict(y=y, z=z, size=size, dy=dy0.to(dy.dtype), dz=dz, bend=bend, dy64=dy0,
                dx=dz @ w, dw=dz.t() @ x, db=dz.sum(0), x=x, w=w)


def close(got, want, tol):
    err = (got.detach().cpu().double() - want).abs()
    assert (err <= tol).all(), f"off by {float((err / tol).max()):.3g} of the tolerance"


def check(dev, x, w, b, r, act, dy, fn=linear_act, grad=True, move=lambda t: t):
    """u is half a step of the type, f half a step of fp32.

    y: the fp32 sum is off by at most (K + 4) f of its terms' sizes, its activation by the steepest slope (1.1) of
    that and 8 f of itself, and it is rounded once. dz: z was rounded to the type (u |z| times the slope's own
    slope, at most 0.5 for swish and 0.1 for sigmoid), and dz itself is rounded once before the products. Products
    of dz carry that share of every term, their own fp32 sum's (N or M + 4) f, and one rounding."""
    t = x.dtype
    o = oracle(x, w, b, r, act, dy)
    u, f, tiny = torch.finfo(t).eps / 2, 2.0 ** -24, torch.finfo(t).tiny
    leaf = lambda v: None if v is None else move(v.to(dev)).detach().requires_grad_(grad)  # noqa: E731
    xd, wd, bd, rd = leaf(x), leaf(w), leaf(b), leaf(r)
    y = fn(xd, wd, bd, residual=rd, act=act)
    assert y.dtype == t and y.shape == (*x.shape[:-1], w.size(0))
    y_off = 1.1 * (x.size(1) + 4) * f * o["size"] + 8 * f * o["y"].abs()
    close(y, o["y"], u * o["y"].abs() + y_off + tiny)
    if not grad:
        return
    leaves = [v for v in (xd, wd, bd, rd) if v is not None]
    got = list(torch.autograd.grad(y, leaves, o["dy"].to(dev)))
    z_off = (u if act in ("swish", "sigmoid") else 0) * o["z"].abs() + (x.size(1) + 4) * f * o["size"]
    slope_off = o["dy64"].abs() * (o["bend"] * z_off + 8 * f)
    dz_off = slope_off + (u * o["dz"].abs() if act != "none" else 0) + tiny
    products = lambda a, k: (k + 4) * f * a  # noqa: E731
    close(got.pop(0), o["dx"], u * o["dx"].abs() + dz_off @ o["w"].abs()
          + products((o["dz"].abs() + dz_off) @ o["w"].abs(), w.size(0)) + tiny)
    close(got.pop(0), o["dw"], u * o["dw"].abs() + dz_off.t() @ o["x"].abs()
          + products((o["dz"].abs() + dz_off).t() @ o["x"].abs(), x.size(0)) + tiny)
    if b is not None:
        close(got.pop(0), o["db"], u * o["db"].abs() + dz_off.sum(0) + products(o["dz"].abs().sum(0), x.size(0)) + tiny)
    if r is not None:
        close(got.pop(0), o["dz"], dz_off)


def inputs(m, k, n, t, bias=True, residual=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(t)  # noqa: E731
    return (r(m, k), (r(n, k) / math.sqrt(k)).to(t), r(n) if bias else None, r(m, n) if residual else None, r(m, n))


SIZES = [
    (1, 1, 1), (1, 8, 8), (3, 5, 7), (128, 64, 64), (129, 72, 65), (64, 1152, 48), (100, 1280, 1000),
    (300, 17, 33), (257, 200, 40), (1000, 64, 256), (33, 2048, 10), (5, 3, 2047), (2500, 24, 144),
    (4100, 40, 24), (40, 520, 520), (20000, 16, 96), (9000, 128, 520),
]


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("t", [BF16, FP16, FP32])
def test_sizes(dev, m, k, n, t):
    x, w, b, r, dy = inputs(m, k, n, t)
    check(dev, x, w, b, r, ACTS[(m + k + n) % 4], dy)


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", [BF16, FP32])
def test_activations_and_missing_terms(dev, act, t):
    for bias in (True, False):
        for residual in (True, False):
            x, w, b, r, dy = inputs(200, 96, 56, t, bias, residual)
            check(dev, x, w, b, r, act, dy)
            check(dev, x, w, b, r, act, dy, grad=False)


@GPU
@pytest.mark.parametrize("m,k,n", [(70000, 64, 256), (40000, 264, 136), (131, 4000, 72)])
def test_large_tiles(m, k, n):
    x, w, b, r, dy = inputs(m, k, n, BF16)
    check("cuda", x, w, b, r, "swish", dy)


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("k,n", [(64, 48), (61, 35)])
def test_a_map_is_a_product_over_pixels(dev, k, n):
    x, w, b, r, dy = inputs(2 * 5 * 6, k, n, BF16)
    as_map = lambda t: t.view(2, 5, 6, -1).permute(0, 3, 1, 2)  # noqa: E731

    def fn(x, w, b, residual, act):
        y = conv1x1_act(as_map(x), w[:, :, None, None], b, as_map(residual), act)
        assert y.shape == (2, n, 5, 6)
        return y.permute(0, 2, 3, 1).reshape(-1, n)
    check(dev, x, w, b, r, "relu", dy, fn=fn)
    nchw = conv1x1_act(as_map(x).contiguous().to(dev), w.to(dev), b.to(dev), as_map(r).contiguous().to(dev), "relu")
    last = conv1x1_act(as_map(x).to(dev), w.to(dev), b.to(dev), as_map(r).to(dev), "relu")
    assert torch.equal(nchw, last)


@pytest.mark.parametrize("dev", DEV)
def test_orders_of_memory(dev):
    x, w, b, r, dy = inputs(60, 48, 40, BF16)
    check(dev, x, w, b, r, "swish", dy, move=lambda t: torch.stack([t, t], -1)[..., 0])
    check(dev, x, w, b, r, "swish", dy, move=lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape))
    lead = linear_act(x.view(3, 4, 5, 48).to(dev), w.to(dev), b.to(dev), r.view(3, 4, 5, 40).to(dev), "swish")
    assert torch.equal(lead.view(60, 40), linear_act(x.to(dev), w.to(dev), b.to(dev), r.to(dev), "swish"))
    vector = linear_act(x[0].to(dev), w.to(dev), b.to(dev), r[0].to(dev), "swish")
    assert vector.shape == (40,)


@pytest.mark.parametrize("dev", DEV)
def test_no_rows(dev):
    x = torch.zeros(0, 8, device=dev, requires_grad=True)
    w = torch.ones(5, 8, device=dev, requires_grad=True)
    b = torch.ones(5, device=dev, requires_grad=True)
    y = linear_act(x, w, b, act="swish")
    assert y.shape == (0, 5)
    y.sum().backward()
    assert x.grad.shape == (0, 8) and not w.grad.any() and not b.grad.any()


@pytest.mark.parametrize("dev", DEV)
def test_what_is_no_number_stays_in_its_row(dev):
    x, w, b, r, _ = inputs(300, 72, 40, BF16)
    for act in ACTS:
        clean = linear_act(x.to(dev), w.to(dev), b.to(dev), r.to(dev), act)
        xx, rr = x.clone(), r.clone()
        xx[7, 3], xx[200, 71], rr[9, 5], rr[299, 39] = math.nan, math.inf, math.nan, -math.inf
        y = linear_act(xx.to(dev), w.to(dev), b.to(dev), rr.to(dev), act).cpu()
        want = torch.zeros(300, 40, dtype=torch.bool)
        want[7], want[200], want[9, 5], want[299, 39] = True, True, True, True
        assert torch.isnan(y[7]).all() and torch.isnan(y[9, 5])
        assert torch.equal(y[~want], clean.cpu()[~want])


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("t", [FP32, BF16])
@pytest.mark.parametrize("n", [40, 33])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_relu_holds_back_gradients_that_are_no_numbers(dev, t, n, bad):
    g = torch.Generator().manual_seed(5)
    x, w, b, r, dy = (torch.randn(*s, generator=g).to(t).to(dev) for s in ((70, 24), (n, 24), (n,), (70, n), (70, n)))
    grads = []
    for fill in (0.0, bad):
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b, r)]
        y = linear_act(*leaves, act="relu")
        assert (y == 0).any()
        grads.append(torch.autograd.grad(y, leaves, torch.where(y.detach() == 0, torch.tensor(fill, dtype=t, device=dev), dy)))
    for a, c in zip(*grads):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dev", DEV)
def test_only_what_is_asked_for(dev):
    x, w, b, r, dy = (t.to(dev) for t in inputs(200, 72, 40, BF16))
    full = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    want = torch.autograd.grad(linear_act(full[0], full[1], full[2], full[3], "swish"), full, dy)
    for i in range(4):
        ts = [t.clone() for t in (x, w, b, r)]
        ts[i].requires_grad_(True)
        got, = torch.autograd.grad(linear_act(ts[0], ts[1], ts[2], ts[3], "swish"), ts[i], dy)
        assert torch.equal(got, want[i])


def test_the_formula_against_differences():
    x, w, b, r, dy = (t.double() for t in inputs(3, 4, 5, FP32))
    for act in ("none", "swish", "sigmoid"):
        want = oracle(x, w, b, r, act, dy)
        value = lambda *v: float((oracle(*v, act, dy)["y"] * dy).sum())  # noqa: E731
        h = 1e-5
        for i, name in ((0, "dx"), (1, "dw"), (2, "db"), (3, "dz")):
            for j in range((x, w, b, r)[i].numel()):
                up, down = ([t.clone() for t in (x, w, b, r)] for _ in range(2))
                up[i].view(-1)[j] += h
                down[i].view(-1)[j] -= h
                assert abs((value(*up) - value(*down)) / (2 * h) - float(want[name].reshape(-1)[j])) < 1e-6


def test_refusals():
    x, w = torch.zeros(3, 8), torch.zeros(5, 8)
    for bad in (dict(act="gelu"), dict(weight=torch.zeros(5, 7)), dict(weight=torch.zeros(8)), dict(bias=torch.zeros(8)),
                dict(residual=torch.zeros(3, 8)), dict(residual=torch.zeros(5)), dict(weight=torch.zeros(0, 8)),
                dict(x=torch.zeros(3, 0), weight=torch.zeros(5, 0))):
        with pytest.raises(ValueError):
            linear_act(**{"x": x, "weight": w, **bad})
    for bad in (dict(x=x.double(), weight=w.double()), dict(weight=w.bfloat16()), dict(bias=torch.zeros(5).half()),
                dict(x=x.long())):
        with pytest.raises(TypeError):
            linear_act(**{"x": x, "weight": w, **bad})
    for bad in (dict(x=x), dict(weight=torch.zeros(5, 8, 3, 3)), dict(residual=torch.zeros(3, 5))):
        with pytest.raises(ValueError):
            conv1x1_act(**{"x": torch.zeros(1, 8, 2, 2), "weight": w, **bad})


@GPU
def test_a_second_derivative_is_refused():
    x, w, b, r, _ = (t.cuda() for t in inputs(20, 8, 8, FP32))
    x.requires_grad_(True)
    g, = torch.autograd.grad(linear_act(x, w, act="swish").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@GPU
@pytest.mark.parametrize("m,k,n", [(128, 1152, 48), (3000, 64, 256)])
def test_captured_and_replayed(m, k, n):
    ts = [t.cuda() for t in inputs(m, k, n, BF16)]
    for t in ts[:4]:
        t.requires_grad_(True)

    def go():
        y = linear_act(ts[0], ts[1], ts[2], ts[3], "swish")
        return [y.detach(), *torch.autograd.grad(y, ts[:4], ts[4])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = go()
    for seed in range(1, 5):
        with torch.no_grad():
            for t, v in zip(ts, inputs(m, k, n, BF16, seed=seed)):
                t.copy_(v)
        eager = go()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(held, eager):
            assert torch.equal(a, c)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """The last rows of results and residuals of more than 2^31 values are what they are by themselves."""
    g = torch.Generator("cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=BF16)  # noqa: E731
    m, k, n = 2 ** 22 + 77, 24, 520
    x, w, b, res = r(m, k), r(n, k), r(n), r(m, n)
    dy = r(m, n)
    assert m * n > 2 ** 31
    outs = []
    for rows in (slice(None), slice(m - 1000, None)):
        leaves = [x[rows].clone().requires_grad_(True), res[rows].clone().requires_grad_(True)]
        y = linear_act(leaves[0], w, b, leaves[1], act="swish")
        outs.append([t[-1000:] for t in (y.detach(), *torch.autograd.grad(y, leaves, dy[rows]))])
        del y, leaves
    # sums of 24 and of 520 terms in the same order of k: a step of bf16 where tiles differ
    for a, c in zip(*outs):
        assert torch.allclose(a.float(), c.float(), rtol=2.0 ** -7, atol=2.0 ** -7)



@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("act", ["swish", "sigmoid"])
@pytest.mark.parametrize("m,k,n", [(40, 16, 24), (300, 8, 33), (3000, 24, 256), (131, 4000, 72)])
def test_sums_beyond_fp16_have_their_slopes(dev, act, m, k, n):
    """A sum of -120000 has no slope, one of 120000 swish's 1 and sigmoid's 0, though neither is a number of fp16. The
    sums are exact and every slope is 0 or 1, so that gradients are those of the rows that have one, once rounded."""
    x = torch.zeros(m, k, dtype=FP16)
    x[:, 0] = torch.tensor([60000.0, -60000.0])[torch.arange(m) % 2]
    w = torch.zeros(n, k, dtype=FP16)
    w[:, 0] = 2.0
    b = torch.zeros(n, dtype=FP16)
    dy = torch.randint(-3, 4, (m, n), generator=torch.Generator().manual_seed(1)).to(FP16)
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w, b, torch.zeros(m, n, dtype=FP16))]
    y = linear_act(leaves[0], leaves[1], leaves[2], leaves[3], act=act)
    dx, dw, db, dr = (t.cpu() for t in torch.autograd.grad(y, leaves, dy.to(dev)))
    dz = dy * (torch.arange(m) % 2 == 0).view(-1, 1) if act == "swish" else torch.zeros_like(dy)
    assert torch.equal(dr, dz)
    assert torch.equal(dx[:, 0], (2 * dz.double().sum(1)).to(FP16)) and not dx[:, 1:].any()
    assert torch.equal(db, dz.double().sum(0).to(FP16))
    assert torch.equal(dw[:, 0], (60000 * dz.double().sum(0)).to(FP16)) and not dw[:, 1:].any()


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("act", ["swish", "sigmoid"])
@pytest.mark.parametrize("t", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,k,n", [(128, 1152, 48), (77, 40, 33), (3000, 24, 256), (131, 4000, 72)])
def test_a_slope_is_that_of_the_sum_in_32_bits(dev, act, t, m, k, n):
    """The residual's gradient is dy times the slope, rounded once: the sum behind the slope is off by its fp32 terms'
    (K + 4) f and the exponential's 2 f |z|, the slope by 8 f of its own, and nothing else is in fewer bits."""
    x, w, b, r, dy = inputs(m, k, n, t, seed=2)
    o = oracle(x, w, b, r, act, dy)
    leaves = [v.to(dev).requires_grad_(True) for v in (x, w, b, r)]
    y = linear_act(leaves[0], leaves[1], leaves[2], leaves[3], act=act)
    got, = torch.autograd.grad(y, leaves[3:], o["dy"].to(dev))
    u, f = torch.finfo(t).eps / 2, 2.0 ** -24
    off = o["dy64"].abs() * (o["bend"] * ((k + 4) * f * o["size"] + 2 * f * o["z"].abs()) + 8 * f)
    # half of a type's smallest step besides, where a result is smaller than its smallest normal number
    close(got, o["dz"], u * (o["dz"].abs() + off) + off + torch.finfo(t).tiny * u)


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("act", ["swish", "sigmoid"])
@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -17])
@pytest.mark.parametrize("m,k,n", [(128, 1152, 48), (100, 48, 1152), (77, 40, 33), (3000, 24, 256), (2500, 264, 136),
                                   (131, 4000, 72), (33, 520, 2047)])
def test_products_have_the_gradient_behind_the_activation_to_more_than_the_type(dev, act, t, scale, m, k, n):
    """dz, made of fp32 slopes (see above), is held as two numbers of the type: half a step u of the first, whose
    own error is u of that again, or half a smallest step where that is more (2^-25 in fp16, and there the second is
    held times 2048: 2^-36). Products carry that, their fp32 sums (2 and 4 more terms of N or M, both passes) and one
    rounding."""
    x, w, b, r, dy = inputs(m, k, n, t, seed=3)
    o = oracle(x, w, b, r, act, (dy.float() * scale).to(t))
    leaves = [v.to(dev).requires_grad_(True) for v in (x, w, b)]
    y = linear_act(leaves[0], leaves[1], leaves[2], r.to(dev), act=act)
    dx, dw, _ = torch.autograd.grad(y, leaves, o["dy"].to(dev))
    u, f = torch.finfo(t).eps / 2, 2.0 ** -24
    off = o["dy64"].abs() * (o["bend"] * ((k + 4) * f * o["size"] + 2 * f * o["z"].abs()) + 8 * f)
    off = off + u * u * o["dz"].abs() + (2.0 ** -36 if t == FP16 else 2.0 ** -133)
    least = torch.finfo(t).tiny * u
    dz, ax, aw = o["dz"].abs(), o["x"].abs(), o["w"].abs()
    tol_x, tol_w = off @ aw + (2 * n + 4) * f * (dz @ aw), off.t() @ ax + (2 * m + 4) * f * (dz.t() @ ax)
    close(dx, o["dx"], u * (o["dx"].abs() + tol_x) + tol_x + least)
    close(dw, o["dw"], u * (o["dw"].abs() + tol_w) + tol_w + least)
    # what a dz rounded once gives would not pass where sums are short: the share of long ones grows with their length
    if n < 64 and t == BF16 and scale == 1.0:
        once = o["dz"].to(t).double() @ o["w"]
        assert (once.to(t).double() - o["dx"]).abs().gt(u * (o["dx"].abs() + tol_x) + tol_x + least).any()


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("act", ["swish", "sigmoid"])
@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("m,k,n", [(60, 16, 24), (300, 72, 33), (3000, 24, 256), (131, 4000, 72)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_gradient_that_is_no_number_stays_in_its_row_and_column(dev, act, t, m, k, n, bad):
    x, w, b, r, dy = inputs(m, k, n, t, seed=4)
    x, w = (torch.where(v == 0, torch.ones_like(v), v) for v in (x, w))       # 0 times infinity is no infinity
    grads = []
    for value in (1.0, bad):
        dy[7, 5] = value
        leaves = [v.to(dev).requires_grad_(True) for v in (x, w, b, r)]
        y = linear_act(*leaves[:3], residual=leaves[3], act=act)
        grads.append([g.cpu() for g in torch.autograd.grad(y, leaves, dy.to(dev))])
    (dx0, dw0, db0, dr0), (dx, dw, db, dr) = grads
    z = x[7].double() @ w[5].double() + b[5].double() + r[7, 5].double()
    sig = torch.sigmoid(z)
    want = torch.tensor(bad) * (sig * (1 + z * (1 - sig)) if act == "swish" else 1)
    for got, value in ((dx[7], want * w[5].double()), (dw[5], want * x[7].double()), (db[5], want), (dr[7, 5], want)):
        assert torch.equal(torch.isnan(got), torch.isnan(value).expand(got.shape)), "NaN"
        if not math.isnan(bad):
            assert torch.equal(got.double(), value)
    rows, cols = torch.arange(m) != 7, torch.arange(n) != 5
    assert torch.equal(dx[rows], dx0[rows]) and torch.equal(dw[cols], dw0[cols]) and torch.equal(db[cols], db0[cols])
    dr[7, 5] = dr0[7, 5]
    assert torch.equal(dr, dr0)


# forward tiles of 128x128, 128x64, 64x64, 32x32; dW's k split in 256, 2, 64, 42 and 17, or not; lines that are widened;
# k of the forward product and of dx split; one chunk of rows, or many, for db
WHOLE = [(70001, 64, 64), (3001, 392, 1000), (70001, 64, 256), (90001, 264, 136), (40003, 264, 136), (50003, 61, 35),
         (20011, 16, 96), (131, 4000, 72), (33, 520, 5003), (131, 1152, 48), (9001, 128, 520), (130, 5, 2047)]


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("t", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,k,n", WHOLE)
def test_sums_of_whole_numbers_are_exact(dev, act, t, m, k, n):
    """Products and sums of small whole numbers are exact in fp32 in any order: results are theirs, rounded once, so
    that a part of a sum that is lost or counted twice shows, however long the sum is."""
    g = torch.Generator().manual_seed(m + k + n)
    whole = lambda most, *s: torch.randint(-most, most + 1, s, generator=g).to(t)  # noqa: E731
    x, w, b, r, dy = whole(2, m, k), whole(2, n, k), whole(3, n), whole(3, m, n), whole(2, m, n)
    z = x.float() @ w.float().t() + b.float() + r.float()        # below 2^24 throughout
    assert 4 * max(m, n, k) + 6 < 2 ** 24
    dz = torch.where(z > 0, dy, torch.zeros_like(dy)) if act == "relu" else dy
    leaves = [v.to(dev).requires_grad_(True) for v in (x, w, b, r)]
    y = linear_act(leaves[0], leaves[1], leaves[2], leaves[3], act=act)
    got = torch.autograd.grad(y, leaves, dy.to(dev))
    want = [dz.float() @ w.float(), dz.float().t() @ x.float(), dz.double().sum(0), dz]
    assert torch.equal(y.detach().cpu(), (z.relu() if act == "relu" else z).to(t))
    for name, a, c in zip(("dx", "dw", "db", "dr"), got, want):
        assert torch.equal(a.cpu(), c.to(t)), name


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("act", ["swish", "sigmoid"])
@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("m,k,n", WHOLE)
def test_both_numbers_of_a_gradient_reach_every_part_of_a_sum(dev, act, t, m, k, n):
    """x (or W) has two rows with 1 and -1 in each column, spread over the whole sum, and zeros: a column of dW (dx) is
    the difference of two rows of dz, which are near each other, so that what bf16 or fp16 leaves of one would show.
    Their slopes (see above) and the two numbers of each are off as before, and four terms are added."""
    g = torch.Generator().manual_seed(m + k + n + 1)
    r = lambda *s: torch.randn(*s, generator=g).to(t)  # noqa: E731
    rows = m if m >= n else n                                   # the longer sum: dW's or dx's
    at = torch.randperm(rows, generator=g)[:2 * k] if rows >= 2 * k else torch.randint(0, rows, (2 * k,), generator=g)
    at[0], at[-1] = 0, rows - 1
    pick = torch.zeros(rows, k, dtype=t)
    first, second = at[:k], at[k:]
    pick[first, torch.arange(k)], pick[second, torch.arange(k)] = 1.0, -1.0
    x, w = (pick, r(n, k)) if rows == m else (r(m, k), pick)
    b, res, dy = r(n), (r(m, 1) * 2.0 ** -6).expand(m, n).contiguous() + r(1, n), r(1, n).expand(m, n).contiguous()
    if rows == n:
        b, res, dy = r(n) * 2.0 ** -6, r(m, 1).expand(m, n).contiguous(), r(m, 1).expand(m, n).contiguous()
    o = oracle(x, w, b, res, act, dy)
    leaves = [v.to(dev).requires_grad_(True) for v in (x, w)]
    y = linear_act(leaves[0], leaves[1], b.to(dev), residual=res.to(dev), act=act)
    dx, dw = torch.autograd.grad(y, leaves, dy.to(dev))
    u, f = torch.finfo(t).eps / 2, 2.0 ** -24
    z_off = (k + 4) * f * o["size"] + 2 * f * o["z"].abs()
    off = o["dy64"].abs() * (o["bend"] * z_off + 8 * f) + u * u * o["dz"].abs() + (2.0 ** -36 if t == FP16 else 2.0 ** -133)
    dz, side = o["dz"].abs(), pick.double().abs()
    if rows == m:
        got, want, tol = dw, o["dw"], off.t() @ side + 8 * f * (dz.t() @ side)
    else:
        got, want, tol = dx, o["dx"], off @ side + 8 * f * (dz @ side)
    close(got, want, u * (want.abs() + tol) + tol + torch.finfo(t).tiny * u)
