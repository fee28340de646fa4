"""Group norm with an activation against its definition in 64 bits."""
import math

import pytest
import torch

from fast_autoaugment_amd.ops.groupnorm import group_norm_act

DEV = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
GPU = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def oracle(x, groups, w, b, eps, act, dy):
    """y, dx, dw, db and what their rounding errors are made of, in 64 bits from the definition."""
    n, c = x.shape[:2]
    x64, dy64 = x.double(), dy.double()
    shape = (1, c) + (1,) * (x.dim() - 2)
    w64 = torch.ones(c, dtype=torch.float64) if w is None else w.double()
    b64 = torch.zeros(c, dtype=torch.float64) if b is None else b.double()
    w64, b64 = w64.view(shape), b64.view(shape)
    grouped = lambda t: t.reshape(n, groups, -1)  # noqa: E731
    back = lambda t: t.expand(n, groups, grouped(x64).size(2)).reshape(x.shape)  # noqa: E731
    mean = grouped(x64).mean(2, keepdim=True)
    d = grouped(x64) - mean
    rstd = (d.square().mean(2, keepdim=True) + eps).rsqrt()
    xhat = back(d * rstd)
    z = xhat * w64 + b64
    sig = torch.sigmoid(z)
    y, slope = {"none": (z, torch.ones_like(z)), "relu": (z.clamp_min(0), (z > 0).double()),
                "swish": (z * sig, sig * (1 + z * (1 - sig)))}[act]
    # a value at relu's border may fall to either side: it is given no gradient
    dy64 = torch.where((z.abs() < 1e-3) & torch.tensor(act == "relu"), 0.0, dy64)
    dz = dy64 * slope
    u = dz * w64
    m1, m2 = grouped(u).mean(2, keepdim=True), grouped(u * xhat).mean(2, keepdim=True)
    rs = back(rstd)
    dx = rs * (u - back(m1) - xhat * back(m2))
    red = [0] + list(range(2, x.dim()))
    s = dict(y=y, dx=dx, dw=(dz * xhat).sum(red), db=dz.sum(red), dy=dy64.to(dy.dtype))
    # sizes of the terms that are rounded, with the mean's own error in each xhat
    off = back(grouped(x64.abs()).mean(2, keepdim=True)) * rs
    s["y_size"] = (xhat.abs() + off) * w64.abs() + b64.abs()
    dz_err = dy64.abs() * 1.2 * s["y_size"] + dz.abs()
    s["dx_size"] = rs * (dz_err * w64.abs() + back(grouped(dz_err * w64.abs()).mean(2, keepdim=True))
                         + (xhat.abs() + off) * back(grouped(dz_err * w64.abs() * (1 + xhat.abs() + off)).mean(2, keepdim=True)))
    s["dw_size"] = (dz_err * (1 + xhat.abs() + off)).sum(red)
    s["db_size"] = dz_err.sum(red)
    return s


def close(got, want, size, depth=256):
    """Half a step of the type, and the fp32 sums below it: none is longer than `depth` additions in a row."""
    t = got.dtype
    tol = torch.finfo(t).eps / 2 * want.abs() + depth * 2.0 ** -24 * size + torch.finfo(t).tiny
    err = (got.detach().cpu().double() - want).abs()
    assert (err <= tol).all(), f"off by {float((err / tol).max()):.3g} of the tolerance"


def inputs(shape, t, seed=0, mean=0.5, wt=None, weight=True, bias=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    c = shape[1]
    x = (r(*shape) + mean + r(1, c, *([1] * (len(shape) - 2)))).to(t)
    w = (1 + 0.3 * r(c)).to(wt or t) if weight else None
    b = (0.3 * r(c)).to(wt or t) if bias else None
    return x, w, b, r(*shape).to(t)


def check(dev, x, groups, w, b, act, dy, eps=1e-5, layout=lambda t: t):
    want = oracle(x, groups, w, b, eps, act, dy)
    leaf = lambda t: None if t is None else t.to(dev).requires_grad_(True)  # noqa: E731
    xd, wd, bd = layout(x.to(dev)).detach().requires_grad_(True), leaf(w), leaf(b)
    y = group_norm_act(xd, groups, wd, bd, eps=eps, act=act)
    assert y.shape == x.shape and y.dtype == x.dtype
    leaves = [t for t in (xd, wd, bd) if t is not None]
    grads = list(torch.autograd.grad(y, leaves, layout(want["dy"].to(dev))))
    close(y, want["y"], want["y_size"])
    close(grads.pop(0), want["dx"], want["dx_size"])
    if w is not None:
        close(grads.pop(0), want["dw"], want["dw_size"])
    if b is not None:
        close(grads.pop(0), want["db"], want["db_size"])


SHAPES = [
    ((2, 8, 4, 4), 2), ((3, 6), 3), ((2, 12, 5), 4), ((1, 61, 16, 16), 1), ((2, 24, 7, 9), 8),
    ((2, 112, 14, 14), 8), ((1, 1280, 7, 7), 32), ((2, 35, 3, 3), 5), ((2, 64, 33, 31), 8),
    ((1, 16, 130, 130), 4), ((2, 8, 2, 3, 4), 2), ((4, 2048, 2, 2), 1), ((2, 2047, 2, 1), 1),
    ((5, 32, 32, 32), 32), ((1, 16, 1, 1), 1), ((3, 40, 56, 56), 5), ((2, 256, 56, 56), 32),
    ((300, 16, 2, 2), 2), ((2, 672, 14, 14), 8), ((1, 96, 112, 112), 8), ((2, 4096, 1, 1), 2),
    ((1, 20, 64, 64), 1), ((9, 192, 8, 8), 3), ((5000, 24), 3), ((2, 28, 13, 11), 7), ((2, 36, 90, 90), 2),
    ((128, 16, 56, 56), 8), ((3, 1000, 5, 5), 8), ((2, 1024, 16, 16), 1),
]


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("shape,groups", SHAPES)
@pytest.mark.parametrize("t", [FP32, BF16, FP16])
def test_shapes(dev, shape, groups, t):
    x, w, b, dy = inputs(shape, t)
    act = ["none", "swish", "relu"][(len(shape) + shape[1] + groups) % 3]
    last = (lambda v: v.contiguous(memory_format=torch.channels_last)) if len(shape) == 4 else (lambda v: v)
    check(dev, x, groups, w, b, act, dy, layout=last)


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("act", ["none", "relu", "swish"])
@pytest.mark.parametrize("t", [FP32, BF16])
def test_activations_and_missing_parameters(dev, act, t):
    for weight in (True, False):
        for bias in (True, False):
            x, w, b, dy = inputs((2, 24, 9, 9), t, weight=weight, bias=bias)
            check(dev, x, 4, w, b, act, dy)


@pytest.mark.parametrize("dev", DEV)
def test_fp32_parameters_with_low_precision_maps(dev):
    x, w, b, dy = inputs((2, 32, 9, 9), BF16, wt=FP32)
    check(dev, x, 4, w, b, "swish", dy)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((1100, 8192), 1024), ((1100, 8192, 1, 1), 8192), ((1030, 6144, 1, 2), 768),
                                          ((1030, 2600, 1, 1), 650)])
def test_many_channels_and_few_pixels(shape, groups):
    """Whole samples fit a workgroup's registers here, but the constants of their channels are more than LDS."""
    x, w, b, dy = inputs(shape, BF16)
    check("cuda", x, groups, w, b, "relu", dy)


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("shape,groups", [((2, 16, 40, 40), 2), ((2, 16, 150, 150), 2), ((2, 15, 20, 20), 3)])
def test_a_mean_far_from_zero(dev, shape, groups):
    """The variance is that of the differences: a mean of a thousand spreads costs its own digits alone."""
    x, w, b, dy = inputs(shape, FP32, mean=1000.0)
    check(dev, x, groups, w, b, "none", dy)


@pytest.mark.parametrize("dev", DEV)
def test_a_constant_group(dev):
    x = torch.full((2, 8, 5, 5), 3.0)
    y = group_norm_act(x.to(dev), 2, None, torch.arange(8.0, device=dev), act="none")
    assert torch.equal(y.cpu(), torch.arange(8.0).view(1, 8, 1, 1).expand(2, 8, 5, 5))


@pytest.mark.parametrize("dev", DEV)
def test_what_is_no_number_stays_in_its_group(dev):
    for shape in ((2, 16, 9, 9), (2, 16, 150, 150)):
        x, w, b, _ = inputs(shape, FP32)
        clean = group_norm_act(x.to(dev), 4, w.to(dev), b.to(dev), act="relu")
        x[1, 5, 3, 3] = math.inf
        x[0, 0, 0, 0] = math.nan
        y = group_norm_act(x.to(dev), 4, w.to(dev), b.to(dev), act="relu")
        bad = torch.zeros(2, 16, dtype=torch.bool)
        bad[1, 4:8] = bad[0, 0:4] = True
        assert torch.isnan(y).flatten(2).any(2).cpu().equal(bad)
        assert torch.equal(y.cpu()[~bad], clean.cpu()[~bad])


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("shape", [(2, 16, 8, 8), (2, 16, 130, 130)])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_relu_holds_back_gradients_that_are_no_numbers(dev, shape, bad):
    x, w, b, dy = inputs(shape, FP32)
    grads = []
    for fill in (0.0, bad):
        leaves = [t.to(dev).requires_grad_(True) for t in (x, w, b)]
        y = group_norm_act(leaves[0], 4, leaves[1], leaves[2], act="relu")
        assert (y == 0).any()
        grads.append(torch.autograd.grad(y, leaves, torch.where(y.detach() == 0, fill, dy.to(dev))))
    for a, c in zip(*grads):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dev", DEV)
def test_orders_of_memory(dev):
    x, w, b, dy = inputs((2, 16, 6, 7), BF16)
    for layout in (lambda v: v, lambda v: v.contiguous(memory_format=torch.channels_last),
                   lambda v: v.transpose(2, 3).contiguous().transpose(2, 3),
                   lambda v: torch.cat([v, v], 1)[:, :16], lambda v: torch.cat([v.new_zeros(1), v.flatten()])[1:].view(v.shape)):
        check(dev, x, 4, w, b, "swish", dy, layout=layout)
    # channels last at an odd address
    room = torch.zeros(x.numel() + 1, dtype=BF16)
    check(dev, x, 4, w, b, "swish", dy, layout=lambda v: room.to(dev)[1:].view(2, 6, 7, 16).permute(0, 3, 1, 2).copy_(v))


@pytest.mark.parametrize("dev", DEV)
def test_a_gradient_that_is_broadcast(dev):
    x, w, b, _ = inputs((2, 16, 6, 7), FP32)
    want = oracle(x, 4, w, b, 1e-5, "swish", torch.ones_like(x))
    xd = x.to(dev).requires_grad_(True)
    group_norm_act(xd, 4, w.to(dev), b.to(dev), act="swish").sum().backward()
    close(xd.grad, want["dx"], want["dx_size"])


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("shape", [(0, 8, 3, 3), (2, 8, 0, 3), (0, 8)])
def test_empty_maps(dev, shape):
    x = torch.zeros(shape, device=dev, requires_grad=True)
    w = torch.ones(8, device=dev, requires_grad=True)
    y = group_norm_act(x, 2, w, act="relu")
    assert y.shape == shape
    y.sum().backward()
    assert x.grad.shape == shape and not w.grad.any()


def test_the_formula_against_differences():
    x, w, b, dy = inputs((2, 6, 3, 2), FP32)
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    want = oracle(x, 3, w, b, 1e-5, "swish", dy)
    value = lambda x_, w_, b_: float((oracle(x_, 3, w_, b_, 1e-5, "swish", dy)["y"] * dy).sum())  # noqa: E731
    h = 1e-5    # the error of a central difference is h^2 times a third derivative, and 2^-52/h of the sum
    for i, name in ((0, "dx"), (1, "dw"), (2, "db")):
        for k in range((x, w, b)[i].numel()):
            up, down = ([t.clone() for t in (x, w, b)] for _ in range(2))
            up[i].view(-1)[k] += h
            down[i].view(-1)[k] -= h
            assert abs((value(*up) - value(*down)) / (2 * h) - float(want[name].reshape(-1)[k])) < 1e-6


def test_refusals():
    x = torch.zeros(2, 8, 3, 3)
    for bad in (dict(act="gelu"), dict(num_groups=3), dict(num_groups=0), dict(eps=-1.0),
                dict(weight=torch.ones(7)), dict(bias=torch.ones(8, 1))):
        with pytest.raises(ValueError):
            group_norm_act(x, **{"num_groups": 2, **bad})
    with pytest.raises(ValueError):
        group_norm_act(torch.zeros(8), 2)
    for bad in (dict(x=x.double()), dict(x=x.long()), dict(weight=torch.ones(8).double()),
                dict(weight=torch.ones(8), bias=torch.zeros(8).bfloat16(), x=x.bfloat16())):
        with pytest.raises(TypeError):
            group_norm_act(**{"x": x, "num_groups": 2, **bad})
    if torch.cuda.is_available():
        with pytest.raises(ValueError):
            group_norm_act(x.cuda(), 2, torch.ones(8))


def test_a_second_derivative_is_refused():
    if not torch.cuda.is_available():
        pytest.skip("the CPU path is differentiable twice")
    x = torch.randn(2, 8, 3, 3, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(group_norm_act(x, 2, act="swish").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@GPU
@pytest.mark.parametrize("shape,groups", [((4, 32, 16, 16), 8), ((2, 32, 120, 120), 4)])
def test_captured_and_replayed(shape, groups):
    def data(seed):
        return [t.cuda() for t in inputs(shape, BF16, seed=seed)]

    x, w, b, dy = data(0)
    x = x.contiguous(memory_format=torch.channels_last).requires_grad_(True)
    w.requires_grad_(True)
    b.requires_grad_(True)

    def go():
        y = group_norm_act(x, groups, w, b, act="swish")
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]

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
            for t, v in zip((x, w, b, dy), data(seed)):
                t.copy_(v)
        eager = go()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(held, eager):
            assert torch.equal(a, c)


@GPU
def test_two_streams_at_once():
    sets = [[t.cuda() for t in inputs((8, 64, 40, 40), BF16, seed=s)] for s in range(2)]
    alone = [group_norm_act(x, 8, w, b, act="swish") for x, w, b, _ in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, (x, w, b, _) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(group_norm_act(x, 8, w, b, act="swish"))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y, alone[i])


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((2200, 1024, 31, 31), 32), ((12, 256, 840, 840), 4)])
def test_offsets_beyond_32_bits(shape, groups):
    """The last samples of a map of more than 2^31 values are what they are by themselves."""
    g = torch.Generator("cuda").manual_seed(3)
    make = lambda: torch.randn(shape[0], *shape[2:], shape[1], generator=g, device="cuda",  # noqa: E731
                               dtype=BF16).movedim(-1, 1)
    x, dy = make().requires_grad_(True), make()
    assert x.numel() * 2 > 2 ** 32
    w = torch.rand(shape[1], generator=g, device="cuda", dtype=torch.float32).to(BF16) + 0.5
    y = group_norm_act(x, groups, w, act="swish")
    dx, = torch.autograd.grad(y, x, dy)
    last = x.detach()[-2:].clone(memory_format=torch.channels_last).requires_grad_(True)
    y2 = group_norm_act(last, groups, w, act="swish")
    dx2, = torch.autograd.grad(y2, last, dy[-2:])
    # one sample's sums may be cut in other parts there: a step of bf16, and of values near 0 one of those near 1
    for a, b in ((y[-2:], y2), (dx[-2:], dx2)):
        assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=2.0 ** -12)


def offset_bounds(x, groups, w, b, act, dy, chain=96, eps=1e-5):
    """The gradients in 64 bits, and how far fp32 arithmetic may be off them where a mean lies far from zero.

    f is half a step of fp32, `most` the largest |x| rstd of a group, and no sum is longer than `chain` additions in a
    row. A mean is off by chain f of |x|, and so is each xhat, in spreads: `shift` = chain f most. z = x a + c adds four
    roundings of that size. What follows is linear in `most`: sum dz xhat may be taken as rstd sum dz x + c sum dz, whose
    terms are |dz| most, and dx as dz a + (x p + q), whose last terms are |mean u xhat| most."""
    f = 2.0 ** -24
    n, c = x.shape[:2]
    s = oracle(x, groups, w, b, eps, act, dy)
    col = (1, c) + (1,) * (x.dim() - 2)
    w64, b64, dy64 = w.double().view(col), b.double().view(col), s["dy"].double()
    per = lambda t: t.reshape(n, groups, -1)  # noqa: E731
    back = lambda t: t.expand(n, groups, per(x).size(2)).reshape(x.shape)  # noqa: E731
    mean = lambda t: back(per(t).mean(2, keepdim=True))  # noqa: E731
    g = per(x.double())
    d = g - g.mean(2, keepdim=True)
    r = (d.square().mean(2, keepdim=True) + eps).rsqrt()
    xhat, most, rs = back(d * r), back(g.abs().amax(2, keepdim=True) * r), back(r)
    z = xhat * w64 + b64
    sig = torch.sigmoid(z)
    slope, bend = (sig * (1 + z * (1 - sig)), 0.5) if act == "swish" else (torch.ones_like(z), 0.0)
    dz = dy64 * slope
    u, shift = dz * w64, chain * f * most
    m1, m2 = mean(u).abs(), mean(u * xhat).abs()
    z_err = w64.abs() * (shift + 4 * f * most) + 2 * f * (z.abs() + b64.abs())
    dz_err = (dy64.abs() * (bend * z_err + 8 * f) if act == "swish" else 0.0) + 2 * f * dz.abs()
    u_err = dz_err * w64.abs() + f * u.abs()
    m1_err = mean(u_err) + chain * f * mean(u.abs())
    m2_err = mean(u_err * xhat.abs()) + (2 * chain * f * most + shift) * mean(u.abs())
    # both factors of the last term are off: (xhat + d)(m2 + e) - xhat m2 = xhat e + d m2 + d e, with d up to
    # shift + 6 f most, and the last of these is no smaller than the others where a large group's m2 is near 0
    dx = rs * (u_err + m1_err + xhat.abs() * m2_err + (m2 + m2_err) * (shift + 6 * f * most)
               + (chain + 8) * f * (u.abs() + m1 + xhat.abs() * m2))
    red = [0] + list(range(2, x.dim()))
    dw = (dz_err * xhat.abs() + (2 * chain * f * most + shift) * dz.abs() + (chain + 8) * f * (dz * xhat).abs()).sum(red)
    db = (dz_err + chain * f * dz.abs()).sum(red)
    return s, [(s["dx"], dx), (s["dw"], dw), (s["db"], db)]


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("shape,groups", [((2, 16, 40, 40), 8), ((2, 16, 150, 150), 8), ((2, 15, 20, 20), 5), ((3, 64, 28, 28), 16),
                                          ((2, 256, 56, 56), 64), ((40, 24, 6, 6), 6), ((2, 12, 31, 33), 4), ((500, 16, 2, 2), 2)])
def test_a_variance_between_channels_with_a_mean_far_from_zero(dev, shape, groups):
    """Channels that lie a spread apart at a mean of 1000: the variance is that of their means, whose rounding at 1000
    (6e-5) is no part of it. It is a sum of squares of at most 64 additions in a row, each 2^-24 of it, around a mean
    that is off by at most 64 2^-24 of 1000 spreads, which the variance has squared; rstd has half of these, and the
    quotient and root three roundings. rstd is what the results say: the regression of y - mean y on x - mean x, where
    errors that all values share fall out and those of their own, 2 2^-24 of up to 4 each, are averaged."""
    g = torch.Generator().manual_seed(9)
    n, c = shape[:2]
    x = 1000.0 + torch.randn(1, c, 1, 1, generator=g) + 0.05 * torch.randn(*shape, generator=g)
    y = group_norm_act(x.to(dev), groups).cpu().double().reshape(n, groups, -1)
    d = x.double().reshape(n, groups, -1)
    d = d - d.mean(2, keepdim=True)
    var = d.square().mean(2)
    want = (var + 1e-5).rsqrt()
    got = (d * (y - y.mean(2, keepdim=True))).mean(2) / var
    f, most = 2.0 ** -24, 1010.0 * want
    assert ((got / want - 1).abs() <= 32 * f + 0.5 * (64 * f * most) ** 2 + 3 * f + 8 * f).all()


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("act,mean", [("none", 1000.0), ("none", 30.0), ("swish", 30.0), ("swish", -30.0), ("swish", 3.0)])
@pytest.mark.parametrize("shape,groups", [((2, 16, 40, 40), 2), ((2, 16, 150, 150), 2), ((2, 15, 20, 20), 3),
                                          ((3, 64, 28, 28), 8), ((2, 256, 56, 56), 32), ((40, 24, 6, 6), 4)])
def test_gradients_with_a_mean_far_from_zero(dev, act, mean, shape, groups):
    """The digits that the mean costs its own rounding are all that it costs a gradient."""
    x, w, b, dy = inputs(shape, FP32, mean=mean)
    s, bounds = offset_bounds(x, groups, w, b, act, dy)
    for want, tol in bounds:        # what is no gradient does not pass
        for wrong in (torch.zeros_like(want), -want):
            assert ((wrong - want).abs() > tol + 2.0 ** -24 * want.abs()).any()
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w, b)]
    y = group_norm_act(leaves[0], groups, leaves[1], leaves[2], act=act)
    got = torch.autograd.grad(y, leaves, s["dy"].to(dev))
    for name, a, (want, tol) in zip(("dx", "dw", "db"), got, bounds):
        err, tol = (a.cpu().double() - want).abs(), tol + 2.0 ** -24 * want.abs()
        assert (err <= tol).all(), f"{name} off by {float((err / tol).max()):.3g} of the tolerance"


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("t", [FP32, BF16, FP16])
@pytest.mark.parametrize("shape,groups", [((2, 4096, 3, 3), 1), ((3, 8192, 2, 2), 2), ((1, 16384, 2, 1), 1), ((2, 32768, 3, 1), 2),
                                          ((2, 6001, 5, 5), 1), ((1, 2049, 1, 1), 1), ((70, 4104), 2), ((1, 16384, 30, 30), 1)])
def test_groups_of_many_channels(dev, t, shape, groups):
    """More channels a group than a workgroup holds: up to 16384, whose sums wait in LDS until they are joined."""
    x, w, b, dy = inputs(shape, t)
    check(dev, x, groups, w, b, "swish", dy)


@GPU
def test_a_group_of_too_many_channels_is_refused():
    with pytest.raises(RuntimeError, match="16384"):
        group_norm_act(torch.zeros(2, 16385, device="cuda"), 1)


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("t", [FP32, BF16])
@pytest.mark.parametrize("where", [(0, 0, 0), (-1, -1, -1), (1, 3, 2)])
@pytest.mark.parametrize("shape,groups", [((2, 16, 40, 40), 2), ((2, 16, 150, 150), 2), ((2, 15, 20, 20), 3), ((3, 64, 1, 2), 8)])
def test_an_outlier_wherever_it_lies(dev, t, where, shape, groups):
    """One value ten thousand times the others, at a group's ends or within: it costs the others no digits."""
    x, w, b, dy = inputs(shape, t)
    c, h, v = (i % n if i < 0 else min(i, n - 1) for i, n in zip(where, (shape[1] // groups, *shape[2:])))
    x[:, c, h, v] = 1e4
    x[:, shape[1] // groups + c, h, v] = -1e4
    check(dev, x, groups, w, b, "none", dy)


@GPU
@pytest.mark.parametrize("mean", [1000.0, 30.0, 0.5])
@pytest.mark.parametrize("act", ["none", "swish"])
@pytest.mark.parametrize("shape,groups", [((2, 16, 150, 150), 2), ((2, 16, 40, 40), 2), ((2, 256, 56, 56), 32), ((2, 15, 20, 20), 3)])
def test_results_lose_no_more_than_the_formula_in_fp32(mean, act, shape, groups):
    """The kernels' errors against 64 bits, as a share of a result's norm, are at most twice those of the formula that
    torch computes step by step in fp32, where x less its mean comes first, and four roundings: both are off by what the
    mean's rounding costs (which may be more on one side than on the other) and by their sums' own."""
    from fast_autoaugment_amd.ops.groupnorm import _composed
    x, w, b, dy = inputs(shape, FP32, mean=mean)
    want = oracle(x, groups, w, b, 1e-5, act, dy)
    off = []
    for fn in (lambda *v: group_norm_act(v[0], groups, v[1], v[2], act=act), lambda *v: _composed(v[0], groups, v[1], v[2], 1e-5, act)):
        leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
        y = fn(*leaves)
        got = [y.detach(), *torch.autograd.grad(y, leaves, dy.cuda())]
        off.append([float((a.cpu().double() - want[k]).norm() / want[k].norm()) for a, k in zip(got, ("y", "dx", "dw", "db"))])
    for k, ours, formula in zip(("y", "dx", "dw", "db"), *off):
        assert ours <= 2 * formula + 4 * 2.0 ** -24, (k, ours, formula)
