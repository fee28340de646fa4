"""AdamW over many tensors: the CPU path against the formula in 64 bits, and what is refused."""
import math

import pytest
import torch
from torch import nn

from fast_autoaugment_amd.optim import FusedAdamW
from fast_autoaugment_amd.parallel.flat import FlatParams, flatten_module

SHAPES = [(16, 3, 3, 3), (16,), (5,), (7, 33), (1,), (300, 9), (257,)]
DEV = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def e4m3_near(ratio):
    """The e4m3 numbers that `ratio` may be rounded to by arithmetic of 32 bits: those of a little below and above it.

    ratio = moment * (448 / largest): the moment has three roundings (two products, a sum) and a root one more and
    half of v's, the quotient one, the product one: 8 of 2^-24 of the terms. The terms of a sum are up to 2^4 times
    the sum for all but a few elements, so 2^-17 of the ratio."""
    held = []
    for r in (ratio * (1 - 2.0 ** -17), ratio * (1 + 2.0 ** -17)):
        grid = torch.exp2(torch.floor(torch.log2(r.abs().clamp_min(2.0 ** -6))) - 3)
        held.append(torch.round(r / grid) * grid)
    return held


def check_step(opt, before, grads, weights, decays, lr, clip, betas=(0.9, 0.999), eps=1e-8):
    """One step of `opt` from the state `before` against the formula in 64 bits.

    Weights: one fp32 rounding of p keep, one of the difference, and the update (below 10 lr in size here) to about
    ten roundings of itself. Moments: three roundings of terms whose sizes are their own tolerance."""
    (b1, b2), t = betas, before["t"] + 1
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads if g is not None))
    coef = min(1.0, clip / (norm + 1e-6)) if clip > 0 else 1.0
    assert int(opt.step_count) == t
    second = "exp_avg_sq" if opt.state_bits == 32 else "exp_avg_root"
    offs = [(off, n) for off, n, _ in opt._items] if opt.flat is None else before["places"]
    for (off, n), g, w0, w1, wd in zip(offs, grads, before["w"], weights, decays):
        if g is None:
            continue
        order = lambda x: x.detach().cpu().as_strided((n,), (1,)).double()  # noqa: E731
        g = order(g) * coef
        m0, r0 = before["m"][off:off + n], before["r"][off:off + n]
        v0 = r0 if opt.state_bits == 32 else r0.square()
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
        upd = lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
        w = order(w0) * (1 - lr * wd) - upd
        m_size = b1 * m0.abs() + (1 - b1) * g.abs()
        tol = 2.0 ** -24 * (2 * order(w0).abs() + 2 * upd.abs() + 12 * upd.abs() * (m_size / m.abs().clamp_min(1e-30)))
        assert ((order(w1) - w).abs() <= tol + 1e-30).all()
        if opt.state_bits == 32:
            assert ((opt.exp_avg[off:off + n].cpu().double() - m).abs() <= 2.0 ** -22 * m_size).all()
            assert ((opt.exp_avg_sq[off:off + n].cpu().double() - v).abs() <= 2.0 ** -21 * v).all()
            continue
        hi = -(-n // 256)
        for name, x, least in (("exp_avg", m, 0.0), (second, v.sqrt(), 2.0 ** -9)):
            blocks = torch.zeros(hi * 256, dtype=torch.float64)
            blocks[:n] = x
            blocks = blocks.view(-1, 256)
            scale = getattr(opt, name + "_scale")[off // 256:off // 256 + hi].cpu().double()
            want = blocks.abs().amax(1).clamp_min(2.0 ** -100) / 448
            assert ((scale - want).abs() <= 2.0 ** -20 * want).all()
            lo, up = e4m3_near(blocks / want[:, None])
            if least:
                lo, up = (torch.where(blocks > 0, h.clamp_min(least), h) for h in (lo, up))
            got = getattr(opt, name).float().cpu().double()[off:off + hi * 256].view(-1, 256)
            wrong = (got != lo) & (got != up)
            assert int(wrong.sum()) <= 1 + n // 1000 and ((got - lo).abs() <= lo.abs() / 8 + 2.0 ** -9).all()


def state_of(opt, weights, places=None):
    whole = lambda name: opt._moment(name, 0, getattr(opt, name).numel()).double()  # noqa: E731
    cpu = {k: getattr(opt, k) for k in opt._names}
    for k, v in cpu.items():
        setattr(opt, k, v.cpu())
    s = dict(t=int(opt.step_count), m=whole("exp_avg"), r=whole("exp_avg_sq" if opt.state_bits == 32 else "exp_avg_root"),
             w=[w.detach().clone() for w in weights], places=places)
    for k, v in cpu.items():
        setattr(opt, k, v)
    return s


def tensors(dtype, dev, seed=0, shapes=SHAPES):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * 0.1).to(dtype).to(dev) for s in shapes]


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("clip", [0.0, 0.5])
def test_list_follows_the_formula(dev, bits, dtype, clip):
    ws = tensors(dtype, dev)
    params = [nn.Parameter(w) for w in ws]
    opt = FusedAdamW([{"params": params[:4]}, {"params": params[4:], "weight_decay": 0.0}], lr=1e-2,
                     weight_decay=0.1, grad_clip=clip, state_bits=bits)
    full = [p if m is None else m for p, m in zip(params, opt.masters)]
    for step in range(4):
        grads = tensors(dtype, dev, seed=10 + step)
        for p, g in zip(params, grads):
            p.grad = g
        before = state_of(opt, full)
        opt.step()
        check_step(opt, before, grads, full, [0.1] * 4 + [0.0] * 3, 1e-2, clip)
    for p, w in zip(params, full):      # the copy is the fp32 weight rounded once
        assert torch.equal(p.detach(), w.detach().to(dtype))


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_flat_follows_the_formula_and_leaves_padding(dev, bits, dtype):
    model = nn.Sequential(nn.Conv2d(3, 7, 3), nn.BatchNorm2d(7), nn.Flatten(), nn.Linear(63, 11)).to(dev)
    flat = flatten_module(model, align=256, work_dtype=dtype)
    opt = FusedAdamW(flat, lr=1e-2, weight_decay=0.1, grad_clip=1.0, state_bits=bits)
    full = flat.flat_param if flat.flat_master is None else flat.flat_master
    places = [((p.data_ptr() - flat.flat_param.data_ptr()) // p.element_size(), p.numel()) for p in flat.params]
    weights = [full[o:o + n] for o, n in places]
    for step in range(3):
        g = torch.Generator().manual_seed(step)
        for p in flat.params:
            p.grad.copy_(torch.randn(p.shape, generator=g))
        before = state_of(opt, weights, places)
        opt.step()
        check_step(opt, before, [flat.flat_grad[o:o + n] for o, n in places], weights,
                   [0.1 if o < flat.n_decay else 0.0 for o, _ in places], 1e-2, 1.0)
    used = torch.zeros(flat.numel, dtype=torch.bool)
    for o, n in places:
        used[o:o + n] = True
    assert not full.cpu()[~used].any() and not flat.flat_param.cpu()[~used].any()


@pytest.mark.parametrize("dev", DEV)
def test_a_parameter_without_a_gradient_stays(dev):
    params = [nn.Parameter(w) for w in tensors(torch.float32, dev)]
    before = [p.detach().clone() for p in params]
    opt = FusedAdamW(params, lr=1e-2, weight_decay=0.1, grad_clip=1.0)
    params[3].grad = torch.ones_like(params[3])
    opt.step()
    for i, (p, b) in enumerate(zip(params, before)):
        assert torch.equal(p.detach(), b) == (i != 3)


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("bits", [32, 8])
def test_state_survives_saving(dev, bits, tmp_path):
    def make():
        params = [nn.Parameter(w) for w in tensors(torch.bfloat16, dev)]
        return params, FusedAdamW(params, lr=1e-2, weight_decay=0.1, state_bits=bits)

    def go(params, opt, steps):
        for step in steps:
            for p, g in zip(params, tensors(torch.bfloat16, dev, seed=step)):
                p.grad = g
            opt.step()

    a, opt_a = make()
    go(a, opt_a, range(4))
    b, opt_b = make()
    go(b, opt_b, range(2))
    torch.save({"opt": opt_b.state_dict(), "w": [p.detach() for p in b]}, tmp_path / "s.pth")
    sd = torch.load(tmp_path / "s.pth", weights_only=True)
    c, opt_c = make()
    with torch.no_grad():
        for p, w in zip(c, sd["w"]):
            p.copy_(w)
    opt_c.load_state_dict(sd["opt"])
    go(c, opt_c, range(2, 4))
    for x, y in zip(a, c):
        assert torch.equal(x.detach(), y.detach())


@pytest.mark.parametrize("dev", DEV)
def test_a_second_moment_is_never_lost(dev):
    """A root far below its block's largest is held as the smallest number, and not as zero."""
    p = nn.Parameter(torch.zeros(256, device=dev))
    p.grad = torch.full((256,), 1e-12, device=dev)
    p.grad[0] = 1.0
    opt = FusedAdamW([p], lr=1e-3, state_bits=8)
    for _ in range(3):
        opt.step()
    assert (opt.exp_avg_root.float() > 0).all()
    assert torch.isfinite(p.detach()).all() and p.detach().abs().max() < 0.01


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("bits", [32, 8])
def test_a_gradient_that_is_no_number_shows(dev, bits):
    p = nn.Parameter(torch.zeros(600, device=dev))
    p.grad = torch.ones(600, device=dev)
    p.grad[300] = math.nan
    opt = FusedAdamW([p], lr=1e-3, state_bits=bits)
    opt.step()
    assert torch.isnan(p.detach()).nonzero().flatten().tolist() == [300]
    q = nn.Parameter(torch.zeros(600, device=dev))
    q.grad = p.grad.clone()
    opt = FusedAdamW([q], lr=1e-3, grad_clip=1.0, state_bits=bits)
    opt.step()
    assert torch.isnan(q.detach()).all()


def test_refusals():
    p = lambda n=3, t=torch.float32: nn.Parameter(torch.zeros(n, dtype=t))  # noqa: E731
    for bad in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=0.0), dict(lr=-1.0),
                dict(weight_decay=-1.0), dict(grad_clip=-1.0), dict(state_bits=16)):
        with pytest.raises(ValueError):
            FusedAdamW([p()], **bad)
    with pytest.raises(ValueError):
        FusedAdamW([])
    with pytest.raises(ValueError):
        FusedAdamW([{"params": []}])
    with pytest.raises(ValueError):
        FusedAdamW([{"params": [p()], "lr": 0.1}])
    with pytest.raises(TypeError):
        FusedAdamW([p(3, torch.float64)])
    q = p()
    with pytest.raises(ValueError):
        FusedAdamW([q, q])
    opt = FusedAdamW([q])
    with pytest.raises(ValueError):
        opt.load_state_dict(FusedAdamW([p()], state_bits=8).state_dict())
    with pytest.raises(ValueError):
        opt.load_state_dict(FusedAdamW([p(300)]).state_dict())
    with pytest.raises(ValueError):
        opt.load_state_dict({"momentum_buf": torch.zeros(3)})
    q.grad = torch.zeros(3).to_sparse()
    with pytest.raises(TypeError):
        opt.step()
    strided = nn.Parameter(torch.zeros(4, 6)[:, ::2])
    strided.grad = torch.zeros(4, 3)
    with pytest.raises(ValueError):
        FusedAdamW([strided]).step()
    model = nn.Sequential(nn.Linear(3, 5), nn.Linear(5, 2))
    with pytest.raises(ValueError):
        FusedAdamW(flatten_module(model, align=64), state_bits=8)
    low = torch.zeros(256, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        FusedAdamW(FlatParams(low, low.clone(), 256, [], None))


@pytest.mark.parametrize("dev", DEV)
def test_orders_of_memory(dev):
    """Channels-last weights, gradients in another order than their weights, and views that no vector load fits."""
    w = torch.randn(8, 4, 3, 3, generator=torch.Generator().manual_seed(0)).to(dev)
    g = torch.randn(8, 4, 3, 3, generator=torch.Generator().manual_seed(1)).to(dev)
    ref = nn.Parameter(w.clone())
    ref.grad = g.clone()
    FusedAdamW([ref], lr=0.1, weight_decay=0.1).step()
    for wl in (False, True):
        for gl in (False, True):
            fmt = lambda t, last: t.clone(memory_format=torch.channels_last if last else torch.contiguous_format)  # noqa: E731
            p = nn.Parameter(fmt(w, wl))
            p.grad = fmt(g, gl)
            FusedAdamW([p], lr=0.1, weight_decay=0.1).step()
            assert torch.equal(p.detach(), ref.detach())
    room = torch.zeros(w.numel() + 1, device=dev)
    p = nn.Parameter(room[1:].copy_(w.flatten()).view(8, 4, 3, 3))
    p.grad = torch.cat([g.new_zeros(1), g.flatten()])[1:].view(8, 4, 3, 3)
    FusedAdamW([p], lr=0.1, weight_decay=0.1).step()
    assert torch.equal(p.detach(), ref.detach())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_follow_eager_ones(bits):
    def make():
        params = [nn.Parameter(w) for w in tensors(torch.bfloat16, "cuda")]
        for p in params:
            p.grad = torch.zeros_like(p)
        return params, FusedAdamW(params, lr=1e-2, weight_decay=0.1, grad_clip=0.5, state_bits=bits)

    def fill(params, step):
        for p, g in zip(params, tensors(torch.bfloat16, "cuda", seed=step)):
            p.grad.copy_(g)

    a, opt_a = make()
    b, opt_b = make()
    for opt, ps in ((opt_a, a), (opt_b, b)):
        fill(ps, 0)
        opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt_b.step()
    assert int(opt_b.step_count) == 1
    for step in range(1, 6):
        opt_a.param_groups[0]["lr"] = opt_b.param_groups[0]["lr"] = 1e-2 / step
        fill(a, step)
        fill(b, step)
        opt_a.step()
        opt_b.sync_lr()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(a, b):
            assert torch.equal(x.detach(), y.detach())
    assert int(opt_b.step_count) == 6
    a[0].grad = torch.zeros_like(a[0])
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt_a.step()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [0.0, 0.5])
def test_the_gpu_s_moments_are_the_cpu_s(bits, clip):
    """Bit for bit, over steps that build on each other: a rounding more or less would show in 8 bits now and then."""
    out = []
    for dev in ("cpu", "cuda"):
        p = nn.Parameter(tensors(torch.bfloat16, dev, shapes=[(200_000,)])[0])
        opt = FusedAdamW([p], lr=1e-2, weight_decay=0.1, grad_clip=clip, state_bits=bits)
        for step in range(4):
            p.grad = tensors(torch.bfloat16, dev, seed=30 + step, shapes=[(200_000,)])[0]
            opt.step()
        out.append([getattr(opt, k).float().cpu() for k in opt._names])
    for x, y in zip(*out):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_gpu_refusals():
    p = nn.Parameter(torch.zeros(300, device="cuda"))
    p.grad = torch.ones(300, device="cuda")
    opt = FusedAdamW([p])
    opt.step()
    p.grad = torch.ones(300, device="cuda").to_sparse()
    with pytest.raises(TypeError):
        opt.step()
    p.grad = torch.ones(300, device="cuda")
    p.data = torch.zeros(200, device="cuda")
    p.grad = torch.ones(200, device="cuda")
    with pytest.raises(ValueError):
        opt.step()
    with pytest.raises(ValueError):
        FusedAdamW([nn.Parameter(torch.zeros(3, device="cuda")), nn.Parameter(torch.zeros(3))])


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("before,after", [(torch.float32, torch.bfloat16), (torch.float16, torch.float32)])
def test_a_parameter_that_changes_its_type_is_refused(dev, before, after):
    """Its fp32 weights would be read from memory of another type and length."""
    p = nn.Parameter(tensors(before, dev, shapes=[(5000,)])[0])
    opt = FusedAdamW([p])
    p.grad = torch.zeros_like(p)
    opt.step()
    p.grad = None
    p.data = p.data.to(after)
    p.grad = torch.zeros_like(p)
    with pytest.raises((TypeError, ValueError), match="changed its size, type"):
        opt.step()


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("bits", [32, 8])
def test_weights_that_were_loaded_are_taken_over(dev, bits):
    """Weights loaded behind the optimizer's back are stepped from, and those it wrote itself keep their fp32 digits."""
    p = nn.Parameter(tensors(torch.bfloat16, dev, shapes=[(5000,)])[0])
    opt = FusedAdamW([p], lr=1e-3, state_bits=bits)
    for step in range(3):
        p.grad = torch.ones_like(p)
        opt.step()
        held = opt.masters[0].clone()
        with torch.no_grad():
            p[:2000] = 3.0
        opt.lr = opt.param_groups[0]["lr"] = 0.0
        opt.step()
        # a step of lr 1e-3 from 3 still rounds to 3 in bf16 (its numbers lie 2^-6 apart there), and is kept
        want = torch.where(held[:2000].bfloat16() == 3.0, held[:2000], 3.0)
        assert torch.equal(opt.masters[0], torch.cat([want, held[2000:]])) and (p.detach()[:2000] == 3.0).all()
        opt.param_groups[0]["lr"] = 1e-3
    assert not torch.equal(held[2000:], held[2000:].bfloat16().float())


@pytest.mark.gpu
def test_a_captured_step_outlives_new_gradients():
    """A graph keeps the tables it was captured with, whatever eager steps on other gradients make later."""
    p = nn.Parameter(torch.zeros(5000, device="cuda"))
    first = p.grad = torch.ones(5000, device="cuda")
    opt = FusedAdamW([p], lr=1e-2)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    held = []
    for i in range(4):
        p.grad = torch.full((5000,), float(i), device="cuda")
        opt.step()
        held.append(torch.full((64,), -1, dtype=torch.int64, device="cuda"))      # where old tables may have been
    torch.cuda.synchronize()
    first.fill_(1.0)
    before, moment = p.detach().clone(), opt.exp_avg.clone()
    graph.replay()
    torch.cuda.synchronize()
    want = 0.9 * moment[:5000] + 0.1 * first
    assert torch.allclose(opt.exp_avg[:5000], want, rtol=2.0 ** -22) and not torch.equal(before, p.detach())


@pytest.mark.gpu
def test_new_gradients_every_step_and_another_stream():
    a = [nn.Parameter(w) for w in tensors(torch.float32, "cuda")]
    b = [nn.Parameter(w.clone()) for w in tensors(torch.float32, "cuda")]
    opt_a, opt_b = FusedAdamW(a, grad_clip=1.0), FusedAdamW(b, grad_clip=1.0)
    side = torch.cuda.Stream()
    for step in range(5):
        grads = tensors(torch.float32, "cuda", seed=step)
        for p, q, g in zip(a, b, grads):
            p.grad, q.grad = g, g.clone()
        opt_a.step()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            opt_b.step()
        torch.cuda.current_stream().wait_stream(side)
        opt_a.zero_grad(set_to_none=True)
        opt_b.zero_grad(set_to_none=True)
    for p, q in zip(a, b):
        assert torch.equal(p.detach(), q.detach())


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("n", [1, 3, 255, 256, 4095, 4096, 4097, 300_001])
@pytest.mark.parametrize("bits", [32, 8])
def test_odd_lengths(dev, n, bits):
    p = nn.Parameter(tensors(torch.float32, dev, shapes=[(n,)])[0])
    opt = FusedAdamW([p], lr=1e-2, weight_decay=0.1, grad_clip=0.5, state_bits=bits)
    for step in range(2):
        p.grad = tensors(torch.float32, dev, seed=5 + step, shapes=[(n,)])[0]
        before = state_of(opt, [p])
        opt.step()
        check_step(opt, before, [p.grad], [p], [0.1], 1e-2, 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_beyond_32_bits(bits):
    """The end of a tensor of more than 2^31 elements, and the tensor behind it, are stepped as they are alone."""
    g = torch.Generator("cuda").manual_seed(3)
    r = lambda n: torch.randn(n, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    n = 2 ** 31 + 3 * 4096
    weights, grads = [r(n), r(5000)], [r(n), r(5000)]
    end = slice(n - 8192, None)
    got = []
    for ws, gs in ((weights, grads), ([weights[0][end].clone(), weights[1].clone()], [grads[0][end].clone(), grads[1]])):
        ps = [nn.Parameter(w.clone()) for w in ws]
        for p, grad in zip(ps, gs):
            p.grad = grad
        opt = FusedAdamW(ps, lr=1e-2, weight_decay=0.1, state_bits=bits)
        opt.step()
        opt.step()
        held = [getattr(opt, k) for k in opt._names]
        held = [h[-(8192 + 5120) // 256:].float() if k.endswith("scale") else h[-(8192 + 5120):].float()
                for k, h in zip(opt._names, held)]
        got.append([ps[0].detach()[-8192:], ps[1].detach(), opt.masters[0][-8192:], *held])
        del ps, opt
    for a, b in zip(*got):
        assert torch.equal(a, b)



def flat_model(dev, dtype, seed=0):
    torch.manual_seed(seed)
    model = nn.Sequential(nn.Conv2d(3, 7, 3), nn.BatchNorm2d(7), nn.Flatten(), nn.Linear(63, 11)).to(dev)
    return model, flatten_module(model, align=256, work_dtype=dtype)


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("how", ["model", "buffer", "before"])
def test_flat_weights_that_were_loaded_are_taken_over(dev, bits, dtype, how):
    """As those of lists: through the model or the buffer, and those that were loaded before the first step."""
    model, flat = flat_model(dev, dtype)
    opt = FusedAdamW(flat, lr=1e-3, state_bits=bits)

    def load(value):
        if how == "buffer":
            with torch.no_grad():
                flat.flat_param.fill_(value)
        else:
            model.load_state_dict({k: torch.full_like(v, value) for k, v in model.state_dict().items()})

    for step in range(1 if how == "before" else 3):
        if how != "before":
            flat.flat_grad.fill_(1.0)
            opt.step()
        held = flat.flat_master.clone()
        load(3.0)
        opt.param_groups[0]["lr"] = 0.0
        flat.flat_grad.fill_(1.0)
        opt.step()
        # a step of lr 1e-3 from 3 still rounds to 3 in bf16 (its numbers lie 2^-6 apart there), and is kept
        for p in flat.params:
            at = (p.data_ptr() - flat.flat_param.data_ptr()) // p.element_size()
            mine, before = (t[at:at + p.numel()] for t in (flat.flat_master, held))
            assert torch.equal(mine, torch.where(before.to(dtype) == 3.0, before, 3.0)) and (p.detach() == 3.0).all()
        opt.param_groups[0]["lr"] = 1e-3


@pytest.mark.parametrize("dev", DEV)
def test_flat_weights_that_the_step_wrote_keep_their_fp32_digits(dev):
    model, flat = flat_model(dev, torch.bfloat16)
    opt = FusedAdamW(flat, lr=1e-3)
    for step in range(3):
        flat.flat_grad.fill_(1.0)
        opt.step()
    assert not torch.equal(flat.flat_master, flat.flat_param.float())
    held = flat.flat_master.clone()
    with torch.no_grad():
        for p in flat.params:
            p.copy_(p.clone())            # written, and nothing changed
    opt.param_groups[0]["lr"] = 0.0
    opt.step()
    assert torch.equal(flat.flat_master, held)


@pytest.mark.gpu
def test_a_capture_refuses_flat_weights_that_were_written():
    model, flat = flat_model("cuda", torch.bfloat16)
    opt = FusedAdamW(flat, lr=1e-3)
    opt.step()
    with torch.no_grad():
        flat.flat_param.fill_(1.0)
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    graph = torch.cuda.CUDAGraph()
    opt.step()          # an eager one takes them over, and the next is captured
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    flat.flat_grad.fill_(1.0)
    before = flat.flat_master.clone()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert not torch.equal(flat.flat_master, before)
        before = flat.flat_master.clone()


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("order", ["weights first", "state first"])
def test_flat_state_survives_saving(dev, bits, dtype, order, tmp_path):
    """A run that was saved with its weights as the trainer saves them goes on bit by bit."""
    def go(flat, opt, steps):
        for step in steps:
            g = torch.Generator().manual_seed(step)
            for p in flat.params:
                p.grad.copy_(torch.randn(p.shape, generator=g))
            opt.step()

    make = lambda seed: (lambda m: (*m, FusedAdamW(m[1], lr=1e-3, weight_decay=0.1, state_bits=bits)))(  # noqa: E731
        flat_model(dev, dtype, seed))
    _, flat_a, opt_a = make(0)
    go(flat_a, opt_a, range(4))
    model, flat_b, opt_b = make(0)
    go(flat_b, opt_b, range(2))
    torch.save({"opt": opt_b.state_dict(), "model": {k: v.float() for k, v in model.state_dict().items()}}, tmp_path / "s.pth")
    sd = torch.load(tmp_path / "s.pth", weights_only=True)
    model, flat_c, opt_c = make(1)
    if order == "state first":
        opt_c.load_state_dict(sd["opt"])
    model.load_state_dict(sd["model"])
    if dtype != torch.float32:
        flat_c.flat_master.copy_(flat_c.flat_param) if order == "weights first" else None
    if order == "weights first":
        opt_c.load_state_dict(sd["opt"])
    go(flat_c, opt_c, range(2, 4))
    full = lambda f: f.flat_param if f.flat_master is None else f.flat_master  # noqa: E731
    assert torch.equal(full(flat_a), full(flat_c)) and torch.equal(flat_a.flat_param, flat_c.flat_param)
    for n in opt_a._names:
        assert torch.equal(getattr(opt_a, n).float(), getattr(opt_c, n).float())


def test_a_state_of_other_weights_is_refused():
    _, flat = flat_model("cpu", torch.bfloat16)
    opt = FusedAdamW(flat)
    sd = opt.state_dict()
    before = opt.exp_avg.fill_(0.5).clone()
    with pytest.raises(ValueError):
        opt.load_state_dict({**sd, "exp_avg": torch.zeros_like(before), "flat_master": torch.zeros(3)})
    assert torch.equal(opt.exp_avg, before)


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [0.0, 1.0])
def test_flat_fp16_follows_the_formula(dev, bits, clip):
    model, flat = flat_model(dev, torch.float16)
    opt = FusedAdamW(flat, lr=1e-2, weight_decay=0.1, grad_clip=clip, state_bits=bits)
    places = [((p.data_ptr() - flat.flat_param.data_ptr()) // p.element_size(), p.numel()) for p in flat.params]
    weights = [flat.flat_master[o:o + n] for o, n in places]
    for step in range(3):
        g = torch.Generator().manual_seed(step)
        for p in flat.params:
            p.grad.copy_(torch.randn(p.shape, generator=g))
        before = state_of(opt, weights, places)
        opt.step()
        check_step(opt, before, [flat.flat_grad[o:o + n] for o, n in places], weights,
                   [0.1 if o < flat.n_decay else 0.0 for o, _ in places], 1e-2, clip)
        assert torch.equal(flat.flat_param, flat.flat_master.half())
    used = torch.zeros(flat.numel, dtype=torch.bool)
    for o, n in places:
        used[o:o + n] = True
    assert not flat.flat_master.cpu()[~used].any() and not flat.flat_param.cpu()[~used].any()
