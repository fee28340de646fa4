"""The batch-independent operators in the models, the trainer and the policy search."""
import os

import pytest
import torch
from torch import nn

from fast_autoaugment_amd.config import Config as C
from fast_autoaugment_amd.models import build_model, to_group_norm
from fast_autoaugment_amd.models.efficientnet import EfficientNet
from fast_autoaugment_amd.models.folded import fold_for_inference
from fast_autoaugment_amd.models.pyramidnet import PyramidNet
from fast_autoaugment_amd.models.resnet import ResNet
from fast_autoaugment_amd.ops.groupnorm import GroupNormAct
from fast_autoaugment_amd.ops.pointwise import LinearAct
from fast_autoaugment_amd.optim import FusedAdamW
from fast_autoaugment_amd.parallel.flat import flatten_module

DEV = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def small_effnet():
    return EfficientNet.from_name("efficientnet-b0", {"num_classes": 7, "image_size": 32})


def test_norm_group_replaces_every_batch_norm():
    for conf in ({"type": "wresnet40_2"}, {"type": "shakeshake26_2x32d"}, {"type": "efficientnet-b0"},
                 {"type": "pyramid", "depth": 29, "alpha": 30, "bottleneck": True}):
        m = build_model({**conf, "norm": "group", "norm_groups": 8}, 10)
        kinds = [type(x) for x in m.modules()]
        assert nn.BatchNorm2d not in kinds and GroupNormAct in kinds and nn.Linear not in kinds and LinearAct in kinds
        assert all(x.num_channels % x.num_groups == 0 for x in m.modules() if isinstance(x, GroupNormAct))
        plain = build_model(conf, 10)
        want = {k for k in plain.state_dict() if not k.endswith(("running_mean", "running_var", "num_batches_tracked"))}
        assert set(m.state_dict()) == want
    with pytest.raises(NameError):
        build_model({"type": "wresnet40_2", "norm": "layer"}, 10)
    with pytest.raises(ValueError):
        to_group_norm(nn.BatchNorm2d(8), 0)


def test_a_sample_does_not_depend_on_its_batch():
    torch.manual_seed(0)
    for m, size in ((build_model({"type": "wresnet40_2", "norm": "group"}, 10), 32), (to_group_norm(small_effnet(), 8), 32)):
        m.eval()
        x = torch.randn(3, 3, size, size)
        with torch.no_grad():
            whole = m(x)
            one = torch.cat([m(x[i:i + 1]) for i in range(3)])
        assert torch.allclose(whole, one, rtol=1e-4, atol=1e-5)


def step(model, dev, dtype, bits):
    """Gradients of one batch and the weights behind one step."""
    model = model.to(dev).to(memory_format=torch.channels_last)
    flat = flatten_module(model, align=256, work_dtype=dtype)
    opt = FusedAdamW(flat, lr=1e-3, weight_decay=0.05, grad_clip=1.0, state_bits=bits)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(8, 3, 32, 32, generator=g).to(dev, dtype).contiguous(memory_format=torch.channels_last)
    t = torch.randint(0, 7, (8,), generator=g).to(dev)
    loss = nn.functional.cross_entropy(model(x).float(), t)
    loss.backward()
    grads = flat.flat_grad.float().cpu().clone()
    opt.step()
    full = flat.flat_param if flat.flat_master is None else flat.flat_master
    return grads, full.float().cpu()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_training_step_on_the_cpu_is_torch_s(bits):
    """Group norm, fused products and AdamW together, against torch's own modules and its optimizer."""
    torch.manual_seed(0)
    ours = build_model({"type": "wresnet40_2", "norm": "group"}, 7)
    torch.manual_seed(0)
    theirs = build_model({"type": "wresnet40_2", "norm": "group"}, 7)
    for m in theirs.modules():
        if isinstance(m, LinearAct):
            m.__class__ = nn.Linear
    flat = flatten_module(ours, align=256)
    opt = FusedAdamW(flat, lr=1e-3, weight_decay=0.05, state_bits=bits)
    norms = {id(p) for m in theirs.modules() if isinstance(m, nn.GroupNorm) for p in m.parameters()}
    ref = torch.optim.AdamW([{"params": [p for p in theirs.parameters() if id(p) not in norms], "weight_decay": 0.05},
                             {"params": [p for p in theirs.parameters() if id(p) in norms], "weight_decay": 0.0}], lr=1e-3)
    x, t = torch.randn(4, 3, 32, 32), torch.tensor([0, 1, 2, 3])
    for m in (ours, theirs):
        nn.functional.cross_entropy(m(x), t).backward()
    for a, b in zip(ours.parameters(), theirs.parameters()):
        # fp32 moves an activation by some 1e-7 of itself; of the 4 million that relu sees, about one lies that near
        # its border and changes side, and is one of 8192 values or more of its layer: 1/sqrt(8192) of a norm
        assert (a.grad - b.grad).norm() <= 8192 ** -0.5 * b.grad.norm()
        # a first step is lr times nearly the sign of a gradient: both optimizers are given the same ones
        b.grad.copy_(a.grad)
    opt.step()
    ref.step()
    for a, b in zip(ours.parameters(), theirs.parameters()):
        # the update is 1e-3 at most and a few roundings; so is the rest of the weight
        assert torch.allclose(a, b, rtol=4 * 2.0 ** -24, atol=1e-3 * 32 * 2.0 ** -24)


@pytest.mark.gpu
@pytest.mark.parametrize("make", [lambda: build_model({"type": "wresnet40_2", "norm": "group"}, 7),
                                  lambda: to_group_norm(ResNet("cifar10", 29, 7, bottleneck=True), 8)])
def test_a_training_step_on_the_gpu_is_the_cpu_s(make):
    """In fp32 the two paths differ by the order of their sums: gradients agree to what values at relu's border
    make of it (one or two of a layer's 8192 or more), and as a step is lr at most, weights to twice that."""
    torch.backends.cuda.matmul.allow_tf32 = False
    out = []
    for dev in ("cpu", "cuda"):
        torch.manual_seed(0)
        m = make()
        out.append(step(m, dev, torch.float32, 32))
    (g0, w0), (g1, w1) = out
    assert (g0 - g1).norm() <= 2 ** 0.5 * 8192 ** -0.5 * g0.norm()
    assert (w0 - w1).abs().max() <= 2.1e-3


@pytest.mark.gpu
def test_a_bf16_training_step_with_every_operator():
    """EfficientNet with group norm, swish, fused squeeze-and-excitation and 8-bit AdamW in the trainer's flat bf16."""
    torch.manual_seed(0)
    m = to_group_norm(small_effnet(), 8)
    from fast_autoaugment_amd.ops.pointwise import fuse_pointwise
    assert fuse_pointwise(m) > 30
    m._dropout.p = 0.0
    m.eval()
    ref = step(m, "cpu", torch.float32, 32)[0]
    torch.manual_seed(0)
    m = to_group_norm(small_effnet(), 8)
    fuse_pointwise(m)
    m._dropout.p = 0.0
    m.eval()
    g, w = step(m, "cuda", torch.bfloat16, 8)
    assert torch.isfinite(g).all() and torch.isfinite(w).all()
    cos = torch.nn.functional.cosine_similarity(g, ref, dim=0)
    assert cos > 0.95, float(cos)       # the same direction: bf16 through 80 layers


def randomised(model, seed=0):
    """Statistics and affine parameters as after some training."""
    g = torch.Generator().manual_seed(seed)
    for m in model.modules():
        if isinstance(m, nn.BatchNorm2d):
            m.running_mean.copy_(0.2 * torch.randn(m.num_features, generator=g))
            m.running_var.copy_(0.5 + torch.rand(m.num_features, generator=g))
            with torch.no_grad():
                m.weight.copy_(1 + 0.1 * torch.randn(m.num_features, generator=g))
                m.bias.copy_(0.1 * torch.randn(m.num_features, generator=g))
    return model.eval()


MODELS = [lambda: ResNet("cifar10", 29, 10, bottleneck=True), lambda: ResNet("imagenet", 50, 10, bottleneck=True),
          lambda: PyramidNet("cifar10", depth=29, alpha=30, num_classes=10, bottleneck=True), small_effnet]


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("make", MODELS)
def test_folded_networks_answer_as_before(dev, make):
    torch.manual_seed(0)
    model = randomised(make()).to(dev).to(memory_format=torch.channels_last)
    x = torch.randn(3, 3, 32, 32).to(dev).contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        want = model(x)
        n = fold_for_inference(model)
        got = model(x)
    assert n > 0
    # fp32 through some 30 layers in another order of products
    assert (got - want).abs().max() <= 1e-3 * want.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("make", MODELS)
def test_folded_networks_in_bf16(make):
    """bf16 under autocast is off by its own rounding; folding rounds less often and is off by no more than twice that."""
    torch.manual_seed(0)
    model = randomised(make()).cuda().to(memory_format=torch.channels_last)
    x = torch.randn(16, 3, 32, 32).cuda().contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        exact = model(x)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            before = model(x).float()
            fold_for_inference(model, torch.bfloat16)
            after = model(x).float()
    assert (after - exact).norm() <= 2 * (before - exact).norm() + 1e-3 * exact.norm()


def test_a_model_in_training_is_not_folded():
    with pytest.raises(ValueError):
        fold_for_inference(ResNet("cifar10", 29, 10, bottleneck=True))
    m = to_group_norm(ResNet("cifar10", 29, 10, bottleneck=True)).eval()
    assert fold_for_inference(m) == 0       # group norm is no affine map


@pytest.mark.parametrize("dev", DEV)
@pytest.mark.parametrize("bits", [32, 8])
def test_the_trainer_trains_and_resumes_with_adamw(dev, bits, tmp_path):
    os.environ["FAA_SYNTH_TRAIN"], os.environ["FAA_SYNTH_TEST"] = "64", "32"
    from fast_autoaugment_amd.data import api as data_api
    from fast_autoaugment_amd.engine import train_and_eval
    try:
        if dev == "cpu" and torch.cuda.is_available():
            pytest.skip("the trainer takes the GPU where there is one")
        data_api._STORE_CACHE.clear()
        conf = {
            "model": {"type": "wresnet40_2", "norm": "group"}, "dataset": "cifar10", "aug": "default", "cutout": 0,
            "batch": 32, "epoch": 1, "lr": 0.001,
            "lr_schedule": {"type": "cosine", "warmup": {"multiplier": 1, "epoch": 0}},
            "optimizer": {"type": "adamw", "decay": 0.05, "clip": 5, "state_bits": bits, "ema": 0},
        }
        C.replace(conf)
        path = str(tmp_path / "m.pth")
        r = train_and_eval("", "./data", save_path=path, evaluation_interval=1)
        assert r["epoch"] == 1
        saved = torch.load(path, weights_only=True)
        assert saved["optimizer"]["step"] == 2 and saved["optimizer"]["state_bits"] == bits
        C.replace({**conf, "epoch": 2})
        data_api._STORE_CACHE.clear()
        r = train_and_eval("", "./data", save_path=path, evaluation_interval=1)
        # as the trainer resumes: the epoch of the checkpoint is run again, with the optimizer's state behind it
        assert torch.load(path, weights_only=True)["optimizer"]["step"] == 6
    finally:
        os.environ.pop("FAA_SYNTH_TRAIN", None)
        os.environ.pop("FAA_SYNTH_TEST", None)
        data_api._STORE_CACHE.clear()


def test_the_search_scores_a_folded_child(tmp_path):
    """The density-matching score of a folded bottleneck child is that of the child."""
    os.environ["FAA_SYNTH_TRAIN"], os.environ["FAA_SYNTH_TEST"] = "200", "40"
    from fast_autoaugment_amd.data import api as data_api
    from fast_autoaugment_amd.search import density_match
    try:
        data_api._STORE_CACHE.clear()
        density_match._MODEL_CACHE.clear()
        conf = {"model": {"type": "pyramid", "depth": 29, "alpha": 12, "bottleneck": True}, "dataset": "cifar10",
                "aug": "default", "cutout": 0, "batch": 32, "epoch": 1, "lr": 0.1}
        torch.manual_seed(0)
        path = str(tmp_path / "child.pth")
        torch.save({"model": randomised(build_model(conf["model"], 10)).state_dict()}, path)
        augment = {"cv_ratio_test": 0.4, "cv_fold": 0, "save_path": path, "dataroot": "./data", "num_policy": 1, "num_op": 1,
                   "policy_0_0": 2, "prob_0_0": 0.0, "level_0_0": 0.5}
        scores = [density_match.eval_tta({**conf, "fold_inference": fold}, dict(augment)) for fold in (False, True)]
        assert abs(scores[0]["minus_loss"] - scores[1]["minus_loss"]) <= 1e-2 * abs(scores[0]["minus_loss"]) + 1e-3
    finally:
        os.environ.pop("FAA_SYNTH_TRAIN", None)
        os.environ.pop("FAA_SYNTH_TEST", None)
        data_api._STORE_CACHE.clear()
        density_match._MODEL_CACHE.clear()


def test_a_child_of_another_norm_is_not_the_cached_one(tmp_path):
    """Group norms of other group counts load the same checkpoint, but are other networks."""
    from fast_autoaugment_amd.search.density_match import _cached_model
    path = str(tmp_path / "child.pth")
    torch.save(build_model({"type": "wresnet40_2", "norm": "group"}, 10).state_dict(), path)
    groups = set()
    for n in (8, 4):
        conf = C()
        conf["model"] = {"type": "wresnet40_2", "norm": "group", "norm_groups": n}
        model = _cached_model(conf, 10, path, "cpu")
        groups.add(max(m.num_groups for m in model.modules() if isinstance(m, torch.nn.GroupNorm)))
    assert groups == {8, 4}


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", [{"type": "sgd", "decay": 0.0}, {"type": "rmsprop", "decay": 0.0},
                                       {"type": "adamw", "decay": 0.05}, {"type": "adamw", "decay": 0.05, "state_bits": 8}])
@pytest.mark.parametrize("loaded", ["average", "bare checkpoint"])
def test_the_trainer_steps_from_weights_that_were_loaded(optimizer, loaded, tmp_path, monkeypatch):
    """An average that is copied into the model at an epoch's end, or a checkpoint of weights alone, is what the fp32
    weights of the next epoch start from: those round to the model's, and the model's are what was loaded."""
    monkeypatch.setenv("FAA_SYNTH_TRAIN", "64")
    monkeypatch.setenv("FAA_SYNTH_TEST", "32")
    from fast_autoaugment_amd.data import api as data_api
    from fast_autoaugment_amd.engine import trainer
    starts, run_epoch = [], trainer.run_epoch

    def watched(model, loader, loss_fn, opt, *args, **kwargs):
        if opt is not None:
            flat = opt.flat
            starts.append(({k: v.detach().clone() for k, v in model.state_dict().items()},
                           torch.equal(flat.flat_master.bfloat16(), flat.flat_param)))
        return run_epoch(model, loader, loss_fn, opt, *args, **kwargs)

    monkeypatch.setattr(trainer, "run_epoch", watched)
    averages, ema = [], trainer.EMA
    monkeypatch.setattr(ema, "state_dict", lambda self: averages.append({k: v.clone() for k, v in self.shadow.items()})
                        or {k: v.clone() for k, v in self.shadow.items()})
    conf = {
        "model": {"type": "wresnet40_2", "norm": "group"}, "dataset": "cifar10", "aug": "default", "cutout": 0,
        "batch": 32, "epoch": 2, "lr": 0.05, "lr_schedule": {"type": "cosine", "warmup": {"multiplier": 1, "epoch": 0}},
        "optimizer": {**optimizer, "clip": 5, "ema": 0.5 if loaded == "average" else 0, "ema_interval": 1},
    }
    path = None
    if loaded != "average":
        path = str(tmp_path / "weights.pth")
        torch.manual_seed(123)
        averages = [{k: v.float() for k, v in build_model(conf["model"], 10).state_dict().items()}]
        torch.save(averages[0], path)
    try:
        data_api._STORE_CACHE.clear()
        C.replace(conf)
        trainer.train_and_eval("", "./data", save_path=path, evaluation_interval=5)
    finally:
        data_api._STORE_CACHE.clear()
    weights, rounded = starts[1 if loaded == "average" else 0]
    assert rounded
    for k, v in averages[0].items():
        assert torch.equal(weights[k].float().cpu(), v.to(weights[k].dtype).float().cpu())


@pytest.mark.parametrize("call,after", [("bn_relu", torch.relu), ("bn_only", lambda t: t), ("bn_swish", nn.functional.silu)])
def test_group_norms_in_fp64_run_as_torch_s(call, after):
    from fast_autoaugment_amd.ops import modules
    torch.manual_seed(0)
    gn, x = nn.GroupNorm(2, 8).double(), torch.randn(2, 8, 5, 5, dtype=torch.float64)
    with torch.no_grad():
        gn.weight.normal_()
        gn.bias.normal_()
    assert torch.equal(getattr(modules, call)(x, gn), after(gn(x)))


@pytest.mark.parametrize("make", [lambda: build_model({"type": "wresnet40_2", "norm": "group"}, 7),
                                  lambda: build_model({"type": "efficientnet-b0", "norm": "group"}, 7)])
def test_group_models_answer_in_fp64(make):
    """What a model gives in 64 bits is what it gives in 32, to the roundings of some forty or eighty layers."""
    torch.manual_seed(0)
    model = make().eval()
    x = torch.randn(2, 3, 32, 32)
    with torch.no_grad():
        low, full = model(x), model.double()(x.double())
    assert full.dtype == torch.float64
    assert (low - full).abs().max() <= 1e-4 * full.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_from_the_same_gradients_are_the_cpu_s(dtype, bits):
    """Both devices are given the CPU's gradients of a batch: weights then differ by an update's own roundings (about 32
    of it, below 2 lr in size here) and by those of the weight and its decay, step by step."""
    flats, opts, lr = [], [], 1e-3
    for dev in ("cpu", "cuda"):
        torch.manual_seed(0)
        model = build_model({"type": "wresnet40_2", "norm": "group"}, 7).to(dev)
        flats.append(flatten_module(model, align=256, work_dtype=dtype))
        opts.append(FusedAdamW(flats[-1], lr=lr, weight_decay=0.05, state_bits=bits))
    torch.manual_seed(0)
    source = build_model({"type": "wresnet40_2", "norm": "group"}, 7)
    grads = flatten_module(source, align=256)
    g = torch.Generator().manual_seed(1)
    weights = lambda f: (f.flat_param if f.flat_master is None else f.flat_master).cpu()  # noqa: E731
    for done in range(1, 4):
        nn.functional.cross_entropy(source(torch.randn(4, 3, 32, 32, generator=g)), torch.arange(4)).backward()
        for f, opt in zip(flats, opts):
            before = weights(f).clone()
            f.flat_grad.copy_(grads.flat_grad)
            opt.step()
        a, b = (weights(f) for f in flats)
        assert ((a - b).abs() <= done * (4 * 2.0 ** -24 * a.abs() + 2 * lr * 32 * 2.0 ** -24)).all()
        assert (a - before).abs().max() > lr / 2
        for name in opts[0]._names:
            x, y = (getattr(o, name).cpu() for o in opts)
            assert torch.equal(x.float(), y.float()), name


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    """Calls that run beside each other have workspaces of their own: chunks, joins, split and small products."""
    from fast_autoaugment_amd.ops.groupnorm import group_norm_act
    from fast_autoaugment_amd.ops.pointwise import linear_act
    g = torch.Generator("cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731

    def norm(x, w, b, dy):
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        y = group_norm_act(x, 4, w, b, act="swish")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    def product(x, w, b, dy):
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        y = linear_act(x, w, b, act="swish")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    cases = [(norm, [r(4, 16, 130, 130), r(16), r(16), r(4, 16, 130, 130)]), (norm, [r(9, 64, 14, 14), r(64), r(64), r(9, 64, 14, 14)]),
             (product, [r(20000, 64), r(96, 64), r(96), r(20000, 96)]), (product, [r(131, 4000), r(72, 4000), r(72), r(131, 72)]),
             (product, [r(3001, 61), r(35, 61), r(35), r(3001, 35)])]
    alone = [f(*args) for f, args in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(20):
        torch.cuda.synchronize()
        out = []
        for s, k in zip(streams, (i % 5, (i // 5 + i + 1) % 5)):
            with torch.cuda.stream(s):
                out.append((k, cases[k][0](*cases[k][1])))
        torch.cuda.synchronize()
        for k, got in out:
            for a, b in zip(got, alone[k]):
                assert torch.equal(a, b)
