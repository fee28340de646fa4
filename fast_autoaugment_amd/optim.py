"""Optimizers: TF-semantics RMSprop + the fused flat-buffer SGD step.

RMSpropTF reproduces the reference tf_port/rmsprop.py semantics exactly:
``ms`` initialized to ONES (not zeros) and epsilon added INSIDE the sqrt
(rmsprop.py:80,93,97) — both differ from torch.optim.RMSprop.

FusedSGD is the MI355X-native training step: parameters live as views into
one flat fp32 buffer ordered [decay-params | no-decay-params] (see
parallel.flat), and one step = three HIP kernels over contiguous memory:
  1. wd_add:    g += wd * p on the decay segment (manual non-BN weight decay,
                reference train.py:40,61 — the WD term participates in the
                clip norm because the reference adds it to the loss)
  2. l2norm:    ||g||^2 of the whole flat grad -> 1-elem device tensor
  3. sgd_step:  clip coef read on-device, nesterov momentum update
No host sync anywhere, so the whole step is hipGraph-capturable.

FusedAdamW is AdamW (decoupled decay) over the same flat buffers or over any
list of tensors, with its two moments in 32 or in 8 bits: one launch for all
tensors, one more for the step's scalars and one for the norm if it clips.
"""
from __future__ import annotations

import math
import operator
import struct

import torch
from torch.optim.optimizer import Optimizer


class RMSpropTF(Optimizer):
    def __init__(self, params, lr=1e-2, alpha=0.99, eps=1e-8, momentum=0.0,
                 weight_decay=0.0):
        if momentum <= 0.0:
            raise ValueError("RMSpropTF requires momentum > 0")
        defaults = dict(lr=lr, momentum=momentum, alpha=alpha, eps=eps,
                        weight_decay=weight_decay)
        super().__init__(params, defaults)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                grad = p.grad
                state = self.state[p]
                if len(state) == 0:
                    state["step"] = 0
                    state["ms"] = torch.ones_like(p)     # TF init
                    state["mom"] = torch.zeros_like(p)
                if group["weight_decay"] > 0:
                    grad = grad.add(p, alpha=group["weight_decay"])
                rho = group["alpha"]
                ms, mom = state["ms"], state["mom"]
                state["step"] += 1
                ms.add_((grad * grad - ms) * (1.0 - rho))
                # eps inside sqrt (TF): lr * g / sqrt(ms + eps)
                mom.mul_(group["momentum"]).addcdiv_(grad, (ms + group["eps"]).sqrt(),
                                                     value=group["lr"])
                p.add_(mom, alpha=-1.0)
        return loss


class FusedSGD:
    """Flat-buffer nesterov SGD with fused manual-WD + global grad clip.

    Operates on a parallel.flat.FlatParams object. Matches the reference
    update chain: loss += wd/2*sum(p^2) over non-BN params (train.py:61),
    clip_grad_norm_(all params, clip) (train.py:63-65), then
    optim.SGD(momentum, nesterov, weight_decay=0).step().
    """

    def __init__(self, flat, lr: float, momentum: float = 0.9, nesterov: bool = True,
                 weight_decay: float = 0.0, grad_clip: float = 5.0):
        self.flat = flat
        self.lr = lr
        self.momentum = momentum
        self.nesterov = nesterov
        self.weight_decay = weight_decay
        self.grad_clip = grad_clip
        base = flat.flat_master if flat.flat_master is not None else flat.flat_param
        self.momentum_buf = torch.zeros_like(base)
        self._normsq = torch.zeros(1, device=flat.flat_param.device, dtype=torch.float32)
        # lr lives on-device so the step kernels are hipGraph-replayable;
        # the host writes it through a pinned staging scalar before replay
        dev = flat.flat_param.device
        self._lr_t = torch.full((1,), lr, device=dev, dtype=torch.float32)
        self._lr_host = (torch.zeros(1, dtype=torch.float32, pin_memory=True)
                         if dev.type == "cuda" else torch.zeros(1))
        self._last_lr = lr
        # mirror of torch.optim param_groups API surface used by the trainer
        self.param_groups = [{"lr": lr}]

    def sync_lr(self):
        """Push param_groups[0]['lr'] to the device scalar (call pre-replay)."""
        lr = self.param_groups[0]["lr"]
        if lr != self._last_lr:
            self._lr_host[0] = lr
            self._lr_t.copy_(self._lr_host, non_blocking=True)
            self._last_lr = lr

    def zero_grad(self, set_to_none: bool = False):
        self.flat.flat_grad.zero_()

    @torch.no_grad()
    def step(self):
        self.lr = self.param_groups[0]["lr"]
        p = self.flat.flat_param
        g = self.flat.flat_grad
        nd = self.flat.n_decay
        master = self.flat.flat_master
        if p.is_cuda:
            from .ops import ext
            C = ext()
            self.sync_lr()
            if master is not None:
                C.sgd_fused_step_mixed(master, p, g, self.momentum_buf, self._normsq,
                                       self._lr_t, nd, self.weight_decay,
                                       self.grad_clip, self.momentum,
                                       1 if self.nesterov else 0)
            else:
                C.sgd_fused_step(p, g, self.momentum_buf, self._normsq, self._lr_t, nd,
                                 self.weight_decay, self.grad_clip,
                                 self.momentum, 1 if self.nesterov else 0)
            return
        # CPU reference path (also defines the mixed-kernel semantics)
        pm = master if master is not None else p
        gf = g.float()
        if self.weight_decay > 0 and nd > 0:
            gf[:nd].add_(pm[:nd].float(), alpha=self.weight_decay)
        if self.grad_clip > 0:
            total = gf.norm(2)
            coef = min(1.0, self.grad_clip / (float(total) + 1e-6))
            if coef < 1.0:
                gf.mul_(coef)
        buf = self.momentum_buf
        buf.mul_(self.momentum).add_(gf)
        upd = gf.add(buf, alpha=self.momentum) if self.nesterov else buf
        pm.add_(upd.to(pm.dtype), alpha=-self.lr)
        if master is not None:
            p.copy_(master.to(p.dtype))

    def state_dict(self):
        return {"momentum_buf": self.momentum_buf, "lr": self.lr,
                "momentum": self.momentum, "nesterov": self.nesterov,
                "weight_decay": self.weight_decay, "grad_clip": self.grad_clip}

    def load_state_dict(self, sd):
        self.momentum_buf.copy_(sd["momentum_buf"])
        self.lr = sd.get("lr", self.lr)
        self.param_groups[0]["lr"] = self.lr


def build_optimizer(conf_opt, model_params, lr: float):
    """Per-parameter (non-flat) optimizer factory for the generic trainer path.

    conf_opt: the conf['optimizer'] dict. Weight decay is handled manually
    by the trainer (added to the loss), so decay here is 0 — matching the
    reference train.py:139-156.
    """
    typ = conf_opt["type"]
    if typ == "sgd":
        return torch.optim.SGD(model_params, lr=lr,
                               momentum=conf_opt.get("momentum", 0.9),
                               weight_decay=0.0,
                               nesterov=conf_opt.get("nesterov", True))
    if typ == "rmsprop":
        return RMSpropTF(model_params, lr=lr, weight_decay=0.0,
                         alpha=0.9, momentum=0.9, eps=0.001)
    if typ == "adamw":
        return build_adamw(conf_opt, model_params, lr)
    raise ValueError(f"invalid optimizer type={typ}")


def build_adamw(conf_opt, params, lr: float):
    """FusedAdamW from a conf['optimizer'] dict: decay (decoupled), betas, eps, clip and state_bits (8 or 32)."""
    return FusedAdamW(params, lr=lr, betas=tuple(conf_opt.get("betas", (0.9, 0.999))),
                      eps=float(conf_opt.get("eps", 1e-8)), weight_decay=conf_opt.get("decay", 0.0),
                      grad_clip=conf_opt.get("clip", 5.0), state_bits=conf_opt.get("state_bits", 32))


class FusedRMSpropTF:
    """Flat-buffer TF-semantics RMSprop (reference tf_port/rmsprop.py) on
    bf16 working weights + fp32 master, with manual non-BN WD and optional
    global clip — the EfficientNet training step as 1-2 HIP kernels."""

    def __init__(self, flat, lr: float, alpha: float = 0.9, momentum: float = 0.9,
                 eps: float = 1e-3, weight_decay: float = 0.0, grad_clip: float = 0.0):
        assert flat.flat_master is not None, "FusedRMSpropTF needs bf16 flat mode"
        self.flat = flat
        self.lr = lr
        self.alpha = alpha
        self.momentum = momentum
        self.eps = eps
        self.weight_decay = weight_decay
        self.grad_clip = grad_clip
        dev = flat.flat_param.device
        self.ms = torch.ones_like(flat.flat_master)      # TF init (rmsprop.py:80)
        self.mom = torch.zeros_like(flat.flat_master)
        self._normsq = torch.zeros(1, device=dev, dtype=torch.float32)
        self._lr_t = torch.full((1,), lr, device=dev, dtype=torch.float32)
        self._lr_host = (torch.zeros(1, dtype=torch.float32, pin_memory=True)
                         if dev.type == "cuda" else torch.zeros(1))
        self._last_lr = lr
        self.param_groups = [{"lr": lr}]

    def sync_lr(self):
        lr = self.param_groups[0]["lr"]
        if lr != self._last_lr:
            self._lr_host[0] = lr
            self._lr_t.copy_(self._lr_host, non_blocking=True)
            self._last_lr = lr

    def zero_grad(self, set_to_none: bool = False):
        self.flat.flat_grad.zero_()

    @torch.no_grad()
    def step(self):
        self.lr = self.param_groups[0]["lr"]
        master = self.flat.flat_master
        g = self.flat.flat_grad
        nd = self.flat.n_decay
        if master.is_cuda:
            from .ops import ext
            self.sync_lr()
            ext().rmsprop_fused_step_mixed(master, self.flat.flat_param, g,
                                           self.ms, self.mom, self._normsq,
                                           self._lr_t, nd, self.weight_decay,
                                           self.grad_clip, self.alpha,
                                           self.momentum, self.eps)
            return
        # CPU reference path (defines the kernel's semantics)
        gf = g.float()
        if self.weight_decay > 0 and nd > 0:
            gf[:nd].add_(master[:nd], alpha=self.weight_decay)
        if self.grad_clip > 0:
            coef = min(1.0, self.grad_clip / (float(gf.norm(2)) + 1e-6))
            if coef < 1.0:
                gf.mul_(coef)
        self.ms.add_((gf * gf - self.ms) * (1.0 - self.alpha))
        self.mom.mul_(self.momentum).addcdiv_(gf, (self.ms + self.eps).sqrt(),
                                              value=self.lr)
        master.add_(self.mom, alpha=-1.0)
        self.flat.flat_param.copy_(master.to(self.flat.flat_param.dtype))

    def state_dict(self):
        return {"ms": self.ms, "mom": self.mom, "lr": self.lr}

    def load_state_dict(self, sd):
        self.ms.copy_(sd["ms"])
        self.mom.copy_(sd["mom"])


class FusedAdamW:
    """AdamW over all tensors of a model at once, moments in 32 or 8 bits.

        g' = g * min(1, grad_clip / (||g|| + 1e-6))      (grad_clip > 0; norm over all tensors)
        m  = b1 m + (1-b1) g'        v = b2 v + (1-b2) g'^2
        p  = p (1 - lr wd) - lr (m / (1-b1^t)) / (sqrt(v / (1-b2^t)) + eps)

    ``params`` is a ``parallel.flat.FlatParams`` (its decay segment decays, the
    rest does not), an iterable of parameters, or a list of
    ``{"params": [...], "weight_decay": w}`` groups. Parameters are contiguous,
    fp32, bf16 or fp16, and all on one device; bf16 and fp16 ones get fp32
    weights that the optimizer keeps (FlatParams brings its own), which are
    updated and rounded back into the parameters. Such a parameter that was
    written since the last step (a checkpoint that was loaded), or a flat buffer
    or one of its parameters, is taken over where it is not its fp32 weight
    rounded; a write through ``p.data`` is not seen. A parameter whose ``grad`` is None is left as it is. The step count is one for all parameters.

    ``state_bits=8`` holds m and sqrt(v) as e4m3 numbers (``exp_avg``,
    ``exp_avg_root``) with one fp32 scale for every 256 neighbours of a tensor
    (``*_scale``); the step uses the moments before they are rounded. A flat
    buffer then has to start each tensor at a multiple of 256
    (``flatten_module(align=256)``). A NaN stays in its element; an infinite
    moment makes its block of 256 NaN from the next step on.

    The step count and the learning rate are on the device: a captured step
    replays, with ``sync_lr()`` before a replay pushing a changed rate. Under
    capture the gradients have to be where an eager step saw them. Weights that
    were written between replays are not seen by these: an eager step comes first.
    """

    BLOCK = 256         # elements under one scale
    CHUNK = 4096        # elements a workgroup takes
    _NORM_PARTS = 1024
    _KINDS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.0, grad_clip: float = 0.0, state_bits: int = 32):
        b1, b2 = (float(b) for b in betas)
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"FusedAdamW: betas={betas} have to lie in [0, 1)")
        if not (eps > 0.0 and lr >= 0.0 and weight_decay >= 0.0 and grad_clip >= 0.0):
            raise ValueError("FusedAdamW: eps > 0 and lr, weight_decay, grad_clip >= 0 are needed")
        if state_bits not in (8, 32):
            raise ValueError(f"FusedAdamW: state_bits={state_bits} is neither 8 nor 32")
        self.betas, self.eps = (b1, b2), float(eps)
        self.weight_decay, self.grad_clip, self.state_bits = float(weight_decay), float(grad_clip), state_bits
        self.flat = params if hasattr(params, "flat_param") else None
        if self.flat is not None:
            total = self._init_flat()
        else:
            total = self._init_list(params)
        self.lr = lr
        self.param_groups = [{"lr": lr}]
        self._last_lr = lr
        dev = self._dev
        zeros = lambda n, t: torch.zeros(n, dtype=t, device=dev)  # noqa: E731
        if state_bits == 32:
            self.exp_avg, self.exp_avg_sq = zeros(total, torch.float32), zeros(total, torch.float32)
            self._names = ("exp_avg", "exp_avg_sq")
        else:
            total = -(-total // self.BLOCK) * self.BLOCK
            self.exp_avg, self.exp_avg_root = (
                zeros(total, torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
            self.exp_avg_scale = zeros(total // self.BLOCK, torch.float32)
            self.exp_avg_root_scale = zeros(total // self.BLOCK, torch.float32)
            self._names = ("exp_avg", "exp_avg_scale", "exp_avg_root", "exp_avg_root_scale")
        self.step_count = zeros(1, torch.int64)
        self._lr_t = torch.full((1,), lr, device=dev, dtype=torch.float32)
        self._scal = zeros(3, torch.float32)
        self._part = zeros(self._NORM_PARTS * 3, torch.float64)
        self._seen = None       # addresses that the tables on the device were made for
        self._tables = None
        self._captured = []

    # ---- what there is to update: (weights fp32, low-precision copy, gradient's owner, offset, n, decay)

    def _init_flat(self):
        f = self.flat
        n, nd = f.flat_param.numel(), f.n_decay
        if f.flat_param.dtype not in self._KINDS or f.flat_grad.dtype != f.flat_param.dtype:
            raise TypeError("FusedAdamW: flat buffers are fp32, bf16 or fp16, weights and gradients alike")
        if f.flat_param.dtype != torch.float32 and f.flat_master is None:
            raise ValueError("FusedAdamW: low-precision flat weights need flat_master")
        if self.state_bits == 8 and (nd % self.BLOCK or any(
                (p.data_ptr() - f.flat_param.data_ptr()) // f.flat_param.element_size() % self.BLOCK
                for p in f.params)):
            raise ValueError("FusedAdamW: 8-bit moments need tensors that start at multiples of "
                             "256 in the flat buffer: flatten_module(align=256)")
        self._dev = f.flat_param.device
        self._items = [(0, nd, self.weight_decay), (nd, n - nd, 0.0)]
        self._flat_stamp = None
        self._counted = [p for p in f.params if not p.is_inference()]
        return n

    def _init_list(self, params):
        groups = list(params)
        if not groups:
            raise ValueError("FusedAdamW: no parameters")
        if not isinstance(groups[0], dict):
            groups = [{"params": groups}]
        self.params, self._items, total, seen = [], [], 0, set()
        for g in groups:
            odd = set(g) - {"params", "weight_decay"}
            if odd:
                raise ValueError(f"FusedAdamW: a group holds params and weight_decay, not {sorted(odd)}")
            wd = float(g.get("weight_decay", self.weight_decay))
            if not wd >= 0.0:
                raise ValueError("FusedAdamW: weight_decay >= 0 is needed")
            ps = [g["params"]] if isinstance(g["params"], torch.Tensor) else list(g["params"])
            for p in ps:
                if p.dtype not in self._KINDS:
                    raise TypeError(f"FusedAdamW: a parameter of {p.dtype}: fp32, bf16 and fp16 are stepped")
                if id(p) in seen:
                    raise ValueError("FusedAdamW: a parameter is listed twice")
                seen.add(id(p))
                self.params.append(p)
                self._items.append((total, p.numel(), wd))
                total += -(-p.numel() // self.BLOCK) * self.BLOCK
        if not self.params:
            raise ValueError("FusedAdamW: no parameters")
        self._dev = self.params[0].device
        if any(p.device != self._dev for p in self.params):
            raise ValueError("FusedAdamW: the parameters are on several devices")
        self.masters = [None if p.dtype == torch.float32 else p.detach().float() for p in self.params]
        self._stamps = [self._stamp(p) for p in self.params]
        return total

    @staticmethod
    def _stamp(p):
        """What changes when a tensor is written by torch or put elsewhere."""
        return p.data_ptr(), 0 if p.is_inference() else p._version

    def _take_over_flat(self):
        """Weights that were written into low-precision flat buffers since the last step go to the fp32 ones."""
        f = self.flat
        if f.flat_param.dtype == torch.float32:
            return
        # a parameter of the buffer counts its own writes
        stamp = (*self._stamp(f.flat_param), sum(map(operator.attrgetter("_version"), self._counted)))
        if stamp == self._flat_stamp:
            return
        if self._dev.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW: the flat weights were written since the last eager step: step once before capture")
        full, low = f.flat_master, f.flat_param
        full.copy_(torch.where(full.to(low.dtype) == low, full, low.float()))
        self._flat_stamp = stamp

    @staticmethod
    def _same_order(a, b):
        """Whether two tensors of one shape lie in memory in the same order, without gaps."""
        return (a.is_contiguous() and b.is_contiguous()) or (
            a.stride() == b.stride() and a.dim() == 4 and a.is_contiguous(memory_format=torch.channels_last))

    def _views(self):
        """(type, fp32 weights, low-precision copy or None, gradient or None, offset, n, decay) of every tensor."""
        if self.flat is not None:
            f = self.flat
            low = f.flat_param if f.flat_param.dtype != torch.float32 else None
            full = f.flat_param if low is None else f.flat_master
            return [(f.flat_param.dtype, full[off:off + n], None if low is None else low[off:off + n],
                     f.flat_grad[off:off + n], off, n, wd) for off, n, wd in self._items if n > 0]
        views = []
        for i, (p, master, (off, n, wd)) in enumerate(zip(self.params, self.masters, self._items)):
            if n == 0:
                continue
            w, low = (p.detach(), None) if master is None else (master, p.detach())
            if (p.numel() != n or p.device != self._dev or (p.dtype == torch.float32) != (low is None)
                    or not self._same_order(p, w)):
                raise ValueError("FusedAdamW: a parameter is not contiguous, or changed its size, type, device or order")
            if low is not None and self._stamp(p) != self._stamps[i]:
                w.copy_(torch.where(w.to(low.dtype) == low, w, low.float()))
                self._stamps[i] = self._stamp(p)
            g = p.grad
            if g is not None:
                if g.layout != torch.strided or g.dtype != p.dtype or g.device != self._dev or g.shape != p.shape:
                    raise TypeError("FusedAdamW: a gradient is sparse, or of another type, shape or device than its parameter")
                if not self._same_order(g, p):
                    p.grad = g = torch.empty_like(p).copy_(g)
            views.append((p.dtype, w, low, g, off, n, wd))
        return views

    def _addresses(self):
        """What the device tables depend on: every tensor's place and memory order."""
        if self.flat is not None:
            f = self.flat
            return (f.flat_param.data_ptr(), f.flat_grad.data_ptr(),
                    0 if f.flat_master is None else f.flat_master.data_ptr())
        from .ops import ext
        return ext().tensor_addresses(self.params)

    def _refresh_tables(self):
        """The device tables of addresses, made anew where an address changed."""
        capturing = torch.cuda.is_current_stream_capturing()
        if self._addresses() == self._seen:
            if capturing and not any(t is self._tables for t in self._captured):
                self._captured.append(self._tables)     # a graph reads them as long as it is replayed
            return self._tables
        if capturing:
            raise RuntimeError("FusedAdamW: the gradients' addresses changed since the last eager step, or parameters "
                               "were written: keep gradients in place (zero_grad() fills them) and step once before capture")
        by = {}
        for kind, w, low, g, off, n, wd in self._views():
            rows, lengths = by.setdefault(self._KINDS[kind], ([], []))
            pw, pl, pg = (0 if t is None else t.data_ptr() for t in (w, low, g))
            esize = kind.itemsize
            aligned = pw % 16 == 0 and off % 4 == 0 and pl % (4 * esize) == 0 and pg % (4 * esize) == 0
            bits = struct.unpack("<I", struct.pack("<f", wd))[0]
            rows.append((pw, pl, pg, off, n, bits | (int(aligned) << 32)))
            lengths.append(-(-n // self.CHUNK))

        def chunk_table(lengths):
            """(row, chunk in the row) of every workgroup."""
            count = torch.tensor(lengths)
            row = torch.repeat_interleave(torch.arange(len(lengths)), count)
            first = torch.cumsum(count, 0) - count
            return torch.stack([row, torch.arange(row.numel()) - first[row]], 1).to(torch.int32)

        up = lambda t: t.contiguous().pin_memory().to(self._dev, non_blocking=True)  # noqa: E731
        rows = [up(torch.tensor(r, dtype=torch.int64).view(-1, 6)) for r, _ in by.values()]
        chunks = [up(chunk_table(n)) for _, n in by.values()]
        self._tables = (rows, chunks, list(by))
        self._seen = self._addresses()
        return self._tables

    def sync_lr(self):
        """Push param_groups[0]['lr'] to the device scalar (call pre-replay)."""
        lr = self.param_groups[0]["lr"]
        if lr != self._last_lr:
            self._lr_t.fill_(lr)
            self._last_lr = lr

    def zero_grad(self, set_to_none: bool = False):
        if self.flat is not None:
            self.flat.flat_grad.zero_()
        elif set_to_none:
            for p in self.params:
                p.grad = None
        else:
            grads = [p.grad for p in self.params if p.grad is not None]
            if grads:
                torch._foreach_zero_(grads)

    @torch.no_grad()
    def step(self):
        self.lr = self.param_groups[0]["lr"]
        if self.flat is not None:
            self._take_over_flat()
        if self._dev.type != "cuda":
            return self._step_cpu()
        from .ops import ext
        if not torch.cuda.is_current_stream_capturing():
            self.sync_lr()
        rows, chunks, kinds = self._refresh_tables()
        m = self.exp_avg
        r = self.exp_avg_sq if self.state_bits == 32 else self.exp_avg_root
        ms = self._scal if self.state_bits == 32 else self.exp_avg_scale
        rs = self._scal if self.state_bits == 32 else self.exp_avg_root_scale
        ext().adamw_step(rows, chunks, kinds, m, r, ms, rs, self.step_count, self._scal,
                         self._part, self._lr_t, self.betas[0], self.betas[1], self.eps,
                         self.grad_clip)

    # ---- CPU reference path (defines the kernels' semantics: they round each of these operations alike)

    def _moment(self, name, off, n):
        if self.state_bits == 32:
            return getattr(self, name)[off:off + n].clone()
        lo, hi = off // self.BLOCK, -(-(off + n) // self.BLOCK)
        held = getattr(self, name)[lo * self.BLOCK:hi * self.BLOCK].float().view(-1, self.BLOCK)
        return (held * getattr(self, name + "_scale")[lo:hi, None]).view(-1)[:n]

    def _hold(self, name, off, n, value, least):
        if self.state_bits == 32:
            getattr(self, name)[off:off + n] = value
            return
        lo, hi = off // self.BLOCK, -(-(off + n) // self.BLOCK)
        v = torch.zeros((hi - lo) * self.BLOCK)
        v[:n] = value
        v = v.view(-1, self.BLOCK)
        finite = torch.nan_to_num(v.abs(), nan=0.0, posinf=math.inf)
        top = finite.amax(1, keepdim=True).clamp_min(2.0 ** -100)
        q = (v * (top.reciprocal() * 448.0)).to(torch.float8_e4m3fn)
        if least:
            q = torch.where((v > 0) & (q.float() == 0), torch.tensor(2.0 ** -9), q.float()).to(torch.float8_e4m3fn)
        getattr(self, name).view(torch.uint8)[lo * self.BLOCK:hi * self.BLOCK] = q.view(-1).view(torch.uint8)
        getattr(self, name + "_scale")[lo:hi] = (top * (1.0 / 448.0)).view(-1)

    def _step_cpu(self):
        (b1, b2), lr = self.betas, self.lr
        views = self._views()
        self.step_count += 1
        t = int(self.step_count)
        coef = torch.ones(())
        if self.grad_clip > 0:
            sq = sum(float(g.float().square().sum(dtype=torch.float64)) for _, _, _, g, *_ in views if g is not None)
            norm = torch.tensor(math.sqrt(sq) if sq == sq else math.nan)
            coef = ((norm + 1e-6).reciprocal() * self.grad_clip).clamp_max(1.0)
        second = "exp_avg_sq" if self.state_bits == 32 else "exp_avg_root"
        flat = lambda x: x.as_strided((x.numel(),), (1,))  # noqa: E731
        for _, w, low, g, off, n, wd in views:
            if g is None:
                continue
            gf = flat(g).float() * coef
            m = b1 * self._moment("exp_avg", off, n) + (1 - b1) * gf
            v = self._moment(second, off, n)
            v = b2 * (v if self.state_bits == 32 else v.square()) + ((1 - b2) * gf) * gf
            root = v.double().sqrt().float()       # torch's fp32 root on the CPU is off by a step at times
            wf = flat(w)
            wf.mul_(1 - lr * wd).sub_(lr * (m / (1 - b1 ** t)) / (root / math.sqrt(1 - b2 ** t) + self.eps))
            if low is not None:
                flat(low).copy_(wf)
            self._hold("exp_avg", off, n, m, False)
            self._hold(second, off, n, v if self.state_bits == 32 else root, True)
        if self.flat is None:
            self._stamps = [self._stamp(p) for p in self.params]
        elif self._flat_stamp is not None:
            self._flat_stamp = (*self._stamp(self.flat.flat_param), self._flat_stamp[-1])

    def state_dict(self):
        sd = {"step": int(self.step_count), "lr": self.lr, "state_bits": self.state_bits}
        sd.update({n: getattr(self, n) for n in self._names})
        if self.flat is None and any(m is not None for m in self.masters):
            sd["masters"] = self.masters
        elif self.flat is not None and self.flat.flat_param.dtype != torch.float32:
            sd["flat_master"] = self.flat.flat_master
        return sd

    @torch.no_grad()
    def load_state_dict(self, sd):
        if "exp_avg" not in sd or "step" not in sd:
            raise ValueError("FusedAdamW: this is not the state of a FusedAdamW")
        bits = 32 if "exp_avg_sq" in sd else 8
        if bits != self.state_bits:
            raise ValueError(f"FusedAdamW: the state is held in {bits} bits, this optimizer's in {self.state_bits}")
        for n in self._names:
            if sd[n].shape != getattr(self, n).shape or sd[n].dtype != getattr(self, n).dtype:
                raise ValueError(f"FusedAdamW: {n} has another shape or type than this optimizer's")
        low = self.flat is not None and self.flat.flat_param.dtype != torch.float32
        if low and "flat_master" in sd and sd["flat_master"].shape != self.flat.flat_master.shape:
            raise ValueError("FusedAdamW: flat_master has another shape than this optimizer's")
        for n in self._names:
            getattr(self, n).copy_(sd[n])
        if low and "flat_master" in sd:
            self.flat.flat_master.copy_(sd["flat_master"])
        if self.flat is None and "masters" in sd:
            for mine, theirs in zip(self.masters, sd["masters"]):
                if mine is not None:
                    mine.copy_(theirs)
        self.step_count.fill_(int(sd["step"]))
        self.lr = sd.get("lr", self.lr)
        self.param_groups[0]["lr"] = self.lr
