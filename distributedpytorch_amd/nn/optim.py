"""Fused arena optimizers: Adam(lr=1e-3) and SGD(lr=1e-3, momentum=0.9)+StepLR(1, 0.1) as selected by the reference
(/root/reference/classif.py:122-131,168-169).  One launch updates a contiguous arena range (the whole model, or one
DDP bucket so the update of bucket k overlaps the all-reduce of bucket k+1).  lr / step / 1/world live in a device
vector so a captured hipGraph stays valid when they change.  `state_dict()` reproduces torch.optim's layout
(per-parameter `step` 0-d fp32 tensor, `exp_avg`, `exp_avg_sq` / `momentum_buffer`) in torchvision's
OIHW layout so the reference's `optimizer.load_state_dict` accepts it.

"adamw" decouples the weight decay and applies it to matrices and filters only: biases and norm scales are a parameter group
of their own, without decay, and `state_dict()` has the layout of torch.optim.AdamW over those two groups (decayed parameters
first).  "adamw8" is the same with states of 8 bits (ops.adamw8_step): 2.125 bytes a parameter instead of 8.  It is saved as the
32-bit values its states stand for, with the scales as entries of the first parameter group; loading rounds to nearest,
which gives the same codes again.  A checkpoint of one kind loads into the other.
"""
from __future__ import annotations

import torch

from .. import ops
from .engine import ALIGN, ParamStore, pad_to

# hyper vector slots (csrc/hip/optim.hip)
LR, B1, B2, EPS, WD, STEP, MOM, GSCALE, OMB1, OMB2, B1LO, B2LO = range(12)


def make_hyper(lr, beta1, beta2, eps, weight_decay, step, momentum, grad_scale, device=None):
    """The 12-float hyper-parameter vector of the optimizer kernels.  Slots 8-11 carry what torch.optim keeps in Python
    doubles: float(1 - beta) for the moment increments and the low parts beta - float(beta), from which the kernel
    rebuilds the double betas for the bias corrections (csrc/hip/optim.hip)."""
    import struct

    def f32(x):
        return struct.unpack("f", struct.pack("f", x))[0]
    return torch.tensor([lr, beta1, beta2, eps, weight_decay, step, momentum, grad_scale, 1.0 - beta1, 1.0 - beta2,
                         beta1 - f32(beta1), beta2 - f32(beta2)], dtype=torch.float32, device=device)


class ArenaOptimizer:
    def __init__(self, store: ParamStore, kind="adam", lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=None,
                 momentum=0.9, grad_scale=1.0, seed=0):
        """weight_decay: 0.01 for "adamw" and "adamw8", 0 for the others where it is not given.  seed: of the stochastic rounding
        of 8-bit states; ranks that share a model must share it."""
        if kind not in ("adam", "SGD", "adamw", "adamw8"):
            raise ValueError(f"Invalid optimizer {kind!r}")
        self.store, self.kind = store, kind
        self.adamw = kind in ("adamw", "adamw8")
        if weight_decay is None:
            weight_decay = 0.01 if self.adamw else 0.0
        dev = store.device
        self.hyper = make_hyper(lr, betas[0], betas[1], eps, weight_decay, 0.0, momentum if kind == "SGD" else 0.0,
                                grad_scale, device=dev)
        self.m_scale = self.v_scale = self.groups = self.group_ids = None
        self.seed = int(seed) & 0xFFFFFFFF
        if kind == "adamw8":
            n = store.p.numel()
            self.m = torch.zeros(n, dtype=torch.float8_e4m3fn, device=dev)
            self.v = torch.zeros(n, dtype=torch.float8_e5m2, device=dev)
            self.m_scale, self.v_scale = torch.zeros(n // ALIGN, device=dev), torch.zeros(n // ALIGN, device=dev)
        else:
            self.m = torch.zeros_like(store.p)
            self.v = torch.zeros_like(store.p) if kind != "SGD" else None
        if self.adamw:
            ids = torch.zeros(store.p.numel() // ALIGN, dtype=torch.uint8)
            for spec in store.params:
                if spec.kind == "vec":
                    ids[spec.offset // ALIGN: (spec.offset + pad_to(spec.numel, ALIGN)) // ALIGN] = 1
            self.group_ids = ids.to(dev)
            self.groups = torch.tensor([[1.0, 1.0], [1.0, 0.0]], device=dev)
        self.defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, momentum=momentum)
        self.base_lr = lr
        self._host_step = 0
        self._host_lr = lr

    # ------------------------------------------------------------------ stepping
    def step_range(self, lo, hi):
        s = self.store
        if self.kind == "adam":
            ops.adam_step(s.p, s.g, self.m, self.v, s.p16, self.hyper, lo, hi)
        elif self.kind == "adamw":
            ops.adamw_step(s.p, s.g, self.m, self.v, s.p16, self.hyper, self.groups, self.group_ids, lo, hi)
        elif self.kind == "adamw8":
            ops.adamw8_step(s.p, s.g, self.m, self.v, self.m_scale, self.v_scale, s.p16, self.hyper, self.groups, self.group_ids,
                            self.seed, lo, hi)
        else:
            ops.sgd_step(s.p, s.g, self.m, s.p16, self.hyper, lo, hi)

    def finish_step(self):
        ops.advance_step(self.hyper)
        self._host_step += 1

    def step(self):
        for lo, hi in self.store.trainable_ranges():
            self.step_range(lo, hi)
        self.finish_step()

    def state_tensors(self):
        """Everything a step changes beside the parameters: what a capture's warm-up has to put back."""
        return [t for t in (self.m, self.v, self.m_scale, self.v_scale, self.hyper) if t is not None]

    def set_lr(self, lr):
        self._host_lr = lr
        self.hyper[LR] = lr

    def get_lr(self):
        return self._host_lr

    def set_grad_scale(self, s):
        self.hyper[GSCALE] = s

    # ------------------------------------------------------------------ torch.optim-compatible state
    def state_dict(self):
        # The reference builds the optimizer over model.parameters() - ALL of them, frozen ones included
        # (/root/reference/classif.py:124, utils.py:107-110) - so `params` indexes every parameter in registration
        # order and `state` holds entries only for those that received gradients (the trainable ones).
        st = self.store
        state = {}
        step = float(self.hyper[STEP].item())
        order = self._order()
        if step > 0:
            for i, spec in enumerate(order):
                if not spec.trainable:
                    continue
                m, v = self._moments(spec)
                if self.kind != "SGD":
                    state[i] = {"step": torch.tensor(step, dtype=torch.float32), "exp_avg": st.storage_to_logical(spec, m),
                                "exp_avg_sq": st.storage_to_logical(spec, v)}
                else:
                    state[i] = {"momentum_buffer": st.storage_to_logical(spec, m)}
        lr = float(self.get_lr())
        if self.kind != "SGD":
            group = {"lr": lr, "betas": tuple(self.defaults["betas"]), "eps": self.defaults["eps"],
                     "weight_decay": self.defaults["weight_decay"], "amsgrad": False, "maximize": False, "foreach": None,
                     "capturable": False, "differentiable": False, "fused": None, "decoupled_weight_decay": self.adamw}
        else:
            group = {"lr": lr, "momentum": self.defaults["momentum"], "dampening": 0, "weight_decay":
                     self.defaults["weight_decay"], "nesterov": False, "maximize": False, "foreach": None,
                     "differentiable": False, "fused": None, "initial_lr": self.base_lr}
        groups = [dict(group, params=list(range(len(order))))]
        if self.adamw:
            k = sum(spec.kind != "vec" for spec in order)
            groups = [dict(group, params=list(range(k))), dict(group, weight_decay=0.0, params=list(range(k, len(order))))]
        if self.kind == "adamw8" and step > 0:
            groups[0].update(m_scale=self.m_scale.clone(), v_scale=self.v_scale.clone())
        return {"state": state, "param_groups": groups}

    def _order(self):
        """The parameters as torch numbers them: in registration order, group by group."""
        ps = self.store.params
        return [s for s in ps if s.kind != "vec"] + [s for s in ps if s.kind == "vec"] if self.adamw else ps

    def _moments(self, spec):
        """(exp_avg or momentum, exp_avg_sq or None) of a parameter, fp32, in storage layout."""
        sl = slice(spec.offset, spec.offset + spec.numel)
        if self.kind != "adamw8":
            return self.m[sl].view(spec.storage_shape), None if self.v is None else self.v[sl].view(spec.storage_shape)
        lo, hi = spec.offset, spec.offset + pad_to(spec.numel, ALIGN)
        b = slice(lo // ALIGN, hi // ALIGN)
        return tuple(ops.adamw8_decode(t[lo:hi], s[b])[: spec.numel].view(spec.storage_shape)
                     for t, s in ((self.m, self.m_scale), (self.v, self.v_scale)))

    def _set_moment(self, spec, which, logical):
        st = self.store
        logical = logical.to(st.device, torch.float32)
        t = self.m if which == "m" else self.v
        if self.kind != "adamw8":
            st.logical_to_storage(spec, logical, t[spec.offset: spec.offset + spec.numel].view(spec.storage_shape))
            return
        lo, hi = spec.offset, spec.offset + pad_to(spec.numel, ALIGN)
        full = torch.zeros(hi - lo, device=st.device)
        st.logical_to_storage(spec, logical, full[: spec.numel].view(spec.storage_shape))
        codes, scales = ops.adamw8_encode(full, torch.full_like(full, 0.5), which)
        t[lo:hi] = codes
        (self.m_scale if which == "m" else self.v_scale)[lo // ALIGN: hi // ALIGN] = scales

    def load_state_dict(self, sd):
        st = self.store
        groups, order = sd["param_groups"], self._order()
        have = [len(g["params"]) for g in groups]
        k = sum(spec.kind != "vec" for spec in order)
        want = [k, len(order) - k] if self.adamw else [len(order)]
        if have != want:
            raise ValueError(f"optimizer state_dict covers {sum(have)} parameters in groups of {have}, the model has "
                             f"{len(st.params)} in groups of {want}" if self.adamw or len(have) > 1 else
                             f"optimizer state_dict covers {have[0]} parameters, the model has {len(st.params)}")
        self.set_lr(float(groups[0]["lr"]))
        step = 0.0
        for i, spec in enumerate(order):
            s = sd["state"].get(i)
            if s is None or not spec.trainable:
                continue
            if self.kind != "SGD":
                step = float(s["step"])
                self._set_moment(spec, "m", s["exp_avg"])
                self._set_moment(spec, "v", s["exp_avg_sq"])
            else:
                step = max(step, 1.0)
                self._set_moment(spec, "m", s["momentum_buffer"])
        for key, mine in (("m_scale", self.m_scale), ("v_scale", self.v_scale)):
            was = groups[0].get(key)
            if mine is not None and torch.is_tensor(was) and was.numel() == mine.numel():
                # a code times its scale, rounded, may give a scale some units in the last place away: the saved one is exact.
                # (Another compute type may have laid the arena out in another way: then nothing is near, and nothing taken.)
                was = was.to(mine.device)
                mine.copy_(torch.where((was - mine).abs() <= 2.0 ** -21 * mine, was, mine))
        self.hyper[STEP] = step
        self._host_step = int(step)


class StepLR:
    """lr = base_lr * gamma ** (epoch // step_size); the reference steps it once per epoch for SGD only."""

    def __init__(self, optimizer: ArenaOptimizer, step_size=1, gamma=0.1, last_epoch=0):
        self.opt, self.step_size, self.gamma, self.epoch = optimizer, step_size, gamma, last_epoch
        self.opt.set_lr(self.opt.base_lr * self.gamma ** (self.epoch // self.step_size))

    def step(self):
        self.epoch += 1
        self.opt.set_lr(self.opt.base_lr * self.gamma ** (self.epoch // self.step_size))
