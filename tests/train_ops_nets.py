"""Group norm, linear products and AdamW together, as layers, networks and an optimizer use them; shared by the CPU and GPU tests."""
import copy

import torch
import torch.nn.functional as F

from distributedpytorch_amd.models.factory import get_model
from distributedpytorch_amd.nn.engine import Act, Context, ParamStore, Tape
from distributedpytorch_amd.nn.layers import AvgPool2d, Conv2d, ConvGNAct, GNAct, GroupNorm2d, Mlp
from distributedpytorch_amd.nn.loss import Criterion
from distributedpytorch_amd.nn.optim import ArenaOptimizer
from distributedpytorch_amd.parallel.ddp import DistributedModel

E = 2.0 ** -24
ACT = {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}


def rel(a, b):
    a, b = a.detach().cpu().double(), b.detach().cpu().double()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


class SmallNet:
    """conv + group norm + act, group norm + act alone, conv + group norm + residual + act, pool, residual MLP, MLP."""

    def __init__(self, store, act, mlp_act):
        self.act, self.mlp_act = act, mlp_act
        self.c1 = ConvGNAct(Conv2d(store, "c1", 3, 16, 3, 1, 1, bias=False), GroupNorm2d(store, "n1", 16, 4), act)
        self.n2 = GNAct(GroupNorm2d(store, "n2", 16, 2), act)
        self.c3 = ConvGNAct(Conv2d(store, "c3", 16, 16, 3, 1, 1, bias=False), GroupNorm2d(store, "n3", 16, 8), act)
        self.pool = AvgPool2d(adaptive=1)
        self.block = Mlp(store, "block", (16, 40, 16), mlp_act)
        self.one = Mlp(store, "one", (16, 16), mlp_act)
        self.head = Mlp(store, "head", (16, 24, 24, 10), mlp_act)

    def forward(self, ctx, x):
        a = self.c1(ctx, x)
        b = self.n2(ctx, a, residual=a)
        x = self.pool(ctx, self.c3(ctx, b, residual=a))
        x = self.block(ctx, x, residual=x)
        x = self.one(ctx, x, residual=x)
        return self.head(ctx, x)

    def plain(self, p, x):
        """The same in torch on a dict of parameters, NCHW."""
        act, mact = ACT[self.act], ACT[self.mlp_act]
        a = act(F.group_norm(F.conv2d(x, p["c1.weight"], padding=1), 4, p["n1.weight"], p["n1.bias"]))
        b = act(F.group_norm(a, 2, p["n2.weight"], p["n2.bias"]) + a)
        x = act(F.group_norm(F.conv2d(b, p["c3.weight"], padding=1), 8, p["n3.weight"], p["n3.bias"]) + a).mean((2, 3))
        x = F.linear(mact(F.linear(x, p["block.0.weight"], p["block.0.bias"])), p["block.2.weight"], p["block.2.bias"]) + x
        x = F.linear(x, p["one.weight"], p["one.bias"]) + x
        for i in (0, 2, 4):
            x = F.linear(x if i == 0 else mact(x), p[f"head.{i}.weight"], p[f"head.{i}.bias"])
        return x


def check_layers(device, act, mlp_act):
    torch.manual_seed(11)
    store = ParamStore(device, torch.float32)
    net = SmallNet(store, act, mlp_act)
    store.finalize()
    for spec in store.params:          # norms that scale and shift
        if spec.kind == "vec":
            store.set_logical(spec, store.get_logical(spec).cpu() + 0.3 * torch.randn(spec.logical_shape))
    x, dy = torch.randn(5, 3, 7, 6), torch.randn(5, 10)
    xin = torch.zeros(5, 7, 6, 4, device=device)
    xin[..., :3] = x.permute(0, 2, 3, 1).to(device)
    ctx = Context(store, True, Tape())
    out = net.forward(ctx, Act(xin, False))
    out.grad = torch.zeros_like(out.data)
    out.grad[..., :10] = dy.view(5, 1, 1, 10).to(device)
    got = out.data[:, 0, 0, :10].clone()
    ctx.tape.backward()
    p = {s.name: store.get_logical(s).cpu().double().requires_grad_() for s in store.params}
    want = net.plain(p, x.double())
    want.backward(dy.double())
    # eight layers of at most 544 roundings each (a group's sum of 512 terms, 32 elementwise), and a norm's backward pass, which
    # takes mean and slope off its gradient, leaves at least a quarter of its size on random data
    tol = 8 * 544 * E * 4
    assert rel(got, want) <= tol
    for s in store.params:
        g = store.storage_to_logical(s, store.gview(s))
        assert rel(g, p[s.name].grad) <= tol, (s.name, rel(g, p[s.name].grad))


def check_adamw_torch(device):
    """Five steps of the optimizer against torch.optim.AdamW with the two parameter groups it stands for, and the state both ways."""
    torch.manual_seed(3)
    store = ParamStore(device, torch.float32)
    net = SmallNet(store, "relu", "relu")  # noqa: F841
    store.finalize()
    opt = ArenaOptimizer(store, "adamw", lr=3e-3, weight_decay=0.1)
    order = opt._order()
    ps = [store.get_logical(s).cpu().clone() for s in order]
    k = sum(s.kind != "vec" for s in order)
    topt = torch.optim.AdamW([{"params": ps[:k]}, {"params": ps[k:], "weight_decay": 0.0}], lr=3e-3, weight_decay=0.1)

    # a step: 4 roundings of p and 32 of the update, which |m| / sqrt(v) <= 1 / sqrt(1 - b2) < 32 bounds; both sides, each step
    def close(a, b, steps):
        err = (a.cpu().double() - b.double()).abs()
        assert bool((err <= 2 * steps * E * (4 * b.double().abs() + 32 * 3e-3 * 32)).all()), float(err.max())

    def steps(n, seed, o):
        gen = torch.Generator().manual_seed(seed)
        for _ in range(n):
            for s, p in zip(order, ps):
                p.grad = torch.randn(s.logical_shape, generator=gen)
                store.logical_to_storage(s, p.grad.to(device), store.gview(s))
            o.step()
            topt.step()
    steps(5, 1, opt)
    for s, p in zip(order, ps):
        close(store.get_logical(s), p, 5)
    sd = opt.state_dict()
    topt.load_state_dict(copy.deepcopy(sd))          # torch takes the layout (its state shares memory, like torch's own)
    back = ArenaOptimizer(store, "adamw", lr=1.0)
    back.load_state_dict(topt.state_dict())
    assert torch.equal(back.m, opt.m) and torch.equal(back.v, opt.v) and torch.equal(back.hyper[5], opt.hyper[5])
    assert back.get_lr() == opt.get_lr()
    steps(2, 2, opt)
    for s, p in zip(order, ps):
        close(store.get_logical(s), p, 7)


def model(device, dtype, kind, name="resnet", seed=0, **kw):
    torch.manual_seed(seed)
    kw = dict(dict(norm="group", act="silu", head_hidden=(48,)), **kw)
    net, _ = get_model(name, 10, device=device, dtype=dtype, small_input=True, **kw)
    net.seed_rng(1234)
    return DistributedModel(net, Criterion(), ArenaOptimizer(net.store, kind, lr=1e-3, seed=5))


def batch(n, net, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.zeros(n, 32, 32, net.in_channels, dtype=dtype)
    x[..., :3] = torch.randn(n, 32, 32, 3, generator=gen).to(dtype)
    return x.to(net.store.device), torch.randint(0, 10, (n,), generator=gen).to(net.store.device)


def check_training(device, dtype, kind, n=4, steps=3):
    """Training runs, is reproducible bit for bit, goes on from a checkpoint as if it had not stopped, and its evaluation is the
    forward pass of training."""
    runs = []
    for resume in (False, True, False):
        dm = model(device, dtype, kind)
        for i in range(steps):
            if resume and i == 2:
                sd, od, rng = dm.net.state_dict(""), dm.opt.state_dict(), dm.net.rng.clone()
                dm = model(device, dtype, kind, seed=99)
                dm.net.load_state_dict(sd)
                dm.opt.load_state_dict(od)
                dm.net.rng.copy_(rng)
            dm.reset_epoch_metrics()
            dm.train_step(*batch(n, dm.net, dtype, i))
        runs.append((dm.epoch_metrics()[0], dm.net.store.p.clone()))
    assert all(r[0] == runs[0][0] for r in runs) and all(torch.equal(r[1], runs[0][1]) for r in runs), [r[0] for r in runs]
    assert torch.isfinite(runs[0][1]).all()
    x, _ = batch(n, dm.net, dtype, 7)
    dm.net.train()
    a = dm.net.forward(x)[1].data.clone()
    dm.net.eval()
    assert torch.equal(a, dm.net.forward(x)[1].data)
