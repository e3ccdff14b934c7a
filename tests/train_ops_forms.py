"""Forms of the group-norm and linear operators that each kernel of theirs has to take, shared by the CPU and GPU tests."""
import pytest
import torch

from distributedpytorch_amd import ops
from distributedpytorch_amd.nn.engine import Act, Context, ParamStore, Tape
from distributedpytorch_amd.nn.layers import Mlp
from tests import train_ops_cases as cases
from tests import train_ops_nets as nets
from tests import train_ops_oracle as O

# (n, h, w, c, groups): layouts without 16-byte vectors, small and large; with them, an image in one pass and in two
DRES = [(2, 40, 40, 30, 3), (2, 5, 5, 30, 3), (2, 6, 6, 64, 8), (1, 112, 112, 64, 32)]


def check_dresidual_alone(case, act, dtype, device):
    """The gradient under the activation is asked for, and there is no residual."""
    n, h, w, c, groups = case
    gen = torch.Generator().manual_seed(n + h + c)
    x, dy = (torch.randn(n, h, w, c, generator=gen).to(dtype) for _ in range(2))
    gamma, beta = torch.rand(c, generator=gen) + 0.5, 0.5 * torch.randn(c, generator=gen)
    xd, gd, bd = x.to(device), gamma.to(device), beta.to(device)
    y, (mean, rstd) = torch.empty_like(xd), torch.empty(2, n, groups, device=device)
    ops.group_norm_fwd(xd, gd, bd, groups, 1e-5, y, mean, rstd, act=act)
    for mask in (None, y) if act == "relu" else (None,):
        want, err = O.gn_backward(dy, x, gamma, beta, groups, mean.cpu(), rstd.cpu(), act, None if mask is None else mask.cpu(), None)
        dx, dres = (torch.full_like(xd, float("nan")) for _ in range(2))
        dg, db = torch.full((2, c), float("nan"), device=device)
        ops.group_norm_bwd(dy.to(device), xd, gd, bd, groups, mean, rstd, dx, dg, db, act=act, y=mask, dresidual=dres)
        for k, got in enumerate((dx, dg, db, dres)):
            O.close(("dx", "dgamma", "dbeta", "dresidual")[k], got, want[k], err[k], dtype if k in (0, 3) else torch.float32)


# What the plans choose beyond the cases of train_ops_cases: images of 2 to 13 vectors a thread, in groups of whole vectors and of parts
# of them, layers of 28 x 28 x 512 and 31 x 31 x 512
GN = [(1, 1, 86, 24, 8, "relu", True, ""), (1, 7, 37, 4, 4, "silu", True, ""), (1, 9, 2, 824, 4, "gelu", True, ""), (1, 113, 2, 36, 4, "relu", False, ""),
      (1, 7, 11, 104, 1, "silu", True, "inplace"), (1, 1, 17, 1544, 8, "relu", True, ""), (1, 3, 43, 216, 1, "relu", True, "inplace"),
      (1, 9, 2, 764, 4, "silu", False, ""), (1, 1, 66, 208, 1, "gelu", True, ""), (1, 14, 3, 1144, 8, "silu", True, "inplace"),
      (1, 2, 158, 168, 1, "relu", True, ""), (1, 5, 6, 788, 4, "none", True, ""), (1, 108, 1, 232, 1, "gelu", False, ""),
      (2, 3, 43, 216, 1, "gelu", True, "slice"), (16, 28, 28, 512, 32, "relu", True, ""), (16, 31, 31, 512, 32, "silu", True, "")]

# (rows, out, in, act, addend, extra), as train_ops_cases.LINEAR: every tile, split and way to the bias gradient in each direction
LINEAR = [(29, 200, 264, "gelu", True, ""), (130, 300, 2100, "relu", True, ""), (130, 2100, 300, "gelu", False, "accumulate"),
          (1500, 1500, 320, "silu", True, ""), (1500, 328, 1501, "gelu", True, ""), (2100, 2200, 320, "relu", False, ""), (2101, 320, 2199, "silu", False, ""),
          (1000, 520, 4100, "gelu", True, "accumulate"), (600, 4104, 1000, "relu", True, "slice"), (4200, 600, 1000, "none", True, "accumulate"),
          (1100, 1100, 1050, "silu", False, "accumulate"), (1100, 1700, 1600, "relu", False, ""), (1101, 2101, 2200, "gelu", True, "accumulate"),
          (1700, 1600, 264, "gelu", True, ""), (1700, 264, 1600, "relu", True, "slice"), (1000, 1600, 600, "silu", True, ""), (300, 1700, 1600, "none", False, "accumulate"),
          (5000, 40, 1600, "none", False, ""), (3701, 3499, 393, "gelu", True, ""), (3704, 392, 3504, "silu", True, "slice"), (392, 3704, 3504, "relu", False, ""),
          (401, 3701, 3499, "none", False, "accumulate")]

NARROW = [(16, 4, 10), (16, 1, 3), (512, 3, 2, 10), (24, 7, 1)]


def check_narrow_mlp(widths, device):
    """Hidden layers of fewer units than a 16-byte vector holds, against torch."""
    torch.manual_seed(sum(widths))
    store = ParamStore(device, torch.float32)
    m = Mlp(store, "m", widths, "gelu")
    store.finalize()
    x, dy = torch.randn(9, widths[0]), torch.randn(9, widths[-1])
    ctx = Context(store, True, Tape())
    xa = Act(x.view(9, 1, 1, -1).to(device), True)
    out = m(ctx, xa)
    out.grad = torch.zeros_like(out.data)
    out.grad[..., : widths[-1]] = dy.view(9, 1, 1, -1).to(device)
    y = out.data[:, 0, 0, : widths[-1]].clone()
    ctx.tape.backward()
    p = {s.name: store.get_logical(s).cpu().double().requires_grad_() for s in store.params}
    xd = x.double().requires_grad_()
    h = xd
    for i in range(len(widths) - 1):
        h = torch.nn.functional.linear(h if i == 0 else torch.nn.functional.gelu(h), p[f"m.{2 * i}.weight"], p[f"m.{2 * i}.bias"])
    h.backward(dy.double())
    # three products of at most 512 + 16 roundings and 32 elementwise ones each, forward and back, in norm over random data
    tol = 6 * 560 * O.E
    assert nets.rel(y, h) <= tol and nets.rel(xa.grad.view(9, -1), xd.grad) <= tol
    for s in store.params:
        assert nets.rel(store.storage_to_logical(s, store.gview(s)), p[s.name].grad) <= tol, s.name


# (rows, out, in): the kernel for few rows and the one behind its bound, tiles and splits of every kind
INF = [(64, 40, 72), (65, 40, 72), (300, 260, 264), (1000, 520, 4100), (3500, 3700, 24)]


def check_infinities(case, dtype, device):
    """Infinities in an operand: an infinity of the right sign, or NaN where the formula in fp32 has one, whatever kernel takes the sizes."""
    m, n, k = case
    gen = torch.Generator().manual_seed(m + n + k)
    x, w, dy = (torch.randn(*s, generator=gen).to(dtype) for s in ((m, k), (n, k), (m, n)))
    # numbers of one bf16 part beside those of three, and zeros: infinity times zero is NaN
    for t in (x, w, dy):
        t[:, 1::5] = t[:, 1::5].sign()
        t[::7, 3::5] = 0
    x[5, 3], x[9, 2], x[9, 7], x[m - 1, k - 1] = float("inf"), float("inf"), -float("inf"), -float("inf")
    w[11, 6] = -float("inf")
    dy[7, 4], dy[2, 0], dy[m - 1, 9] = float("inf"), -float("inf"), float("nan")
    xd, wd, dyd = x.to(device), w.to(device), dy.to(device)

    def nan(*s, dt=dtype):
        return torch.full(s, float("nan"), dtype=dt, device=device)
    for act in ("none", "relu"):
        y = nan(m, n)
        ops.linear_fprop(xd, wd, y, act=act)
        want, err = O.product(x, w)
        O.close("y", y, torch.where(want.isnan(), want, O.phi(want, act)[0]), err, dtype)
    dx, add = nan(m, k), torch.randn(m, k, generator=gen).to(dtype)
    ops.linear_dgrad(dyd, wd, dx, addend=add.to(device))
    want, err = O.product(dy, w.t())
    O.close("dx", dx, want + add.to(O.D), err + 2 * O.E * (want.abs() + add.to(O.D).abs()), dtype)
    dw, db = nan(n, k, dt=torch.float32), nan(n, dt=torch.float32)
    ops.linear_wgrad(dyd, xd, dw, db)
    want, err = O.product(dy.t(), x.t())
    O.close("dw", dw, want, err)
    O.close("db", db, dy.to(O.D).sum(0), (m + 8) * O.E * dy.to(O.D).abs().sum(0))


def _norm(device, which, **kw):
    a = dict(x=torch.randn(2, 4, 4, 8, device=device), dy=torch.randn(2, 4, 4, 8, device=device), gamma=torch.ones(8, device=device), beta=torch.zeros(8, device=device),
             mean=torch.zeros(4, device=device), rstd=torch.ones(4, device=device), y=torch.empty(2, 4, 4, 8, device=device), dx=torch.empty(2, 4, 4, 8, device=device),
             dg=torch.empty(8, device=device), db=torch.empty(8, device=device), res=None, dres=None)
    for k, v in kw.items():
        a[k] = v(a)
    if which == "fwd":
        ops.group_norm_fwd(a["x"], a["gamma"], a["beta"], 2, 1e-5, a["y"], a["mean"], a["rstd"], residual=a["res"])
    else:
        ops.group_norm_bwd(a["dy"], a["x"], a["gamma"], a["beta"], 2, a["mean"], a["rstd"], a["dx"], a["dg"], a["db"], residual=a["res"], dresidual=a["dres"])


def _product(device, which, **kw):
    a = dict(x=torch.randn(8, 8, device=device), w=torch.randn(8, 8, device=device), y=torch.empty(8, 8, device=device), z=torch.empty(8, 8, device=device),
             bias=torch.randn(8, device=device), dy=torch.randn(8, 8, device=device), dw=torch.empty(8, 8, device=device), db=torch.empty(8, device=device))
    for k, v in kw.items():
        a[k] = v(a)
    if which == "fprop":
        ops.linear_fprop(a["x"], a["w"], a["y"], bias=a["bias"], act="gelu", preact=a["z"])
    else:
        ops.linear_wgrad(a["dy"], a["x"], a["dw"], db=a["db"])


# arguments that share memory: what a kernel writes another block may still read
SHARED = {
    "mean is rstd": lambda d: _norm(d, "fwd", mean=lambda a: a["rstd"]),
    "mean inside gamma": lambda d: _norm(d, "fwd", mean=lambda a: a["gamma"][2:6]),
    "rstd inside y": lambda d: _norm(d, "fwd", rstd=lambda a: a["y"].view(-1)[8:12]),
    "rstd inside x": lambda d: _norm(d, "fwd", rstd=lambda a: a["x"].view(-1)[-4:]),
    "beta inside y": lambda d: _norm(d, "fwd", beta=lambda a: a["y"].view(-1)[16:24]),
    "mean inside the residual": lambda d: _norm(d, "fwd", res=lambda a: a["x"].clone(), mean=lambda a: a["res"].view(-1)[:4]),
    "dgamma is dbeta": lambda d: _norm(d, "bwd", dg=lambda a: a["db"]),
    "dgamma is gamma": lambda d: _norm(d, "bwd", dg=lambda a: a["gamma"]),
    "dbeta inside mean and beyond": lambda d: (lambda b: _norm(d, "bwd", mean=lambda a: b[:4], db=lambda a: b[3:11]))(torch.zeros(16, device=d)),
    "dbeta inside dx": lambda d: _norm(d, "bwd", db=lambda a: a["dx"].view(-1)[:8]),
    "dbeta inside dy": lambda d: _norm(d, "bwd", db=lambda a: a["dy"].view(-1)[:8]),
    "gamma inside dx": lambda d: _norm(d, "bwd", gamma=lambda a: a["dx"].view(-1)[:8]),
    "rstd inside dresidual": lambda d: _norm(d, "bwd", res=lambda a: a["x"].clone(), dres=lambda a: torch.empty_like(a["x"]), rstd=lambda a: a["dres"].view(-1)[:4]),
    "bias inside y": lambda d: _product(d, "fprop", bias=lambda a: a["y"][3]),
    "bias inside preact": lambda d: _product(d, "fprop", bias=lambda a: a["z"][7]),
    "db inside dw": lambda d: _product(d, "wgrad", db=lambda a: a["dw"][0]),
    "db inside dy": lambda d: _product(d, "wgrad", db=lambda a: a["dy"][7]),
    "db inside x": lambda d: _product(d, "wgrad", db=lambda a: a["x"][0]),
}


def check_shared(name, device):
    with pytest.raises(ValueError, match="overlaps"):
        SHARED[name](device)


def check_neighbours(device):
    """Arguments that lie side by side in one buffer are apart."""
    b = torch.zeros(4 + 4 + 8 + 8 + 256 + 8 + 8, device=device)
    part = lambda lo, n: b[lo: lo + n]  # noqa: E731
    y = part(24, 256).view(2, 4, 4, 8)
    _norm(device, "fwd", mean=lambda a: part(0, 4), rstd=lambda a: part(4, 4), gamma=lambda a: part(8, 8), beta=lambda a: part(16, 8), y=lambda a: y)
    _norm(device, "bwd", mean=lambda a: part(0, 4), rstd=lambda a: part(4, 4), gamma=lambda a: part(8, 8), beta=lambda a: part(16, 8), dx=lambda a: y,
          dg=lambda a: part(280, 8), db=lambda a: part(288, 8))
    c = torch.zeros(8 + 64 + 8, device=device)
    _product(device, "fprop", bias=lambda a: c[:8], y=lambda a: c[8:72].view(8, 8))
    _product(device, "wgrad", db=lambda a: c[72:], dw=lambda a: c[8:72].view(8, 8))


# (n, h, w, c, groups): vector kernels in one pass and two, one channel a lane, any layout; up to 104 values a thread
FAR = [(4, 28, 28, 512, 32), (2, 7, 7, 64, 8), (2, 112, 112, 64, 32), (2, 13, 13, 30, 3), (2, 40, 40, 30, 3), (1, 64, 64, 48, 4)]


def check_far_means(case, device):
    """Means of 330 with a spread of 0.1.  m values summed one behind another round E (1 + ... + m) of their size, so E m / 2 of the sum:
    52 for 104 values a thread, as many again where the partial sums of a group's threads are added (at most 128), some 20 for
    trees, joins and the division.  The second moment holds that error squared, and 512 roundings of its own."""
    n, h, w, c, groups = case
    gen = torch.Generator().manual_seed(h + c)
    x = torch.randn(n, h, w, c, generator=gen) * 0.1 + 330 + 0.002 * torch.arange(c)
    gamma, beta = torch.rand(c, generator=gen) + 0.5, torch.randn(c, generator=gen)
    xd, y, (mean, rstd) = x.to(device), torch.empty(n, h, w, c, device=device), torch.empty(2, n, groups, device=device)
    ops.group_norm_fwd(xd, gamma.to(device), beta.to(device), groups, 1e-5, y, mean, rstd)
    t = O.grouped(x, groups)
    mu = t.mean((1, 3))
    d = t - mu[:, None, :, None]
    rs = 1 / ((d * d).mean((1, 3)) + 1e-5).sqrt()
    off = 136 * O.E * mu.abs()
    e_rs = rs * (0.5 * (off * rs) ** 2 + 544 * O.E)
    O.close("mean", mean, mu, off)
    O.close("rstd", rstd, rs, e_rs)
    hat = (d * rs[:, None, :, None]).reshape(x.shape)
    e = gamma.to(O.D) * (hat.abs() * O._per(e_rs / rs, x, groups) + O._per(off * rs, x, groups)) + 8 * O.E * (hat.abs() + beta.abs())
    O.close("y", y, hat * gamma.to(O.D) + beta.to(O.D), e)


def check_long_sums(device):
    """Parameter gradients over 300 thousand pixels and rows, of one sign: at most 2^13 roundings in a row."""
    gen = torch.Generator().manual_seed(3)
    n, h, w, c, groups = 1, 600, 500, 8, 2
    x, dy = torch.randn(n, h, w, c, generator=gen), torch.rand(n, h, w, c, generator=gen) + 0.5
    xd, y, (mean, rstd), (dg, db) = x.to(device), torch.empty(n, h, w, c, device=device), torch.empty(2, n, groups, device=device), torch.empty(2, c, device=device)
    ga, be = torch.ones(c, device=device), torch.zeros(c, device=device)
    ops.group_norm_fwd(xd, ga, be, groups, 1e-5, y, mean, rstd)
    ops.group_norm_bwd(dy.to(device), xd, ga, be, groups, mean, rstd, y, dg, db)
    O.close("dbeta", db, dy.to(O.D).sum((0, 1, 2)), 2 ** 13 * O.E * dy.to(O.D).sum((0, 1, 2)))
    dw, db = torch.empty(c, c, device=device), torch.empty(c, device=device)
    ops.linear_wgrad(dy.view(-1, c).to(device), xd.view(-1, c), dw, db)
    O.close("db", db, dy.to(O.D).sum((0, 1, 2)), 2 ** 13 * O.E * dy.to(O.D).sum((0, 1, 2)))
