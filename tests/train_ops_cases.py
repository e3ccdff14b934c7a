"""Cases of the group-norm, linear and AdamW operators, run on the CPU and on the GPU by the tests beside this file."""
import pytest
import torch

from tests import train_ops_oracle as O
from distributedpytorch_amd import ops
from distributedpytorch_amd.nn.optim import make_hyper

# (n, h, w, c, groups, act, residual, extra): extra "slice": channel slices of a wider buffer; "far": means far from zero;
# "flat": constant images; "inplace": outputs are inputs
GN = [(1, 1, 1, 8, 1, "none", False, ""), (1, 1, 1, 8, 8, "relu", True, ""), (2, 1, 1, 64, 2, "silu", False, ""), (1, 7, 7, 512, 32, "relu", False, ""),
      (2, 9, 5, 24, 3, "gelu", True, ""), (3, 5, 5, 30, 3, "silu", True, ""), (2, 4, 4, 7, 7, "relu", False, ""), (1, 33, 3, 90, 6, "silu", False, ""),
      (2, 14, 14, 320, 32, "relu", True, ""), (2, 8, 8, 96, 32, "silu", False, ""), (1, 3, 3, 1504, 1, "gelu", False, ""),
      (1, 2, 2, 2050, 2, "relu", True, ""), (3, 13, 11, 64, 8, "relu", True, "slice"), (2, 6, 6, 24, 4, "silu", True, "slice"),
      (2, 16, 16, 32, 4, "none", False, "far"), (2, 28, 28, 64, 8, "relu", False, "far"), (1, 4, 4, 16, 4, "silu", False, "flat"),
      (2, 12, 12, 64, 8, "relu", True, "inplace"), (2, 12, 12, 64, 8, "silu", True, "inplace"), (2, 5, 5, 18, 2, "gelu", True, "inplace"),
      (1, 64, 64, 32, 8, "relu", True, ""), (1, 56, 56, 256, 32, "relu", True, ""), (1, 57, 55, 64, 2, "silu", True, ""),
      (3, 28, 28, 128, 32, "gelu", True, ""), (70, 3, 3, 16, 2, "relu", True, ""), (1, 112, 112, 64, 32, "silu", False, ""),
      (2, 20, 20, 1024, 1, "none", True, ""), (0, 4, 4, 8, 2, "relu", False, "")]


def _buf(shape, dtype, device, slice_, gen, scale=1.0):
    n, h, w, c = shape
    t = (torch.randn(shape, generator=gen) * scale).to(dtype)
    return _place(t, device, slice_)


def _place(t, device, slice_):
    if not slice_:
        return t.to(device)
    n, h, w, c = t.shape
    pad = 8 if c % 8 == 0 else 4
    wide = torch.full((n, h, w, c + 3 * pad), float("nan"), dtype=t.dtype, device=device)
    wide[..., pad: pad + c] = t.to(device)
    return wide[..., pad: pad + c]


def check_group_norm(case, dtype, device):
    n, h, w, c, groups, act, residual, extra = case
    gen = torch.Generator().manual_seed(7 + n + h + c)
    sl = extra == "slice"
    x = torch.randn(n, h, w, c, generator=gen)
    if extra == "far":
        x = x * 0.1 + 300.0 + torch.arange(c) * 0.5
    if extra == "flat":
        x = torch.full_like(x, 3.25)
    x = x.to(dtype)
    res = torch.randn(n, h, w, c, generator=gen).to(dtype) if residual else None
    dy = torch.randn(n, h, w, c, generator=gen).to(dtype)
    gamma, beta = torch.rand(c, generator=gen) + 0.5, 0.5 * torch.randn(c, generator=gen)
    eps = 1e-5
    want, w_mean, w_rstd, e_y, e_mean, e_rstd = O.gn_forward(x, gamma, beta, groups, eps, act, res)
    xd, dyd, rd = _place(x, device, sl), _place(dy, device, sl), (_place(res, device, sl) if residual else None)
    gd, bd = gamma.to(device), beta.to(device)
    y = torch.full((n, h, w, c), float("nan"), dtype=dtype, device=device)
    if sl:
        y = _place(y, device, True)
    if extra == "inplace":
        y = rd.clone()
        rd_in = y
    else:
        rd_in = rd
    mean, rstd = torch.full((2, n, groups), float("nan"), device=device)
    ops.group_norm_fwd(xd, gd, bd, groups, eps, y, mean, rstd, act=act, residual=rd_in)
    if n:
        O.close("mean", mean, w_mean, e_mean)
        O.close("rstd", rstd, w_rstd, e_rstd)
        O.close("y", y, want, e_y, dtype)
    if sl:
        assert torch.isnan(y._base[..., : y.storage_offset()]).all(), "channels outside the slice were written"

    for use_y in ((False, True) if act == "relu" else (False,)):
        yk = y if use_y else None
        mc, rc, yc = mean.cpu(), rstd.cpu(), (y.cpu() if use_y else None)
        (dx_w, dg_w, db_w, dr_w), (e_dx, e_dg, e_db, e_dr) = O.gn_backward(dy, x, gamma, beta, groups, mc, rc, act, yc, res)
        dx = torch.full((n, h, w, c), float("nan"), dtype=dtype, device=device)
        dres = torch.full_like(dx, float("nan")) if residual else None
        if sl:
            dx = _place(dx, device, True)
            dres = _place(dres, device, True) if residual else None
        dy_in = dyd
        if extra == "inplace":
            dy_in = dyd.clone()
            dres = dy_in
            dx = xd.clone()
            x_in = dx
        else:
            x_in = xd
        dg, db = torch.full((2, c), float("nan"), device=device)
        ops.group_norm_bwd(dy_in, x_in, gd, bd, groups, mean, rstd, dx, dg, db, act=act, y=yk, residual=rd, dresidual=dres)
        O.close("dx", dx, dx_w, e_dx, dtype)
        O.close("dgamma", dg, dg_w, e_dg)
        O.close("dbeta", db, db_w, e_db)
        if residual:
            O.close("dres", dres, dr_w, e_dr, dtype)
        if residual and extra == "":            # parameter gradients that nobody wants, and no residual gradient
            dx2 = torch.empty_like(dx)
            ops.group_norm_bwd(dyd, xd, gd, bd, groups, mean, rstd, dx2, None, None, act=act, y=yk, residual=rd)
            O.close("dx alone", dx2, dx_w, e_dx, dtype)


# (rows, out, in, act, addend, extra): extra "slice": matrices are column slices; "accumulate": weight gradient added
LINEAR = [(1, 1, 1, "none", False, ""), (1, 8, 8, "relu", True, ""), (1, 512, 4096, "relu", False, ""), (3, 1000, 520, "gelu", False, ""),
          (16, 72, 264, "silu", True, ""), (17, 40, 33, "gelu", True, ""), (31, 257, 129, "relu", True, "accumulate"), (64, 64, 64, "none", False, "accumulate"),
          (65, 63, 65, "silu", False, ""), (129, 130, 128, "gelu", True, "slice"), (200, 10, 512, "none", False, ""), (256, 256, 256, "relu", True, "slice"),
          (257, 384, 192, "gelu", True, ""), (300, 520, 72, "silu", True, ""), (1021, 1000, 96, "none", True, ""), (0, 16, 24, "gelu", False, "")]


def _mat(t, device, slice_):
    if not slice_:
        return t.to(device)
    wide = torch.full((t.shape[0], t.shape[1] + 24), float("nan"), dtype=t.dtype, device=device)
    wide[:, 8: 8 + t.shape[1]] = t.to(device)
    return wide[:, 8: 8 + t.shape[1]]


def check_linear(case, dtype, device):
    m, n, k, act, with_add, extra = case
    sl = extra == "slice"
    gen = torch.Generator().manual_seed(m + 3 * n + 5 * k)
    x, w = torch.randn(m, k, generator=gen).to(dtype), (torch.randn(n, k, generator=gen) / k ** 0.5).to(dtype)
    bias, add = torch.randn(n, generator=gen), torch.randn(m, n, generator=gen).to(dtype) if with_add else None
    xd, wd, ad = _mat(x, device, sl), _mat(w, device, sl), (_mat(add, device, sl) if with_add else None)
    # forward
    z, e = O.product(x, w)
    mag = O.L_POINT * O.E * (z.abs() + bias.to(O.D).abs() + (add.to(O.D).abs() if with_add else 0))
    z = z + bias.to(O.D) + (add.to(O.D) if with_add else 0)
    e = e + mag
    smooth = act in ("silu", "gelu")
    y = _mat(torch.full((m, n), float("nan"), dtype=dtype), device, sl)
    pre = _mat(torch.full((m, n), float("nan"), dtype=dtype), device, sl) if act != "none" else None
    ops.linear_fprop(xd, wd, y, bias=bias.to(device), act=act, addend=ad, preact=pre)
    O.close("y", y, O.phi(z, act)[0], 1.2 * e + smooth * O.L_POINT * O.E * (1 + z.abs()), dtype)
    if pre is not None:
        O.close("preact", pre, z, e, dtype)
    y2 = _mat(torch.full((m, n), float("nan"), dtype=dtype), device, sl)
    ops.linear_fprop(xd, wd, y2)
    z2, e2 = O.product(x, w)
    O.close("bare product", y2, z2, e2, dtype)
    # data gradient
    dy = torch.randn(m, n, generator=gen).to(dtype)
    pz = torch.randn(m, k, generator=gen).to(dtype)
    add2 = torch.randn(m, k, generator=gen).to(dtype) if with_add else None
    d, e = O.product(dy, w.t())
    if with_add:
        e = e + O.L_POINT * O.E * (d.abs() + add2.to(O.D).abs())
        d = d + add2.to(O.D)
    slope = O.phi(pz.to(O.D), act)[1]
    dx = _mat(torch.full((m, k), float("nan"), dtype=dtype), device, sl)
    dyd = _mat(dy, device, sl)
    ops.linear_dgrad(dyd, wd, dx, act=act, preact=_mat(pz, device, sl) if act != "none" else None,
                     addend=_mat(add2, device, sl) if with_add else None)
    O.close("dx", dx, d * slope, e * slope.abs() + d.abs() * smooth * O.L_POINT * O.E * (1 + pz.to(O.D).abs()) + O.E * (d * slope).abs(), dtype)
    # weight and bias gradients
    dw = torch.full((n, k), float("nan"), device=device)
    db = torch.full((n,), float("nan"), device=device)
    acc = extra == "accumulate"
    if acc:
        dw.fill_(2.0)
        db.fill_(-3.0)
    ops.linear_wgrad(dyd, xd, dw, db=db, accumulate=acc)
    gw, ew = O.product(dy.t(), x.t())
    gb, eb = dy.to(O.D).sum(0), (m + 8) * O.E * dy.to(O.D).abs().sum(0)
    if acc:
        gw, ew, gb, eb = gw + 2.0, ew + O.E * (gw.abs() + 2), gb - 3.0, eb + O.E * (gb.abs() + 3)
    O.close("dw", dw, gw, ew)
    O.close("db", db, gb, eb)
    if not acc:
        dw2 = torch.full((n, k + 8), float("nan"), device=device)[:, :k]
        ops.linear_wgrad(dyd, xd, dw2)
        O.close("dw without db, in a wider matrix", dw2, gw, ew)


# tensor sizes of an arena
ADAMW = [(1,), (64,), (3, 5000, 64), (70, 1, 900, 64, 40000), (131072, 64)]


def arena(sizes, gen):
    pads = [(s + 63) // 64 * 64 for s in sizes]
    live = torch.cat([torch.cat([torch.ones(s), torch.zeros(q - s)]) for s, q in zip(sizes, pads)])
    ids = torch.cat([torch.full((q // 64,), i % 3, dtype=torch.uint8) for i, q in enumerate(pads)])
    return live, ids, torch.tensor([[1.0, 1.0], [0.5, 0.0], [2.0, 0.1]])


def check_adamw(sizes, bits, device):
    gen = torch.Generator().manual_seed(sum(sizes))
    live, ids, groups = arena(sizes, gen)
    n = live.numel()
    spread = (10.0 ** (-6 * torch.rand(n, generator=gen)))
    p, g = torch.randn(n, generator=gen) * live, torch.randn(n, generator=gen) * spread * live
    m, v = 0.1 * torch.randn(n, generator=gen) * spread * live, (torch.rand(n, generator=gen) * spread ** 2) * live
    lr, b1, b2, eps, wd, step, gs, seed = 2e-3, 0.9, 0.999, 1e-8, 0.1, 6, 0.25, 77
    hyper = make_hyper(lr, b1, b2, eps, wd, float(step), 0.0, gs, device=device)
    per = groups[ids.long()].repeat_interleave(64, 0)
    lr32 = float(torch.tensor(lr))          # the kernels read lr, eps and the decay from a vector of fp32 values
    args = (lr32, b1, b2, float(torch.tensor(eps)), float(torch.tensor(wd)), step, gs)
    dev = lambda t: t.clone().to(device)  # noqa: E731
    pd, gd, p16 = dev(p), dev(g), torch.zeros(n, dtype=torch.bfloat16, device=device)
    lo, hi = (0, None) if len(sizes) < 3 else (64, n - 64)
    sl = slice(lo, n if hi is None else hi)
    if bits == 32:
        md, vd = dev(m), dev(v)
        ops.adamw_step(pd, gd, md, vd, p16, hyper, groups.to(device), ids.to(device), lo, hi)
        m_in, v_in = m, v
    else:
        half = torch.full((n,), 0.5)
        (mc, ms), (vc, vs) = ops.adamw8_encode(m, half, "m"), ops.adamw8_encode(v, half, "v")
        m_in, v_in = ops.adamw8_decode(mc, ms), ops.adamw8_decode(vc, vs)
        md, msd, vd, vsd = dev(mc), dev(ms), dev(vc), dev(vs)
        ops.adamw8_step(pd, gd, md, vd, msd, vsd, p16, hyper, groups.to(device), ids.to(device), seed, lo, hi)
    wp, wm, wv, upd = O.adamw(p, g, m_in, v_in, args, per)
    O.close("p", pd[sl], wp[sl], (O.E * (4 * p.to(O.D).abs() + 24 * upd.abs() + 8 * upd.abs() * (m_in.to(O.D).abs() + g.to(O.D).abs()) / wm.abs().clamp_min(1e-30)))[sl])
    O.close("p16", p16[sl], pd[sl].cpu().to(O.D), 0.0, torch.bfloat16)
    out = torch.ones(n, dtype=torch.bool)
    out[sl] = False
    assert torch.equal(pd.cpu()[out], p[out]) and not p16.cpu()[out].any(), "elements outside the range changed"
    if bits == 32:
        O.close("m", md[sl], wm[sl], (4 * O.E * (m.abs() + g.abs()).to(O.D))[sl])
        O.close("v", vd[sl], wv[sl], (4 * O.E * wv)[sl])
        assert torch.equal(md.cpu()[out], m[out]) and torch.equal(vd.cpu()[out], v[out])
        return
    from distributedpytorch_amd.ops import ref_ops
    rm, rv = ref_ops.adamw8_random(seed, step, 0, n, "cpu")
    for which, want, r, code, scale, (_, top, least, nb) in (("m", wm, rm, md, msd, ref_ops.ADAMW8_FORMATS["m"]), ("v", wv, rv, vd, vsd, ref_ops.ADAMW8_FORMATS["v"])):
        b = want.reshape(-1, 64)
        most = b.abs().amax(1, keepdim=True)
        some = most >= 2.0 ** -100
        y = torch.where(some, b.abs() / most.clamp_min(2.0 ** -100) * top, torch.zeros_like(b))
        grid = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** least))) - nb)
        q = (torch.floor(y / grid + (r.reshape(b.shape).to(O.D) + 0.5) / 65536) * grid).clamp_max(top)
        if which == "v":
            q = torch.where((b > 0) & some, q.clamp_min(2.0 ** (least - nb)), q)
        q = (q * torch.sign(b)).reshape(-1)
        O.close(f"{which} scale", scale[lo // 64: (n if hi is None else hi) // 64],
                torch.where(some, most / top, torch.zeros_like(most)).reshape(-1)[lo // 64: (n if hi is None else hi) // 64],
                (8 * O.E * torch.where(some, most / top, torch.zeros_like(most)).reshape(-1))[lo // 64: (n if hi is None else hi) // 64])
        got = code.cpu().float().to(O.D)
        d = (got - q).abs()[sl]
        # y is within 16 * 8 E of its value in steps, so the floor differs with probability < 2^-16, by one step
        assert int((d > 0).sum()) <= 2 + n * 2.0 ** -15, (which, int((d > 0).sum()))
        assert bool((d <= 2 * torch.maximum(grid.reshape(-1), torch.full_like(q, 2.0 ** (least - nb)))[sl]).all())
        if which == "v":
            assert bool((got[sl][(want > 2.0 ** -60)[sl]] > 0).all()), "a positive second moment became zero"


# ------------------------------------------------------------------------------------------------ refusals
def _gn_args(device, **kw):
    a = dict(x=torch.randn(2, 4, 4, 8, device=device), gamma=torch.ones(8, device=device), beta=torch.zeros(8, device=device), groups=2, eps=1e-5,
             mean=torch.empty(2, 2, device=device), rstd=torch.empty(2, 2, device=device))
    a["y"] = torch.empty_like(a["x"])
    a.update({k: v(a) if callable(v) else v for k, v in kw.items()})
    return a


def _gn_fwd(device, **kw):
    a = _gn_args(device, **kw)
    ops.group_norm_fwd(a["x"], a["gamma"], a["beta"], a["groups"], a["eps"], a["y"], a["mean"], a["rstd"], act=a.get("act", "none"), residual=a.get("res"))


def _gn_bwd(device, **kw):
    a = _gn_args(device, **kw)
    ops.group_norm_bwd(a.get("dy", torch.empty_like(a["x"])), a["x"], a["gamma"], a["beta"], a["groups"], a["mean"], a["rstd"], a.get("dx", torch.empty_like(a["x"])),
                       a.get("dg"), a.get("db"), act=a.get("act", "none"), y=a.get("yv"), residual=a.get("res"), dresidual=a.get("dres"))


def _lin(device, which, **kw):
    a = dict(x=torch.randn(4, 16, device=device), w=torch.randn(8, 16, device=device), y=torch.empty(4, 8, device=device), dy=torch.randn(4, 8, device=device),
             dx=torch.empty(4, 16, device=device), dw=torch.empty(8, 16, device=device))
    a.update({k: v(a) if callable(v) else v for k, v in kw.items()})
    if which == "f":
        ops.linear_fprop(a["x"], a["w"], a["y"], bias=a.get("bias"), act=a.get("act", "none"), addend=a.get("addend"), preact=a.get("preact"))
    elif which == "d":
        ops.linear_dgrad(a["dy"], a["w"], a["dx"], act=a.get("act", "none"), preact=a.get("preact"), addend=a.get("addend"))
    else:
        ops.linear_wgrad(a["dy"], a["x"], a["dw"], db=a.get("db"))


def _adamw(device, bits=32, lo=0, hi=None, **kw):
    n = 256
    a = dict(p=torch.zeros(n, device=device), g=torch.zeros(n, device=device), m=torch.zeros(n, device=device), v=torch.zeros(n, device=device), p16=None,
             hyper=make_hyper(1e-3, 0.9, 0.999, 1e-8, 0.0, 0.0, 0.0, 1.0, device=device), groups=torch.ones(1, 2, device=device),
             ids=torch.zeros(n // 64, dtype=torch.uint8, device=device), ms=torch.zeros(n // 64, device=device), vs=torch.zeros(n // 64, device=device))
    if bits == 8:
        a["m"], a["v"] = a["m"].to(torch.float8_e4m3fn), a["v"].to(torch.float8_e5m2)
    a.update(kw)
    if bits == 32:
        ops.adamw_step(a["p"], a["g"], a["m"], a["v"], a["p16"], a["hyper"], a["groups"], a["ids"], lo, hi)
    else:
        ops.adamw8_step(a["p"], a["g"], a["m"], a["v"], a["ms"], a["vs"], a["p16"], a["hyper"], a["groups"], a["ids"], 1, lo, hi)


REFUSALS = {
    "gn groups do not divide": lambda d: _gn_fwd(d, groups=3),
    "gn no groups": lambda d: _gn_fwd(d, groups=0),
    "gn type": lambda d: _gn_fwd(d, x=torch.randn(2, 4, 4, 8, device=d).half()),
    "gn mixed types": lambda d: _gn_fwd(d, y=torch.empty(2, 4, 4, 8, device=d, dtype=torch.bfloat16)),
    "gn shape of y": lambda d: _gn_fwd(d, y=torch.empty(2, 4, 5, 8, device=d)),
    "gn channels first": lambda d: _gn_fwd(d, x=torch.randn(2, 8, 4, 4, device=d).permute(0, 2, 3, 1)),
    "gn strided rows": lambda d: _gn_fwd(d, x=torch.randn(2, 8, 4, 8, device=d)[:, ::2]),
    "gn strided images": lambda d: _gn_fwd(d, x=torch.randn(4, 4, 4, 8, device=d)[::2]),
    "gn broadcast image": lambda d: _gn_fwd(d, x=torch.randn(1, 4, 4, 8, device=d).expand(2, 4, 4, 8)),
    "gn act": lambda d: _gn_fwd(d, act="tanh"),
    "gn gamma length": lambda d: _gn_fwd(d, gamma=torch.ones(7, device=d)),
    "gn gamma type": lambda d: _gn_fwd(d, gamma=torch.ones(8, device=d).bfloat16()),
    "gn mean length": lambda d: _gn_fwd(d, mean=torch.empty(2, device=d)),
    "gn no pixels": lambda d: _gn_fwd(d, x=torch.randn(2, 0, 4, 8, device=d), y=torch.empty(2, 0, 4, 8, device=d)),
    "gn shifted overlap": lambda d: (lambda b: _gn_fwd(d, x=b[:2], y=b[1:]))(torch.randn(3, 4, 4, 8, device=d)),
    "gn mask without relu": lambda d: _gn_bwd(d, act="silu", yv=lambda a: a["x"]),
    "gn dresidual is x": lambda d: _gn_bwd(d, res=torch.randn(2, 4, 4, 8, device=d), dres=lambda a: a["x"]),
    "gn dgamma length": lambda d: _gn_bwd(d, dg=torch.empty(9, device=d)),
    "gn dy shape": lambda d: _gn_bwd(d, dy=torch.empty(2, 4, 4, 16, device=d)),
    "linear inner size": lambda d: _lin(d, "f", w=torch.randn(8, 15, device=d)),
    "linear mixed types": lambda d: _lin(d, "f", w=torch.randn(8, 16, device=d).bfloat16()),
    "linear type": lambda d: _lin(d, "f", x=torch.randn(4, 16, device=d).half(), w=torch.randn(8, 16, device=d).half()),
    "linear columns not contiguous": lambda d: _lin(d, "f", x=torch.randn(16, 4, device=d).t()),
    "linear broadcast rows": lambda d: _lin(d, "f", x=torch.randn(1, 16, device=d).expand(4, 16)),
    "linear bias": lambda d: _lin(d, "f", bias=torch.randn(7, device=d)),
    "linear act": lambda d: _lin(d, "f", act="swish"),
    "linear preact shape": lambda d: _lin(d, "f", act="gelu", preact=torch.empty(4, 7, device=d)),
    "linear preact is y": lambda d: _lin(d, "f", act="gelu", preact=lambda a: a["y"]),
    "linear y is x": lambda d: _lin(d, "f", x=torch.randn(8, 8, device=d), w=torch.randn(8, 8, device=d), y=lambda a: a["x"]),
    "linear three dimensions": lambda d: _lin(d, "f", x=torch.randn(1, 4, 16, device=d)),
    "linear dgrad without preact": lambda d: _lin(d, "d", act="gelu"),
    "linear dgrad preact alone": lambda d: _lin(d, "d", preact=torch.randn(4, 16, device=d)),
    "linear dgrad inner size": lambda d: _lin(d, "d", dy=torch.randn(4, 9, device=d)),
    "linear wgrad rows": lambda d: _lin(d, "w", dy=torch.randn(5, 8, device=d)),
    "linear wgrad type of dw": lambda d: _lin(d, "w", dw=torch.empty(8, 16, device=d).bfloat16()),
    "linear wgrad db": lambda d: _lin(d, "w", db=torch.empty(16, device=d)),
    "adamw range": lambda d: _adamw(d, lo=32),
    "adamw range end": lambda d: _adamw(d, hi=320),
    "adamw arena size": lambda d: _adamw(d, p=torch.zeros(250, device=d), g=torch.zeros(250, device=d)),
    "adamw g size": lambda d: _adamw(d, g=torch.zeros(192, device=d)),
    "adamw p type": lambda d: _adamw(d, p=torch.zeros(256, device=d).bfloat16()),
    "adamw p16 type": lambda d: _adamw(d, p16=torch.zeros(256, device=d)),
    "adamw groups": lambda d: _adamw(d, groups=torch.ones(2, 3, device=d)),
    "adamw ids": lambda d: _adamw(d, ids=torch.zeros(3, dtype=torch.uint8, device=d)),
    "adamw ids type": lambda d: _adamw(d, ids=torch.zeros(4, dtype=torch.int64, device=d)),
    "adamw hyper": lambda d: _adamw(d, hyper=torch.zeros(8, device=d)),
    "adamw8 state type": lambda d: _adamw(d, bits=8, m=torch.zeros(256, dtype=torch.uint8, device=d)),
    "adamw8 scales": lambda d: _adamw(d, bits=8, ms=torch.zeros(5, device=d)),
}


def check_refusal(name, device):
    with pytest.raises(ValueError):
        REFUSALS[name](device)
