"""Cases for the group-norm, linear-product and AdamW operators: inputs, the plain form of each, and its definition in
64 bits.

Layouts are the framework's: activations [N, H, W, C] with the channels innermost, linear weights [out, in], optimizer
state in flat arenas whose tensors start at multiples of 64 elements."""
import math

import torch

own = False

BF16, FP32 = "bf16", "fp32"
_DTYPE = {BF16: torch.bfloat16, FP32: torch.float32}
BLOCK = 64            # arena alignment, and elements per scale of an 8-bit state
M_MAX, V_MAX = 448.0, 57344.0          # largest values of float8_e4m3fn and float8_e5m2
TINY = 2.0 ** -100    # a block whose largest magnitude is below this holds zeros
MASK32 = 0xFFFFFFFF


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the last stage's norm of one image that is being classified: pure latency
        _gn("gn_fwd_one_image", "fwd", BF16, 1, 7, 7, 512, 32, "relu", False),
        # block output of a residual network at batch 64: norm + residual + ReLU over 51 M elements
        _gn("gn_fwd_block", "fwd", BF16, 64, 56, 56, 256, 32, "relu", True),
        # its backward pass one stage deeper: input, residual and parameter gradients
        _gn("gn_bwd_block", "bwd", BF16, 64, 28, 28, 512, 32, "relu", True),
        # ragged images, channels that fill no vector, 32-bit training with a smooth activation
        _gn("gn_bwd_ragged_fp32", "bwd", FP32, 5, 33, 47, 90, 6, "silu", False),
        # classifier layer for a single image: weights are the traffic
        _lin("linear_fwd_one_row", "fwd", BF16, 1, 4096, 4096, "relu", False),
        # hidden layer of a block over many rows, the pre-activation kept for training
        _lin("linear_fwd_hidden", "fwd", BF16, 8192, 4096, 1024, "gelu", False),
        # the data gradient of the layer behind it, times the derivative of that layer's activation
        _lin("linear_dgrad_hidden", "dgrad", BF16, 8192, 1024, 4096, "gelu", False),
        # weight and bias gradient of the hidden layer
        _lin("linear_wgrad_hidden", "wgrad", BF16, 8192, 4096, 1024, "none", False),
        # 1000-class head in 32 bits with an odd batch and an addend
        _lin("linear_fwd_head_fp32", "fwd", FP32, 1021, 1000, 2048, "none", True),
        # optimizer step of a small convolutional network: a handful of tensors
        _opt("adamw32_small", 32, 8, 21840, 0),
        # optimizer step of a 25 M parameter network with its bf16 compute copy
        _opt("adamw32_25m", 32, 161, 25557032, 1),
        # 132 M parameters with both moments in 8 bits
        _opt("adamw8_132m", 8, 38, 132868840, 1),
    ]


def _gn(name, kind, dtype, n, h, w, c, groups, act, residual):
    return {"name": name, "op": "group_norm", "kind": kind, "dtype": dtype, "n": n, "h": h, "w": w, "c": c, "groups": groups,
            "act": act, "residual": residual}


def _lin(name, kind, dtype, rows, out, inp, act, addend):
    return {"name": name, "op": "linear", "kind": kind, "dtype": dtype, "rows": rows, "out": out, "in": inp, "act": act,
            "addend": addend}


def _opt(name, bits, tensors, params, p16):
    return {"name": name, "op": "adamw", "bits": bits, "tensors": tensors, "params": params, "p16": p16}


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["group_norm", "linear", "adamw"])
    if op == "group_norm":
        while True:
            h = _log_int(rng, 1, 112)
            w = h if rng.random() < 0.5 else _log_int(rng, 1, 112)
            cg, groups = _log_int(rng, 1, 64), rng.choice([1, 2, 3, 4, 6, 8, 16, 32])
            if rng.random() < 0.5:
                cg = max(8, cg // 8 * 8)
            n = _log_int(rng, 1, 256)
            if 2000 <= n * h * w * cg * groups <= 51_380_224 and h * w * cg > 1:
                break
        c = _gn("", rng.choice(["fwd", "bwd"]), rng.choice([BF16, FP32]), n, h, w, cg * groups, groups,
                rng.choice(["none", "relu", "silu", "gelu"]), rng.random() < 0.5)
    elif op == "linear":
        kind = rng.choice(["fwd", "dgrad", "wgrad"])
        dtype = rng.choice([BF16, BF16, FP32])
        most = 8192 * 4096 * 1024 if dtype == BF16 else 8192 * 4096 * 128
        while True:
            rows, out, inp = _log_int(rng, 1, 16384), _log_int(rng, 8, 8192), _log_int(rng, 8, 8192)
            if rng.random() < 0.6:
                out, inp = (out + 7) // 8 * 8, (inp + 7) // 8 * 8
            if 30_000 <= rows * out * inp <= most:
                break
        act = "none" if kind == "wgrad" else rng.choice(["none", "relu", "silu", "gelu"])
        c = _lin("", kind, dtype, rows, out, inp, act, kind != "wgrad" and rng.random() < 0.5)
    else:
        tensors = _log_int(rng, 1, 200)
        c = _opt("", rng.choice([8, 32]), tensors, _log_int(rng, max(1000, 16 * tensors), 100_000_000), rng.choice([0, 1]))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g = _generator(seed)
    return {"group_norm": _prepare_gn, "linear": _prepare_linear, "adamw": _prepare_adamw}[case["op"]](case, seed, g)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _prepare_gn(case, seed, g):
    dt = _DTYPE[case["dtype"]]
    n, h, w, c, groups = (case[k] for k in ("n", "h", "w", "c", "groups"))
    # convolution outputs: every channel has a mean and a spread of its own
    x = (_randn(g, n, h, w, c) * (0.5 + _rand(g, c)) + 0.5 * _randn(g, c)).to(dt)
    s = {"case": case, "x": x, "gamma": 0.5 + _rand(g, c), "beta": 0.3 * _randn(g, c), "eps": 1e-5,
         "res": _randn(g, n, h, w, c, dtype=dt) if case["residual"] else None}
    if case["kind"] == "bwd":
        # what the forward pass left behind: the statistics, and the output where the ReLU mask is taken from it
        mean, var = _moments(x, groups, torch.float64)
        s["mean"], s["rstd"] = mean.float(), torch.rsqrt(var + s["eps"]).float()
        s["dy"] = _randn(g, n, h, w, c, dtype=dt)
        s["y"] = None
        if case["act"] == "relu" and case["residual"]:
            s["y"] = _affine(s, torch.float32).clamp_min(0).to(dt)
    return s


def _prepare_linear(case, seed, g):
    dt = _DTYPE[case["dtype"]]
    m, n, k = case["rows"], case["out"], case["in"]
    s = {"case": case}
    if case["kind"] == "fwd":
        s["x"] = _randn(g, m, k, dtype=dt)
        s["w"] = (_randn(g, n, k) / math.sqrt(k)).to(dt)
        s["bias"] = 0.1 * _randn(g, n)
        s["addend"] = _randn(g, m, n, dtype=dt) if case["addend"] else None
    elif case["kind"] == "dgrad":
        s["dy"] = _randn(g, m, n, dtype=dt)
        s["w"] = (_randn(g, n, k) / math.sqrt(k)).to(dt)
        s["z"] = _randn(g, m, k, dtype=dt)
        s["addend"] = _randn(g, m, k, dtype=dt) if case["addend"] else None
    else:
        s["dy"] = _randn(g, m, n, dtype=dt)
        s["x"] = _randn(g, m, k, dtype=dt)
    return s


def _sizes(case, seed):
    """Tensor sizes that sum to about `params`: a few large weights, many small vectors."""
    import random
    r = random.Random(seed * 7 + case["tensors"])
    share = [math.exp(r.uniform(-6.0, 0.0)) for _ in range(case["tensors"])]
    total = sum(share)
    return [max(1, int(case["params"] * s / total)) for s in share]


def _prepare_adamw(case, seed, g):
    sizes = _sizes(case, 1)          # the layout is the network's: the same for every seed
    padded = [(s + BLOCK - 1) // BLOCK * BLOCK for s in sizes]
    n = sum(padded)
    blocks = torch.tensor([p // BLOCK for p in padded], device="cuda")
    size = torch.repeat_interleave(torch.tensor(sizes, device="cuda"), blocks)
    start = torch.repeat_interleave(torch.cumsum(blocks, 0) - blocks, blocks)
    first = (torch.arange(n // BLOCK, device="cuda") - start) * BLOCK
    live = ((first[:, None] + torch.arange(BLOCK, device="cuda")[None, :]) < size[:, None]).reshape(-1)
    # gradients of layers differ by orders of magnitude, and so do rows within a layer
    spread = torch.pow(10.0, -4.0 + 2.0 * _rand(g, n // BLOCK)).repeat_interleave(BLOCK) * live
    s = {"case": case, "p": 0.05 * _randn(g, n) * live, "g": _randn(g, n) * spread, "lr": 1e-3, "betas": (0.9, 0.999),
         "eps": 1e-8, "wd": 0.05, "step": 100, "seed": 1234 + seed}
    m, v = 0.3 * _randn(g, n) * spread, (0.3 + _rand(g, n)) * spread * spread
    # vectors (norms, biases: the small tensors) are not decayed, and the first tensor learns more slowly
    ids = torch.tensor([1 if z < 4096 else 2 if i == 0 else 0 for i, z in enumerate(sizes)], device="cuda")
    s["group_ids"] = torch.repeat_interleave(ids, blocks).to(torch.uint8)
    s["groups"] = torch.tensor([[1.0, 1.0], [1.0, 0.0], [0.5, 1.0]], device="cuda")
    s["hyper"] = _hyper(s)
    s["p16"] = s["p"].to(torch.bfloat16) if case["p16"] else None
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        half = torch.full((n,), 0.5, device="cuda")
        s["m"], s["m_scale"] = _to_codes(m, half, M_MAX, -6, 3, torch.float8_e4m3fn)
        s["v"], s["v_scale"] = _to_codes(v, half, V_MAX, -14, 2, torch.float8_e5m2)
    return s


def _hyper(s):
    """The framework's vector of hyper-parameters, on the device: lr, betas, eps, weight decay, steps done, momentum,
    gradient scale, 1 - betas, and the betas' low parts."""
    b1, b2 = s["betas"]
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    return torch.tensor([s["lr"], b1, b2, s["eps"], s["wd"], s["step"], 0.0, 1.0, 1.0 - b1, 1.0 - b2, b1 - f32(b1), b2 - f32(b2)],
                        dtype=torch.float32, device="cuda")


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "group_norm":
        return _plain_gn_fwd(state) if case["kind"] == "fwd" else _plain_gn_bwd(state)
    if case["op"] == "linear":
        return _plain_linear(state)
    return _plain_adamw(state)


def _run_own(s):
    from distributedpytorch_amd import ops
    c = s["case"]
    if c["op"] == "group_norm":
        x = s["x"]
        if c["kind"] == "fwd":
            y = torch.empty_like(x)
            mean, rstd = torch.empty(2, c["n"], c["groups"], device=x.device)
            ops.group_norm_fwd(x, s["gamma"], s["beta"], c["groups"], s["eps"], y, mean, rstd, act=c["act"], residual=s["res"])
            return y, mean, rstd
        dx, (dgamma, dbeta) = torch.empty_like(x), torch.empty(2, c["c"], device=x.device)
        dres = torch.empty_like(x) if c["residual"] else None
        ops.group_norm_bwd(s["dy"], x, s["gamma"], s["beta"], c["groups"], s["mean"], s["rstd"], dx, dgamma, dbeta, act=c["act"],
                           y=s["y"], residual=s["res"], dresidual=dres)
        return dx, dgamma, dbeta, dres
    if c["op"] == "linear":
        m, n, k = c["rows"], c["out"], c["in"]
        if c["kind"] == "fwd":
            x = s["x"]
            y = torch.empty(m, n, device=x.device, dtype=x.dtype)
            z = torch.empty_like(y) if c["act"] != "none" else None
            ops.linear_fprop(x, s["w"], y, bias=s["bias"], act=c["act"], addend=s["addend"], preact=z)
            return y, z
        dy = s["dy"]
        if c["kind"] == "dgrad":
            dx = torch.empty(m, k, device=dy.device, dtype=dy.dtype)
            ops.linear_dgrad(dy, s["w"], dx, act=c["act"], preact=s["z"] if c["act"] != "none" else None, addend=s["addend"])
            return dx
        dw, db = torch.empty(n, k, device=dy.device), torch.empty(n, device=dy.device)
        ops.linear_wgrad(dy, s["x"], dw, db=db)
        return dw, db
    if c["bits"] == 32:
        ops.adamw_step(s["p"], s["g"], s["m"], s["v"], s["p16"], s["hyper"], s["groups"], s["group_ids"])
        return s["p"], s["p16"], s["m"], s["v"]
    ops.adamw8_step(s["p"], s["g"], s["m"], s["v"], s["m_scale"], s["v_scale"], s["p16"], s["hyper"], s["groups"], s["group_ids"],
                    s["seed"])
    return s["p"], s["p16"], s["m"], s["v"], s["m_scale"], s["v_scale"]


# ------------------------------------------------------------------------------------------------ plain forms
def _act(u, name):
    if name == "relu":
        return u.clamp_min(0)
    if name == "silu":
        return u * torch.sigmoid(u)
    if name == "gelu":
        return 0.5 * u * (1 + torch.erf(u * math.sqrt(0.5)))
    return u


def _act_slope(u, name):
    if name == "relu":
        return (u > 0).to(u.dtype)
    if name == "silu":
        s = torch.sigmoid(u)
        return s * (1 + u * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(u * math.sqrt(0.5))) + u * torch.exp(-0.5 * u * u) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(u)


def _moments(x, groups, dtype):
    n, h, w, c = x.shape
    t = x.to(dtype).reshape(n, h * w, groups, c // groups)
    mean = t.mean((1, 3))
    d = t - mean[:, None, :, None]
    return mean, (d * d).mean((1, 3))


def _normed(x, mean, rstd, groups):
    n, h, w, c = x.shape
    t = x.to(mean.dtype).reshape(n, h * w, groups, c // groups)
    return ((t - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(n, h, w, c)


def _affine(s, dtype):
    """The values in front of the activation, from saved statistics."""
    u = _normed(s["x"], s["mean"].to(dtype), s["rstd"].to(dtype), s["case"]["groups"]) * s["gamma"].to(dtype) + s["beta"].to(dtype)
    return u if s["res"] is None else u + s["res"].to(dtype)


def _plain_gn_fwd(s):
    c = s["case"]
    mean, var = _moments(s["x"], c["groups"], torch.float32)
    rstd = torch.rsqrt(var + s["eps"])
    u = _affine({**s, "mean": mean, "rstd": rstd}, torch.float32)
    return _act(u, c["act"]).to(s["x"].dtype), mean, rstd


def _plain_gn_bwd(s):
    c, x = s["case"], s["x"]
    n, h, w, ch = x.shape
    g, dt = c["groups"], x.dtype
    xhat = _normed(x, s["mean"], s["rstd"], g)
    dy = s["dy"].float()
    if c["act"] == "relu":
        # the border of the mask: the stored output where there is one, else the sign in 64 bits
        dz = dy * ((s["y"] if s["y"] is not None else _affine(s, torch.float64)) > 0)
    elif c["act"] != "none":
        dz = dy * _act_slope(_affine(s, torch.float32), c["act"])
    else:
        dz = dy
    dbeta, dgamma = dz.sum((0, 1, 2)), (dz * xhat).sum((0, 1, 2))
    t = (dz * s["gamma"]).reshape(n, h * w, g, ch // g)
    xh = xhat.reshape(t.shape)
    dx = (t - t.mean((1, 3), keepdim=True) - xh * (t * xh).mean((1, 3), keepdim=True)) * s["rstd"][:, None, :, None]
    return dx.reshape(x.shape).to(dt), dgamma, dbeta, dz.to(dt) if c["residual"] else None


def _plain_linear(s):
    c = s["case"]
    if c["kind"] == "fwd":
        u = s["x"].float() @ s["w"].float().t() + s["bias"]
        if s["addend"] is not None:
            u = u + s["addend"].float()
        dt = s["x"].dtype
        return _act(u, c["act"]).to(dt), u.to(dt) if c["act"] != "none" else None
    if c["kind"] == "dgrad":
        d = s["dy"].float() @ s["w"].float()
        if s["addend"] is not None:
            d = d + s["addend"].float()
        return (d * _act_slope(s["z"].float(), c["act"])).to(s["dy"].dtype)
    dy = s["dy"].float()
    return dy.t() @ s["x"].float(), dy.sum(0)


def _random16(seed, step, n):
    """Two 16-bit numbers for each element: the finalizer of MurmurHash3 over its index and a key of (seed, step)."""
    def mix(h):
        h = h ^ (h >> 16)
        h = (h * 0x85EBCA6B) & MASK32
        h = h ^ (h >> 13)
        h = (h * 0xC2B2AE35) & MASK32
        return h ^ (h >> 16)
    key = mix(torch.tensor((seed + step * 0x9E3779B9) & MASK32, device="cuda"))
    h = mix(torch.arange(n, device="cuda") ^ key)
    return h & 0xFFFF, h >> 16


def _to_codes(t, u, top, least, bits, dtype):
    """t in blocks of 64 as 8-bit floats times a scale, stochastically rounded with u in (0, 1)."""
    b = t.reshape(-1, BLOCK)
    most = torch.where(torch.isfinite(b), b.abs(), torch.zeros_like(b)).amax(1, keepdim=True)
    some = most >= TINY
    y = torch.nan_to_num(b.abs() * torch.where(some, top / most, torch.zeros_like(most)), nan=top, posinf=top)
    e = (torch.frexp(y).exponent - 1).clamp_min(least)
    q = torch.ldexp(torch.floor(torch.ldexp(y, bits - e) + u.reshape(b.shape)), e - bits).clamp_max(top)
    if dtype == torch.float8_e5m2:          # a second moment that is not zero does not become zero
        q = torch.where((b > 0) & some, q.clamp_min(2.0 ** (least - bits)), q)
    q = torch.copysign(q, b).reshape(-1)
    return q.to(dtype), torch.where(some, most / top, torch.zeros_like(most)).reshape(-1).float()


def _plain_adamw(s):
    c, p = s["case"], s["p"]
    (b1, b2), t = s["betas"], s["step"] + 1
    per = s["groups"][s["group_ids"].long()].repeat_interleave(BLOCK, 0)
    if c["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = s["m"].float() * s["m_scale"].repeat_interleave(BLOCK)
        v = s["v"].float() * s["v_scale"].repeat_interleave(BLOCK)
    m = m + (1 - b1) * (s["g"] - m)
    v = b2 * v + (1 - b2) * s["g"] * s["g"]
    lr = s["lr"] * per[:, 0]
    denom = v.sqrt() / math.sqrt(1 - b2 ** t) + s["eps"]
    s["p"].copy_(p * (1 - lr * s["wd"] * per[:, 1]) - lr / (1 - b1 ** t) * m / denom)
    if s["p16"] is not None:
        s["p16"].copy_(s["p"])
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return s["p"], s["p16"], s["m"], s["v"]
    rm, rv = _random16(s["seed"], s["step"], p.numel())
    s["m"], s["m_scale"] = _to_codes(m, (rm.float() + 0.5) / 65536, M_MAX, -6, 3, torch.float8_e4m3fn)
    s["v"], s["v_scale"] = _to_codes(v, (rv.float() + 0.5) / 65536, V_MAX, -14, 2, torch.float8_e5m2)
    return s["p"], s["p16"], s["m"], s["v"], s["m_scale"], s["v_scale"]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    es = 2 if case.get("dtype") == BF16 else 4
    if case["op"] == "group_norm":
        n, c = case["n"] * case["h"] * case["w"] * case["c"], case["c"]
        stats = 8 * case["n"] * case["groups"]
        if case["kind"] == "fwd":
            return {"bytes": n * es * (2 + int(case["residual"])) + 8 * c + stats, "flops": 8 * n}
        # with a residual: either it or the stored output is read, and its gradient is written
        extra = 0 if not case["residual"] else 1 if case["act"] == "none" else 2
        return {"bytes": n * es * (3 + extra) + 16 * c + stats, "flops": 16 * n}
    if case["op"] == "linear":
        m, n, k = case["rows"], case["out"], case["in"]
        if case["kind"] == "fwd":
            outs = 1 + int(case["act"] != "none") + int(case["addend"])
            b = es * (m * k + n * k + outs * m * n) + 4 * n
        elif case["kind"] == "dgrad":
            outs = 1 + int(case["act"] != "none") + int(case["addend"])
            b = es * (m * n + n * k + outs * m * k)
        else:
            b = es * (m * n + m * k) + 4 * n * k + 4 * n
        return {"bytes": b, "flops": 2 * m * n * k}
    n = sum((s + BLOCK - 1) // BLOCK * BLOCK for s in _sizes(case, 1))
    state = 16.0 if case["bits"] == 32 else 4.0 + 16.0 / BLOCK
    return {"bytes": n * (12.0 + state + 2.0 * case["p16"] + 1.0 / BLOCK), "flops": 16 * n}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    D = torch.float64
    if case["op"] == "group_norm":
        return _exact_gn(s, case, D)
    if case["op"] == "linear":
        if case["kind"] == "wgrad":
            return torch.mm(s["dy"].to(D).t().contiguous(), s["x"].to(D)), s["dy"].sum(0, dtype=D)
        a = s["addend"].to(D) if s["addend"] is not None else 0.0
        if case["kind"] == "fwd":
            z = torch.mm(s["x"].to(D), s["w"].to(D).t().contiguous()) + s["bias"].to(D) + a
            return _phi(z, case["act"])[0], z if case["act"] != "none" else None
        return (torch.mm(s["dy"].to(D), s["w"].to(D)) + a) * _phi(s["z"].to(D), case["act"])[1]
    return _exact_adamw(s, case, D)


def _phi(z, name):
    """(activation, its derivative)."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        on = z > 0
        return torch.where(on, z, torch.zeros_like(z)), on.to(z.dtype)
    if name == "silu":
        e = 1.0 / (1.0 + torch.exp(-z))
        return z * e, e + z * e * (1.0 - e)
    cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
    return z * cdf, cdf + z * torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi)


def _exact_gn(s, case, D):
    n, c, g = case["n"], case["c"], case["groups"]
    px = case["h"] * case["w"]
    # [n, groups, elements of the group]: the channels of a group in front, then the pixels
    by_group = lambda t: t.to(D).reshape(n, px, c).transpose(1, 2).reshape(n, g, -1)  # noqa: E731
    back = lambda t: t.reshape(n, c, px).transpose(1, 2).reshape(s["x"].shape)  # noqa: E731
    weight = s["gamma"].to(D).repeat_interleave(px).reshape(1, g, -1)
    shift = s["beta"].to(D).repeat_interleave(px).reshape(1, g, -1)
    x = by_group(s["x"])
    if case["kind"] == "fwd":
        mu = x.sum(2) / x.shape[2]
        var = (x - mu.unsqueeze(2)).square().sum(2) / x.shape[2]
        inv = (var + s["eps"]).sqrt().reciprocal()
    else:
        mu, inv = s["mean"].to(D), s["rstd"].to(D)
    hat = (x - mu.unsqueeze(2)) * inv.unsqueeze(2)
    z = hat * weight + shift
    if s["res"] is not None:
        z = z + by_group(s["res"])
    if case["kind"] == "fwd":
        return back(_phi(z, case["act"])[0]), mu, inv
    slope = (by_group(s["y"]) > 0).to(D) if s["y"] is not None else _phi(z, case["act"])[1]
    dz = by_group(s["dy"]) * slope
    dgamma = (dz * hat).reshape(n, c, px).sum((0, 2))
    dbeta = dz.reshape(n, c, px).sum((0, 2))
    d = dz * weight
    m = x.shape[2]
    dx = inv.unsqueeze(2) * (d - (d.sum(2, keepdim=True) + hat * (d * hat).sum(2, keepdim=True)) / m)
    return back(dx), dgamma, dbeta, back(dz) if case["residual"] else None


def _exact_adamw(s, case, D):
    b1, b2 = s["betas"]
    t = s["step"] + 1
    n = s["p"].numel()
    rows = lambda v: v.reshape(-1, BLOCK)  # noqa: E731
    g, p = rows(s["g"]).to(D), rows(s["p"]).to(D)
    kind = s["groups"][s["group_ids"].long()].to(D)
    lr = s["lr"] * kind[:, :1]
    m, v = rows(s["m"]).to(D), rows(s["v"]).to(D)
    if case["bits"] == 8:
        m, v = m * s["m_scale"].to(D)[:, None], v * s["v_scale"].to(D)[:, None]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g.square()
    upd = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + s["eps"])
    p = (p - lr * s["wd"] * kind[:, 1:] * p - lr * upd).reshape(-1)
    p16 = p if s["p16"] is not None else None
    if case["bits"] == 32:
        return p, p16, m.reshape(-1), v.reshape(-1)
    rm, rv = _random16(s["seed"], s["step"], n)
    out = []
    for val, r, top, low, bits in ((m, rm, 448.0, -6, 3), (v, rv, 57344.0, -14, 2)):
        big = val.abs().amax(1, keepdim=True)
        keep = big >= TINY
        y = torch.where(keep, val.abs() / big.clamp_min(TINY) * top, torch.zeros_like(val))
        grid = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** low))) - bits)
        code = (torch.floor(y / grid + (rows(r).to(D) + 0.5) / 65536.0) * grid).clamp_max(top)
        if bits == 2:
            code = torch.where((val > 0) & keep, code.clamp_min(2.0 ** (low - bits)), code)
        out.append(((code * torch.sign(val)).reshape(-1), torch.where(keep, big / top, torch.zeros_like(big)).reshape(-1)))
    return p, p16, out[0][0], out[1][0], out[0][1], out[1][1]
