"""Definitions of the group-norm, linear and AdamW operators in 64 bits, and error bounds counted from the arithmetic.

E is half a step of fp32 (2^-24).  Where a bound is L * E * (sum of magnitudes), L counts the roundings on the longest path
from an input to the output: L_STAT for a mean or a sum over a group (partial sums of at most a few hundred terms, joined
pairwise), L_POINT for the elementwise chain behind it."""
import math

import torch

D = torch.float64
E = 2.0 ** -24
L_POINT, L_STAT = 32, 512
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def phi(u, act):
    """(act(u), act'(u))"""
    if act == "relu":
        return u.clamp_min(0), (u > 0).to(D)
    if act == "silu":
        s = torch.sigmoid(u)
        return u * s, s * (1 + u * (1 - s))
    if act == "gelu":
        c = 0.5 * torch.erfc(-u / math.sqrt(2))
        return u * c, c + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)
    return u, torch.ones_like(u)


def close(name, got, want, err, dtype=torch.float32):
    """|got - want| <= err + half a step of the output type (and equal where want is not finite)."""
    got, want = got.detach().cpu().to(D), want.cpu().to(D)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN in other places"
    inf = ~fin & ~torch.isnan(want)
    assert torch.equal(got[inf], want[inf]), f"{name}: infinities differ"
    tol = (err.cpu() if torch.is_tensor(err) else torch.full_like(want, err)).to(D).expand_as(want) * (1 + 2 * HALF_STEP[dtype])
    tol = tol + HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -20) + 1e-37
    bad = ((got - want).abs() > tol) & fin
    if bad.any():
        i = int(((got - want).abs() / tol * fin).nan_to_num(0).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside the bound; worst at {i}: got {got.reshape(-1)[i]!r}, "
                             f"want {want.reshape(-1)[i]!r}, bound {tol.reshape(-1)[i]!r}")


def grouped(t, g):
    n, h, w, c = t.shape
    return t.to(D).reshape(n, h * w, g, c // g)


def gn_forward(x, gamma, beta, groups, eps, act, res):
    """y, mean, rstd, and the bounds of y, mean, rstd"""
    t = grouped(x, groups)
    mean = t.mean((1, 3))
    d = t - mean[:, None, :, None]
    var = (d * d).mean((1, 3))
    rstd = 1 / (var + eps).sqrt()
    size = t.abs().mean((1, 3))                                    # error of the mean, relative to the mean magnitude
    e_mean = L_STAT * E * size
    # the second moment is centred at a rounded mean: (e_mean)^2 more, and L_STAT roundings of its own
    e_rstd = rstd * (L_STAT * E + 0.5 * (e_mean * rstd) ** 2 + L_POINT * E)
    a = (d * rstd[:, None, :, None]).reshape(x.shape) * gamma.to(D)
    u = a + beta.to(D) + (res.to(D) if res is not None else 0)
    y, slope = phi(u, act)
    mag = a.abs() + beta.to(D).abs() + (res.to(D).abs() if res is not None else 0)
    e_u = L_POINT * E * mag + a.abs() * _per(e_rstd / rstd, x, groups) + gamma.to(D).abs() * _per((e_mean + L_POINT * E * mean.abs()) * rstd, x, groups)
    return y, mean, rstd, 1.2 * e_u + L_POINT * E * (1 + u.abs()) * (act in ("silu", "gelu")), e_mean, e_rstd


def _per(t, x, groups):
    n, h, w, c = x.shape
    return t.reshape(n, 1, groups, 1).expand(n, h * w, groups, c // groups).reshape(x.shape)


def gn_backward(dy, x, gamma, beta, groups, mean, rstd, act, y, res):
    """dx, dgamma, dbeta, dres and their bounds, from the given (rounded) statistics"""
    mu, rs = mean.to(D).reshape(-1, 1, groups, 1), rstd.to(D).reshape(-1, 1, groups, 1)
    xh = (grouped(x, groups) - mu) * rs
    xhat = xh.reshape(x.shape)
    e_hat = L_POINT * E * (xhat.abs() + _per((mean.to(D) * rstd.to(D)).abs(), x, groups))
    u = xhat * gamma.to(D) + beta.to(D) + (res.to(D) if res is not None else 0)
    slope = (y.to(D) > 0).to(D) if y is not None else phi(u, act)[1]
    dz = dy.to(D) * slope
    mag = (xhat * gamma.to(D)).abs() + beta.to(D).abs() + (res.to(D).abs() if res is not None else 0)
    smooth = act in ("silu", "gelu")
    e_dz = dy.to(D).abs() * (L_POINT * E * (2 + 2 * mag) + gamma.to(D).abs() * e_hat) * smooth + E * dz.abs()
    dg, db = (dz * xhat), dz
    t = grouped(dz * gamma.to(D), groups)
    c1, c2 = t.mean((1, 3), keepdim=True), (t * xh).mean((1, 3), keepdim=True)
    dx = (rs * (t - c1 - xh * c2)).reshape(x.shape)
    e_t = grouped(e_dz * gamma.to(D).abs(), groups) + E * t.abs()
    e_h = grouped(e_hat, groups)
    e_c1 = (L_STAT * E * t.abs() + e_t).mean((1, 3), keepdim=True)
    e_c2 = (L_STAT * E * (t * xh).abs() + e_t * xh.abs() + t.abs() * e_h).mean((1, 3), keepdim=True)
    e_dx = rs * (e_t + e_c1 + xh.abs() * e_c2 + e_h * c2.abs() + L_POINT * E * (t.abs() + c1.abs() + (xh * c2).abs()))
    s = (0, 1, 2)
    return (dx, dg.sum(s), db.sum(s), dz), (e_dx.reshape(x.shape), (L_STAT * E * dg.abs() + e_dz * xhat.abs() + dz.abs() * e_hat).sum(s),
                                            (L_STAT * E * db.abs() + e_dz).sum(s), e_dz)


def product(a, b):
    """a b^T in 64 bits and the bound of its fp32 evaluation: every one of the K additions rounds, and an operand split into
    three bf16 parts loses products below 2^-23 of the term."""
    k = a.shape[1]
    return a.to(D) @ b.to(D).t(), (k + 16) * E * (a.to(D).abs() @ b.to(D).abs().t())


def adamw(p, g, m, v, hyper_args, per):
    """p', m', v' in 64 bits"""
    lr, b1, b2, eps, wd, step, gs = hyper_args
    t = step + 1
    g, p, m, v = (q.to(D) for q in (g, p, m, v))
    g = g * gs
    lrs, wds = lr * per[:, 0].to(D), wd * per[:, 1].to(D)
    m2 = m + (1 - b1) * (g - m)
    v2 = b2 * v + (1 - b2) * g * g
    upd = lrs / (1 - b1 ** t) * m2 / (v2.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    return p * (1 - lrs * wds) - upd, m2, v2, upd
