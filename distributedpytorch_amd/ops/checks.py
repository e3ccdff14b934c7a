"""Argument checks shared by the GPU and the CPU form of the group-norm, linear and AdamW operators: everything a kernel
assumes about shapes, types, layouts and devices is checked here, on the host, before anything is launched.

A checked tensor comes back as (address, stride, end of its bytes): what the launch needs, and what decides whether an output
overlaps an input.  An output may BE an input (same first element, same strides): every kernel here reads an element before
it writes it; a shifted overlap would be read after it was written."""
from __future__ import annotations

import torch

ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}          # ids of csrc/hip/act.h
FLOATS = (torch.float32, torch.bfloat16)
NOTHING = (0, 0, 0)
TOO_LARGE = 1 << 30


def act_id(act):
    i = ACTS.get(act)
    if i is None:
        raise ValueError(f"act must be one of {tuple(ACTS)}, got {act!r}")
    return i


def _like(t, name, shape, dtype, device):
    if t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the first operand on {device}")
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")


def vec32(t, name, n, device):
    """fp32 vector of n contiguous values -> its address"""
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name}: expected {n} contiguous fp32 values, got {tuple(t.shape)} {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the first operand on {device}")
    return t.data_ptr()


def nhwc(t, name):
    """NHWC tensor, possibly a channel slice of a wider one -> (address, elements from pixel to pixel, end)"""
    s, st = t.shape, t.stride()
    if len(s) != 4 or (st[3] != 1 and s[3] > 1):
        raise ValueError(f"{name}: expected an NHWC tensor with contiguous channels, got {tuple(s)} / {st}")
    n, h, w, c = s
    cs = st[2] if w > 1 else st[1] if h > 1 else st[0] if n > 1 else c
    if (h > 1 and st[1] != w * cs) or (n > 1 and st[0] != h * w * cs):
        raise ValueError(f"{name}: only channel slices of NHWC tensors are supported, got {tuple(s)} / {st}")
    if cs < c:
        raise ValueError(f"{name}: pixels overlap (channel stride {cs} < {c} channels)")
    p = t.data_ptr()
    return p, cs, p + ((n * h * w - 1) * cs + c) * t.element_size() if n * h * w else p


def nhwc_like(t, name, x):
    _like(t, name, x.shape, x.dtype, x.device)
    return nhwc(t, name)


def mat(t, name):
    """Matrix with contiguous rows -> (address, elements from row to row, end)"""
    s, st = t.shape, t.stride()
    if len(s) != 2 or (st[1] != 1 and s[1] > 1):
        raise ValueError(f"{name}: expected a matrix with contiguous rows, got {tuple(s)} / {st}")
    r, c = s
    if r >= TOO_LARGE or c >= TOO_LARGE:
        raise ValueError(f"{name}: {tuple(s)} is larger than a launch can index")
    ld = st[0] if r > 1 else c
    if ld < c:
        raise ValueError(f"{name}: rows overlap (stride {ld} < {c} columns)")
    p = t.data_ptr()
    return p, ld, p + ((r - 1) * ld + c) * t.element_size() if r else p


def mat_like(t, name, shape, dtype, device):
    _like(t, name, shape, dtype, device)
    return mat(t, name)


def apart(name, key, out, span, others):
    """others: (name, tensor, span, may be the output itself)"""
    a, b = span[0], span[2]
    for k, t, s, same in others:
        if t is None or not (a < s[2] and s[0] < b):
            continue
        if s[0] == a and t.stride() == out.stride() and t.shape == out.shape:
            if same:
                continue
            raise ValueError(f"{name}: {key} may not be {k}")
        if not _slices_apart(out, t):
            raise ValueError(f"{name}: {key} overlaps {k} without being the same tensor")


def _slices_apart(a, b):
    """Channel (or column) slices of one wider buffer that touch no common element."""
    if a.dim() != b.dim() or a.element_size() != b.element_size() or a.stride() != b.stride():
        return False
    row = next((st for s, st in zip(reversed(a.shape[:-1]), reversed(a.stride()[:-1])) if s > 1), 0)
    off = (b.data_ptr() - a.data_ptr()) // a.element_size() % row if row else 0
    return row > 0 and a.shape[-1] <= off <= row - b.shape[-1]


# ------------------------------------------------------------------------------------------------ group norm
def group_norm(name, x, gamma, beta, groups, mean, rstd):
    """x's (address, pixel stride, end) and the addresses of the vectors"""
    if x.dtype not in FLOATS:
        raise ValueError(f"{name}: x must be fp32 or bf16, got {x.dtype}")
    xs = nhwc(x, f"{name}: x")
    n, h, w, c = x.shape
    if groups < 1 or c < 1 or c % groups:
        raise ValueError(f"{name}: {c} channels do not divide into {groups} groups")
    if n and h * w == 0:
        raise ValueError(f"{name}: images without pixels have no statistics ({tuple(x.shape)})")
    if h * w >= TOO_LARGE or n * groups >= TOO_LARGE or c >= 1 << 20:
        raise ValueError(f"{name}: {tuple(x.shape)} is larger than a launch can index")
    d = x.device
    return (xs, vec32(gamma, f"{name}: gamma", c, d), vec32(beta, f"{name}: beta", c, d),
            vec32(mean, f"{name}: mean", n * groups, d), vec32(rstd, f"{name}: rstd", n * groups, d))


def group_norm_fwd(x, gamma, beta, groups, y, mean, rstd, act, residual):
    name = "group_norm_fwd"
    a = act_id(act)
    xs, *vecs = group_norm(name, x, gamma, beta, groups, mean, rstd)
    ys = nhwc_like(y, "group_norm_fwd: y", x)
    rs = NOTHING if residual is None else nhwc_like(residual, "group_norm_fwd: residual", x)
    apart(name, "y", y, ys, (("x", x, xs, True), ("residual", residual, rs, True)))
    return a, xs, ys, rs, vecs


def group_norm_bwd(dy, x, gamma, beta, groups, mean, rstd, dx, dgamma, dbeta, act, y, residual, dresidual):
    name = "group_norm_bwd"
    a = act_id(act)
    xs, *vecs = group_norm(name, x, gamma, beta, groups, mean, rstd)
    dys, dxs = nhwc_like(dy, "group_norm_bwd: dy", x), nhwc_like(dx, "group_norm_bwd: dx", x)
    ys = NOTHING if y is None else nhwc_like(y, "group_norm_bwd: y", x)
    rs = NOTHING if residual is None else nhwc_like(residual, "group_norm_bwd: residual", x)
    drs = NOTHING if dresidual is None else nhwc_like(dresidual, "group_norm_bwd: dresidual", x)
    if y is not None and a != 1:
        raise ValueError(f"{name}: y is the mask of a ReLU; act is {act!r}")
    for k, t in (("dgamma", dgamma), ("dbeta", dbeta)):
        vecs.append(0 if t is None else vec32(t, f"{name}: {k}", x.shape[3], x.device))
    apart(name, "dx", dx, dxs, (("dy", dy, dys, True), ("x", x, xs, True), ("y", y, ys, True), ("residual", residual, rs, True)))
    if dresidual is not None:          # x is read again after dresidual was written
        apart(name, "dresidual", dresidual, drs, (("dy", dy, dys, True), ("y", y, ys, True), ("residual", residual, rs, True),
                                                  ("x", x, xs, False), ("dx", dx, dxs, False)))
    return a, xs, dys, dxs, ys, rs, drs, vecs


def group_norm_overlaps(name):
    return ValueError(f"{name}: mean, rstd, dgamma or dbeta overlaps another argument, or an output overlaps gamma, beta, mean or rstd")


def group_norm_vectors(name, outs, maps_out, vecs, maps):
    """What csrc/hip/group_norm.hip: gn_overlap tests on the GPU, for the CPU form.  outs and vecs: vectors that are written and read;
    maps_out and maps: spans of activations; None or NOTHING where there is none."""
    spans = lambda ts: [(t.data_ptr(), t.data_ptr() + 4 * t.numel()) for t in ts if t is not None]  # noqa: E731
    outs, vecs, maps_out, maps = spans(outs), spans(vecs), [(s[0], s[2]) for s in maps_out], [(s[0], s[2]) for s in maps]
    pairs = [(a, b) for i, a in enumerate(outs) for b in outs[i + 1:] + vecs + maps_out + maps] + [(a, b) for a in maps_out for b in vecs]
    if any(a[0] < b[1] and b[0] < a[1] for a, b in pairs):
        raise group_norm_overlaps(name)


# ------------------------------------------------------------------------------------------------ linear
def linear_fprop(x, w, y, bias, act, addend, preact):
    """act's id, the spans of x, w, y, addend, preact, the address of bias"""
    name, dt, dev = "linear_fprop", x.dtype, x.device
    if dt not in FLOATS:
        raise ValueError(f"{name}: x must be fp32 or bf16, got {dt}")
    a, xs = act_id(act), mat(x, "linear_fprop: x")
    m, k = x.shape
    n = w.shape[0] if w.dim() == 2 else 0
    ws = mat_like(w, "linear_fprop: w", (n, k), dt, dev)
    if n < 1 or k < 1:
        raise ValueError(f"{name}: weight of shape {tuple(w.shape)}")
    shape = (m, n)
    ys = mat_like(y, "linear_fprop: y", shape, dt, dev)
    ads = NOTHING if addend is None else mat_like(addend, "linear_fprop: addend", shape, dt, dev)
    zs = NOTHING if preact is None else mat_like(preact, "linear_fprop: preact", shape, dt, dev)
    b = 0 if bias is None else vec32(bias, "linear_fprop: bias", n, dev)
    if b and (ys[0] - 4 * n < b < ys[2] or zs[0] - 4 * n < b < zs[2]):
        raise ValueError(f"{name}: y or preact overlaps bias")
    apart(name, "y", y, ys, (("addend", addend, ads, True), ("x", x, xs, False), ("w", w, ws, False)))
    if preact is not None:
        apart(name, "preact", preact, zs, (("addend", addend, ads, True), ("x", x, xs, False), ("w", w, ws, False), ("y", y, ys, False)))
    return a, xs, ws, ys, ads, zs, b


def linear_dgrad(dy, w, dx, act, preact, addend):
    """act's id, the spans of dy, w, dx, preact, addend"""
    name, dt, dev = "linear_dgrad", dy.dtype, dy.device
    if dt not in FLOATS:
        raise ValueError(f"{name}: dy must be fp32 or bf16, got {dt}")
    a, dys = act_id(act), mat(dy, "linear_dgrad: dy")
    m, n = dy.shape
    k = w.shape[1] if w.dim() == 2 else 0
    ws = mat_like(w, "linear_dgrad: w", (n, k), dt, dev)
    if n < 1 or k < 1:
        raise ValueError(f"{name}: weight of shape {tuple(w.shape)}")
    if (preact is None) == (a != 0):
        raise ValueError(f"{name}: act {act!r} " + ("needs preact" if a else "takes no preact"))
    shape = (m, k)
    dxs = mat_like(dx, "linear_dgrad: dx", shape, dt, dev)
    zs = NOTHING if preact is None else mat_like(preact, "linear_dgrad: preact", shape, dt, dev)
    ads = NOTHING if addend is None else mat_like(addend, "linear_dgrad: addend", shape, dt, dev)
    apart(name, "dx", dx, dxs, (("preact", preact, zs, True), ("addend", addend, ads, True), ("dy", dy, dys, False), ("w", w, ws, False)))
    return a, dys, ws, dxs, zs, ads


def linear_wgrad(dy, x, dw, db):
    """The spans of dy, x, dw, the address of db"""
    name, dt, dev = "linear_wgrad", dy.dtype, dy.device
    if dt not in FLOATS:
        raise ValueError(f"{name}: dy must be fp32 or bf16, got {dt}")
    dys = mat(dy, "linear_wgrad: dy")
    m, n = dy.shape
    k = x.shape[1] if x.dim() == 2 else 0
    xs = mat_like(x, "linear_wgrad: x", (m, k), dt, dev)
    if n < 1 or k < 1:
        raise ValueError(f"{name}: no columns ({tuple(dy.shape)}, {tuple(x.shape)})")
    dws = mat_like(dw, "linear_wgrad: dw", (n, k), torch.float32, dev)
    b = 0 if db is None else vec32(db, "linear_wgrad: db", n, dev)
    apart(name, "dw", dw, dws, (("dy", dy, dys, False), ("x", x, xs, False)))
    if b and (dws[0] - 4 * n < b < dws[2] or dys[0] - 4 * n < b < dys[2] or xs[0] - 4 * n < b < xs[2]):
        raise ValueError(f"{name}: db overlaps dw, dy or x")
    return dys, xs, dws, b


# ------------------------------------------------------------------------------------------------ AdamW
ARENA_BLOCK = 64


def _arena(t, name, key, dtype, n, device):
    if t.dtype != dtype or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name}: {key} must hold {n} contiguous values of {dtype}, got {tuple(t.shape)} {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: {key} is on {t.device}, p on {device}")
    p = t.data_ptr()
    if p % 16:
        raise ValueError(f"{name}: {key} must be 16-byte aligned")
    return p


def adamw(name, p, g, p16, hyper, groups, group_ids, lo, hi, states):
    """The element range [lo, hi) of an arena, both multiples of 64 -> hi, the addresses of p, g, p16, hyper, groups, group_ids
    and the states (name, tensor, dtype, elements)"""
    n, dev = p.numel(), p.device
    hi = n if hi is None else hi
    if n % ARENA_BLOCK or lo % ARENA_BLOCK or hi % ARENA_BLOCK or not 0 <= lo <= hi <= n:
        raise ValueError(f"{name}: [{lo}, {hi}) of {n} elements: ranges are multiples of {ARENA_BLOCK} inside the arena")
    at = [_arena(p, name, "p", torch.float32, n, dev), _arena(g, name, "g", torch.float32, n, dev),
          0 if p16 is None else _arena(p16, name, "p16", torch.bfloat16, n, dev)]
    if hyper.dtype != torch.float32 or hyper.numel() != 12 or not hyper.is_contiguous() or hyper.device != dev:
        raise ValueError(f"{name}: hyper must be the optimizer's vector of 12 fp32 values, on {dev}")
    if (groups.dtype != torch.float32 or groups.dim() != 2 or groups.shape[1] != 2 or not 1 <= groups.shape[0] <= 256
            or not groups.is_contiguous() or groups.device != dev or groups.data_ptr() % 8):
        raise ValueError(f"{name}: groups must be fp32 [1..256, 2] (lr multiplier, decay multiplier), on {dev}")
    if group_ids.dtype != torch.uint8 or group_ids.numel() != n // ARENA_BLOCK or not group_ids.is_contiguous() or group_ids.device != dev:
        raise ValueError(f"{name}: group_ids must be uint8, one for each {ARENA_BLOCK} elements, on {dev}")
    at += [hyper.data_ptr(), groups.data_ptr(), group_ids.data_ptr()]
    at += [_arena(t, name, k, dt, count, dev) for k, t, dt, count in states]
    spans = [(at[0], at[0] + 4 * n), (at[1], at[1] + 4 * n), *((a, a + t.element_size() * count) for a, (_, t, _, count) in zip(at[6:], states))]
    if p16 is not None:
        spans.append((at[2], at[2] + 2 * n))
    spans.sort()
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError(f"{name}: the arenas overlap")
    return hi, at
