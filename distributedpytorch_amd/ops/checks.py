"""Argument checks shared by the GPU and the CPU form of the group-norm, linear and AdamW operators: everything a kernel
assumes about shapes, types, layouts and devices is checked here, on the host, before anything is launched."""
from __future__ import annotations

import torch

ACTS = ("none", "relu", "silu", "gelu")          # ids of csrc/hip/act.h
FLOATS = (torch.float32, torch.bfloat16)


def act_id(act):
    try:
        return ACTS.index(act)
    except ValueError:
        raise ValueError(f"act must be one of {ACTS}, got {act!r}") from None


def same_device(name, first, **others):
    for k, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{name}: {k} is on {t.device}, the first operand on {first.device}")


def nhwc(t, name, shape=None, dtype=None):
    """Channel stride of an NHWC tensor (possibly a channel slice of a wider one)."""
    if t.dim() != 4 or (t.shape[3] > 1 and t.stride(3) != 1):
        raise ValueError(f"{name}: expected an NHWC tensor with contiguous channels, got {tuple(t.shape)} / {t.stride()}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    n, h, w, c = t.shape
    if h * w == 1:
        cs = t.stride(0) if n > 1 else c
    else:
        cs = t.stride(2) if w > 1 else t.stride(1)
        if (w > 1 and h > 1 and t.stride(1) != w * cs) or (n > 1 and t.stride(0) != h * w * cs):
            raise ValueError(f"{name}: only channel slices of NHWC tensors are supported, got strides {t.stride()}")
    if cs < c:
        raise ValueError(f"{name}: pixels overlap (channel stride {cs} < {c} channels)")
    return cs


def vec32(t, name, n):
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name}: expected {n} contiguous fp32 values, got {tuple(t.shape)} {t.dtype}")


def overlap(name, out, **ins):
    """Outputs may BE an input (same first element, same strides); a shifted overlap would be read after it was written."""
    def span(t):
        lo = t.data_ptr()
        return lo, lo + (sum((s - 1) * st for s, st in zip(t.shape, t.stride())) + 1) * t.element_size()
    if out.numel() == 0:
        return
    a, b = span(out)
    for k, t in ins.items():
        if t is None or t.numel() == 0 or (t.data_ptr() == out.data_ptr() and t.stride() == out.stride() and t.shape == out.shape):
            continue
        c, d = span(t)
        if a < d and c < b and not _slices_apart(out, t):
            raise ValueError(f"{name}: the output overlaps {k} without being the same tensor")


def _slices_apart(a, b):
    """Channel (or column) slices of one wider buffer that touch no common element."""
    if a.dim() != b.dim() or a.element_size() != b.element_size() or a.stride() != b.stride():
        return False
    row = a.stride(-2) if a.dim() > 1 and a.shape[-2] > 1 else 0
    off = (b.data_ptr() - a.data_ptr()) // a.element_size()
    return row > 0 and a.shape[-1] <= off <= row - b.shape[-1] or row > 0 and b.shape[-1] <= -off <= row - a.shape[-1]


# ------------------------------------------------------------------------------------------------ group norm
def group_norm(name, x, gamma, beta, groups, mean, rstd):
    if x.dtype not in FLOATS:
        raise ValueError(f"{name}: x must be fp32 or bf16, got {x.dtype}")
    cs = nhwc(x, f"{name}: x")
    n, h, w, c = x.shape
    if groups < 1 or c < 1 or c % groups:
        raise ValueError(f"{name}: {c} channels do not divide into {groups} groups")
    if n and h * w == 0:
        raise ValueError(f"{name}: images without pixels have no statistics ({tuple(x.shape)})")
    if h * w >= 1 << 30 or n >= 1 << 30 or n * groups >= 1 << 31 or c >= 1 << 30:
        raise ValueError(f"{name}: {tuple(x.shape)} is larger than a launch can index")
    vec32(gamma, f"{name}: gamma", c)
    vec32(beta, f"{name}: beta", c)
    vec32(mean, f"{name}: mean", n * groups)
    vec32(rstd, f"{name}: rstd", n * groups)
    same_device(name, x, gamma=gamma, beta=beta, mean=mean, rstd=rstd)
    return cs


# ------------------------------------------------------------------------------------------------ linear
def mat(t, name, rows=None, cols=None, dtype=None):
    """Row stride of a 2-d tensor with contiguous columns."""
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name}: expected a matrix with contiguous rows, got {tuple(t.shape)} / {t.stride()}")
    if (rows is not None and t.shape[0] != rows) or (cols is not None and t.shape[1] != cols):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected ({rows}, {cols})")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if ld < t.shape[1]:
        raise ValueError(f"{name}: rows overlap (stride {ld} < {t.shape[1]} columns)")
    return ld


def matrix_dims(name, *dims):
    for d in dims:
        if d >= 1 << 30:
            raise ValueError(f"{name}: a dimension of {d} is larger than a launch can index")


# ------------------------------------------------------------------------------------------------ AdamW
ARENA_BLOCK = 64


def adamw(name, p, g, p16, hyper, groups, group_ids, lo, hi, states):
    """The element range [lo, hi) of an arena: multiples of 64."""
    n = p.numel()
    hi = n if hi is None else hi
    if p.dtype != torch.float32 or g.dtype != torch.float32 or not p.is_contiguous() or not g.is_contiguous() or g.numel() != n:
        raise ValueError(f"{name}: p and g must be contiguous fp32 arenas of one size")
    if p16 is not None and (p16.dtype != torch.bfloat16 or p16.numel() != n or not p16.is_contiguous()):
        raise ValueError(f"{name}: p16 must be a contiguous bf16 arena of the size of p")
    for k, (t, dt, count) in states.items():
        if t.dtype != dt or t.numel() != count or not t.is_contiguous():
            raise ValueError(f"{name}: {k} must hold {count} contiguous values of {dt}, got {tuple(t.shape)} {t.dtype}")
    if n % ARENA_BLOCK or lo % ARENA_BLOCK or hi % ARENA_BLOCK or not 0 <= lo <= hi <= n:
        raise ValueError(f"{name}: [{lo}, {hi}) of {n} elements: ranges are multiples of {ARENA_BLOCK} inside the arena")
    if hyper.dtype != torch.float32 or hyper.numel() != 12 or not hyper.is_contiguous():
        raise ValueError(f"{name}: hyper must be the optimizer's vector of 12 fp32 values")
    if groups.dtype != torch.float32 or groups.dim() != 2 or groups.shape[1] != 2 or not 1 <= groups.shape[0] <= 256 or not groups.is_contiguous():
        raise ValueError(f"{name}: groups must be fp32 [1..256, 2] (lr multiplier, decay multiplier)")
    if group_ids.dtype != torch.uint8 or group_ids.numel() != n // ARENA_BLOCK or not group_ids.is_contiguous():
        raise ValueError(f"{name}: group_ids must be uint8, one for each {ARENA_BLOCK} elements")
    same_device(name, p, g=g, p16=p16, hyper=hyper, groups=groups, group_ids=group_ids, **{k: v[0] for k, v in states.items()})
    for k, t in (("p", p), ("g", g), ("p16", p16)) + tuple((k, v[0]) for k, v in states.items()):
        if t is not None and t.data_ptr() % 16:
            raise ValueError(f"{name}: {k} must be 16-byte aligned")
    return hi
