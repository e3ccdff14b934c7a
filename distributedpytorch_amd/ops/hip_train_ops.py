"""Group norm, linear products with epilogues and AdamW on the GPU: checks (ops/checks.py), workspaces and launches of
csrc/hip/group_norm.hip, linear.hip and adamw.hip.  Workspaces are torch allocations of the call: they belong to its
stream, and to its graph where the call is captured, so no two calls share one."""
from __future__ import annotations

import ctypes

import torch

from . import checks, native, ref_ops
from .native import I32, I64, VP, F32, _OnDevice, ptr

_DT = {torch.float32: 0, torch.bfloat16: 1}


class GnParams(ctypes.Structure):
    _fields_ = [("x", VP), ("res", VP), ("dy", VP), ("yv", VP), ("y", VP), ("dx", VP), ("dres", VP), ("gamma", VP), ("beta", VP),
                ("mean", VP), ("rstd", VP), ("slab", VP), ("coef", VP), ("dgamma", VP), ("dbeta", VP),
                ("x_cs", I64), ("res_cs", I64), ("dy_cs", I64), ("yv_cs", I64), ("y_cs", I64), ("dx_cs", I64), ("dres_cs", I64),
                ("N", I32), ("HW", I32), ("C", I32), ("G", I32), ("cg", I32), ("S", I32), ("pps", I32), ("eps", F32)]


class LinParams(ctypes.Structure):
    _fields_ = [("a", VP), ("b", VP), ("lda", I64), ("ldb", I64), ("a_part", I64), ("b_part", I64), ("bias", VP), ("addend", VP), ("pre", VP),
                ("out", VP), ("preact", VP), ("ws", VP), ("ld_add", I64), ("ld_pre", I64), ("ld_out", I64), ("ld_z", I64),
                ("rows", I32), ("cols", I32), ("K", I32), ("parts", I32), ("splits", I32), ("accumulate", I32), ("act", I32), ("out32", I32),
                ("vec", I32), ("bias_vec", I32)]


_checked = []


def _lib():
    lib = native.hip_lib()
    if not _checked:
        if lib.dpa_gn_params_size() != ctypes.sizeof(GnParams) or lib.dpa_lin_params_size() != ctypes.sizeof(LinParams):
            raise RuntimeError("GnParams / LinParams ABI mismatch between ops/hip_train_ops.py and csrc/hip")
        _checked.append(True)
    return lib


# ----------------------------------------------------------------------------------------- group norm
def _gn_splits(n, hw, c):
    """Pixel ranges per image: enough blocks for 256 CUs where there are few images and channels."""
    blocks = n * ((c + 63) // 64)
    s = max(1, min((hw + 15) // 16, 2048 // max(blocks, 1), 64))
    pps = (hw + s - 1) // s
    return (hw + pps - 1) // pps, pps


def _gn_params(x, gamma, beta, groups, mean, rstd):
    n, h, w, c = x.shape
    p = GnParams()
    p.x, p.gamma, p.beta, p.mean, p.rstd = ptr(x), ptr(gamma), ptr(beta), ptr(mean), ptr(rstd)
    p.N, p.HW, p.C, p.G, p.cg = n, h * w, c, groups, c // groups
    p.S, p.pps = _gn_splits(n, h * w, c)
    return p


def group_norm_fwd(x, gamma, beta, groups, eps, y, mean, rstd, act="none", residual=None):
    cs = checks.group_norm("group_norm_fwd", x, gamma, beta, groups, mean, rstd)
    a = checks.act_id(act)
    y_cs = checks.nhwc(y, "group_norm_fwd: y", x.shape, x.dtype)
    res_cs = 0 if residual is None else checks.nhwc(residual, "group_norm_fwd: residual", x.shape, x.dtype)
    checks.same_device("group_norm_fwd", x, y=y, residual=residual)
    checks.overlap("group_norm_fwd", y, x=x, residual=residual)
    if x.numel() == 0:
        return y
    p = _gn_params(x, gamma, beta, groups, mean, rstd)
    p.y, p.res, p.x_cs, p.y_cs, p.res_cs, p.eps = ptr(y), ptr(residual), cs, y_cs, res_cs, eps
    with _OnDevice(x) as stream:
        slab = torch.empty(p.N * p.S * 2 * p.C, device=x.device, dtype=torch.float32)
        p.slab = ptr(slab)
        _lib().dpa_group_norm_fwd(ctypes.byref(p), a, _DT[x.dtype], stream)
    return y


def group_norm_bwd(dy, x, gamma, beta, groups, mean, rstd, dx, dgamma=None, dbeta=None, act="none", y=None, residual=None,
                   dresidual=None):
    strides = ref_ops.check_group_norm_bwd(dy, x, gamma, beta, groups, mean, rstd, dx, dgamma, dbeta, act, y, residual, dresidual)
    if x.numel() == 0:
        for t in (dgamma, dbeta):
            if t is not None:
                t.zero_()
        return dx
    p = _gn_params(x, gamma, beta, groups, mean, rstd)
    p.dy, p.dx, p.yv, p.res, p.dres = ptr(dy), ptr(dx), ptr(y), ptr(residual), ptr(dresidual)
    p.x_cs, p.dy_cs, p.dx_cs, p.yv_cs, p.res_cs, p.dres_cs = strides
    p.dgamma, p.dbeta = ptr(dgamma), ptr(dbeta)
    with _OnDevice(x) as stream:
        ws = torch.empty(p.N * p.S * 2 * p.C + 2 * p.N * p.G, device=x.device, dtype=torch.float32)
        p.slab, p.coef = ptr(ws), VP(ws.data_ptr() + 4 * p.N * p.S * 2 * p.C)
        _lib().dpa_group_norm_bwd(ctypes.byref(p), checks.act_id(act), _DT[x.dtype], stream)
    return dx


# ----------------------------------------------------------------------------------------- linear products
_FPROP, _DGRAD, _WGRAD = 0, 1, 2          # csrc/hip/linear.hip
_TILES = ((256, 256), (128, 128), (64, 64))


def _plan(rows, cols, ksteps):
    """(tile, splits of the reduction)"""
    for i, (bm, bn) in enumerate(_TILES):
        blocks = ((rows + bm - 1) // bm) * ((cols + bn - 1) // bn)
        if blocks >= 200:
            return i, 1
    blocks = ((rows + 63) // 64) * ((cols + 63) // 64)
    return 2, max(1, min(256 // blocks, ksteps // 4, 16))


def _aligned(t, ld):
    es = t.element_size()
    return t.data_ptr() % 16 == 0 and (ld * es) % 16 == 0


def _operand(t, ld, stream, keep):
    """(pointer, row stride, stride of its parts, parts): the matrix as the kernel's DMA takes it - bf16 rows of a multiple
    of 8 elements at 16-byte addresses as they are, anything else through lin_pack_kernel."""
    rows, cols = t.shape
    f32 = t.dtype == torch.float32
    if not f32 and cols % 8 == 0 and _aligned(t, ld):
        return ptr(t), ld, 0
    ldd = (cols + 7) // 8 * 8
    buf = torch.empty((3 if f32 else 1) * rows * ldd, device=t.device, dtype=torch.bfloat16)
    keep.append(buf)
    if rows:
        _lib().dpa_linear_pack(ptr(t), I64(ld), rows, cols, ldd, int(_aligned(t, ld)), ptr(buf), _DT[t.dtype], stream)
    return ptr(buf), ldd, rows * ldd


def _product(epi, a, lda, b, ldb, p, k, stream, keep):
    p.a, p.lda, p.a_part = _operand(a, lda, stream, keep)
    p.b, p.ldb, p.b_part = _operand(b, ldb, stream, keep)
    p.K, p.parts = k, 3 if a.dtype == torch.float32 else 1
    tile, p.splits = _plan(p.rows, p.cols, (k + 63) // 64 * (6 if p.parts == 3 else 1))
    if p.splits > 1:
        ws = torch.empty(p.splits * p.rows * p.cols, device=a.device, dtype=torch.float32)
        keep.append(ws)
        p.ws = ptr(ws)
    _lib().dpa_linear(ctypes.byref(p), epi, tile, stream)


def _vec(cols, *mats):
    return int(cols % 8 == 0 and all(t is None or _aligned(t, ld) for t, ld in mats))


def linear_fprop(x, w, y, bias=None, act="none", addend=None, preact=None):
    ldx, ldw, ldy, lda, ldz = ref_ops.check_linear_fprop(x, w, y, bias, act, addend, preact)
    if x.shape[0] == 0:
        return y
    p = LinParams()
    p.bias, p.addend, p.out, p.preact = ptr(bias), ptr(addend), ptr(y), ptr(preact)
    p.ld_add, p.ld_out, p.ld_z = lda, ldy, ldz
    p.rows, p.cols, p.act, p.out32 = x.shape[0], w.shape[0], checks.act_id(act), int(x.dtype == torch.float32)
    p.vec = _vec(p.cols, (y, ldy), (addend, lda), (preact, ldz))
    p.bias_vec = int(bias is not None and p.cols % 8 == 0 and bias.data_ptr() % 16 == 0)
    keep = []
    with _OnDevice(x) as stream:
        _product(_FPROP, x, ldx, w, ldw, p, x.shape[1], stream, keep)
    return y


def linear_dgrad(dy, w, dx, act="none", preact=None, addend=None):
    ldy, ldw, ldx, ldp, lda = ref_ops.check_linear_dgrad(dy, w, dx, act, preact, addend)
    if dy.shape[0] == 0:
        return dx
    p = LinParams()
    p.addend, p.pre, p.out = ptr(addend), ptr(preact), ptr(dx)
    p.ld_add, p.ld_pre, p.ld_out = lda, ldp, ldx
    p.rows, p.cols, p.act, p.out32 = dy.shape[0], w.shape[1], checks.act_id(act), int(dy.dtype == torch.float32)
    p.vec = _vec(p.cols, (dx, ldx), (addend, lda), (preact, ldp))
    keep = []
    with _OnDevice(dy) as stream:
        _product(_DGRAD, dy, ldy, w, ldw, p, dy.shape[1], stream, keep)
    return dx


def linear_wgrad(dy, x, dw, db=None, accumulate=False):
    ldy, ldx, ldw = ref_ops.check_linear_wgrad(dy, x, dw, db)
    p = LinParams()
    p.out, p.ld_out, p.accumulate = ptr(dw), ldw, int(accumulate)
    p.rows, p.cols = dy.shape[1], x.shape[1]
    p.vec = _vec(p.cols, (dw, ldw))
    keep = []
    with _OnDevice(dy) as stream:
        _product(_WGRAD, dy, ldy, x, ldx, p, dy.shape[0], stream, keep)
        if db is not None:
            m, n = dy.shape
            splits = max(1, min((m + 63) // 64, 2048 // ((n + 63) // 64), 64))
            per = max(1, (m + splits - 1) // splits)
            slab = torch.empty(splits * n, device=dy.device, dtype=torch.float32)
            _lib().dpa_linear_colsum(ptr(dy), I64(ldy), m, n, splits, per, ptr(slab), int(accumulate), ptr(db), _DT[dy.dtype], stream)
    return dw


# ----------------------------------------------------------------------------------------- AdamW
def _at(t, lo, esize):
    return VP(t.data_ptr() + lo * esize) if t is not None else VP(0)


def adamw_step(p, g, m, v, p16, hyper, groups, group_ids, lo=0, hi=None):
    n = p.numel()
    hi = checks.adamw("adamw_step", p, g, p16, hyper, groups, group_ids, lo, hi,
                      {"m": (m, torch.float32, n), "v": (v, torch.float32, n)})
    with _OnDevice(p) as stream:
        _lib().dpa_adamw_step(_at(p, lo, 4), _at(g, lo, 4), _at(m, lo, 4), _at(v, lo, 4), _at(p16, lo, 2), ptr(hyper), ptr(groups),
                              _at(group_ids, lo // 64, 1), I64(hi - lo), stream)


def adamw8_step(p, g, m, v, m_scale, v_scale, p16, hyper, groups, group_ids, seed, lo=0, hi=None):
    n = p.numel()
    hi = checks.adamw("adamw8_step", p, g, p16, hyper, groups, group_ids, lo, hi,
                      {"m": (m, torch.float8_e4m3fn, n), "v": (v, torch.float8_e5m2, n),
                       "m_scale": (m_scale, torch.float32, n // 64), "v_scale": (v_scale, torch.float32, n // 64)})
    with _OnDevice(p) as stream:
        _lib().dpa_adamw8_step(_at(p, lo, 4), _at(g, lo, 4), _at(m, lo, 1), _at(v, lo, 1), _at(m_scale, lo // 64, 4),
                               _at(v_scale, lo // 64, 4), _at(p16, lo, 2), ptr(hyper), ptr(groups), _at(group_ids, lo // 64, 1),
                               ctypes.c_uint(seed & 0xFFFFFFFF), I64(lo), I64(hi - lo), stream)
