"""Group norm, linear products with epilogues and AdamW on the GPU: checks (ops/checks.py), workspaces and launches of
csrc/hip/group_norm.hip, linear.hip and adamw.hip.  Workspaces are torch allocations of the call: they belong to its
stream, and to its graph where the call is captured, so no two calls share one.

A small call is bound by what the host does before the launch: everything here works on plain integers, and each operator
is one call into the library."""
from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import checks, native
from .native import I32, I64, VP

_F32 = torch.float32


# GnParams of csrc/hip/group_norm.hip: 15 addresses, 7 strides, 13 integers, eps
_GN_PARAMS = struct.Struct("@15Q7q13if")


# LinCall of csrc/hip/linear.h: operands and their strides; bias, addend, pre, out, preact, workspaces; strides; the operands as they
# are and their strides; nine integers; what the operands are packed into, the bias gradient and its slab; twelve integers
_LIN_CALL = struct.Struct("@2Q4q8Q4q2Q2q9i4Q12i")


_loaded = []


def _lib():
    if _loaded:
        return _loaded[0]
    lib = native.hip_lib()
    if lib.dpa_gn_params_size() != _GN_PARAMS.size or lib.dpa_lin_params_size() != _LIN_CALL.size:
        raise RuntimeError("GnParams or LinCall of csrc/hip has another size than ops/hip_train_ops.py packs")
    for name, types in (("dpa_group_norm", (ctypes.c_char_p, I32, I32, VP)), ("dpa_linear", (ctypes.c_char_p, VP)),
                        ("dpa_adamw_step", (VP,) * 7 + (I32, VP, I64, VP)),
                        ("dpa_adamw8_step", (VP,) * 9 + (I32, VP, ctypes.c_uint, I64, I64, VP))):
        lib.declare(name, types)          # (plain integers are converted faster than wrapped ones)
    _loaded.append(lib)
    return lib


def _run(device, body, *args, **kw):
    """body(stream, *args) with the tensors' device as the current one, on its current stream"""
    i = device.index
    if i == torch._C._cuda_getDevice():
        return body(torch._C._cuda_getCurrentRawStream(i), *args, **kw)
    with torch.cuda.device(device):
        return body(torch._C._cuda_getCurrentRawStream(i), *args, **kw)


def _cdiv(a, b):
    return (a + b - 1) // b


# ----------------------------------------------------------------------------------------- group norm
_ANY, _ONE, _TWO, _LONE = 0, 1, 2, 3          # csrc/hip/group_norm.hip
_plans = {}


def _gn_plan(n, hw, c, cg, v, bwd):
    """(way, threads, W, rows, R, S, pixels of a split) of csrc/hip/group_norm.hip for vectors of v channels (1: layouts without
    16-byte vectors; 0: any layout).

    A block that holds its chunk of an image in registers reads everything once, so it is taken wherever an image fits: the
    chunk as wide as possible, down to 32 bytes of a pixel (times in us, relu + residual, 64 images, bf16; the other side is
    two passes): 40 x 40 x 256 forward in 128 bytes 37, 64 bytes 40, two passes 53, backward in 64 bytes 73, two passes 108;
    56 x 56 x 256 forward in 64 bytes 79, two passes 88, backward in 32 bytes 178, two passes 188.
    Few images make too few blocks: then the chunk is as narrow as it goes (4 images of 28 x 28 x 512: 7.1 forward and 13.2
    backward, 10.5 and 19.1 in 128 bytes), and a large image goes through two passes (4 of 56 x 56 x 256: 15.5 and 26.8, one
    pass 19.9 and 28.5; with 16 images 26.3 and 75.7, one pass 20.4 and 46.8).
    A launch has fewer than 2^32 threads: more chunks of images than that take the kernels for any layout, which loop over images.
    Without 16-byte vectors a lane holds one channel; up to 16 pixels a lane that is faster than the kernels for any layout
    (64 images of 22 x 22 x 90, fp32: 12.6 forward and 16.1 backward, 17.2 and 24.4), with 52 it is not (31 x 31 x 90, bf16 with
    a residual: 33.1 and 63.4, 24.7 and 44.7)."""
    plan = _gn_chunks(n, hw, c, cg, v, bwd) if v else None
    if plan is not None:
        way, threads, w, _, _, s, _ = plan
        if n * s * (c // (w if way == _LONE else w * v)) * threads < 1 << 32:
            return plan
    blocks = n * _cdiv(c, 64)
    s = max(1, min(_cdiv(hw, 16), 2048 // max(blocks, 1), 64), min(_cdiv(hw, 2048), 65535))          # (512 pixels a thread)
    pps = _cdiv(hw, s)
    return _ANY, 256, 1, 1, 1, _cdiv(hw, pps), pps


def _gn_chunks(n, hw, c, cg, v, bwd):
    """The plan of the kernels that own chunks of an image's channels, or None where none of them takes it."""
    if v > 1:
        unit = cg * v // math.gcd(cg, v) // v          # vectors of the smallest chunk of whole groups
        total = c // v
        chunks = [w for w in range(unit, min(total, 256) + 1, unit) if total % w == 0]
        sizes = ((256, 1), (256, 2), (512, 4), (512, 7), (512, 13)) + (() if bwd else ((1024, 13),))
        for want in (8, 4, 2) if n * (total // 8) >= 128 else (2,):
            for threads, r in sizes:
                for w in chunks:
                    if (w >= want or w == chunks[-1]) and w <= threads and hw <= threads // w * r and w * v // cg <= 1024:
                        if hw > 1024 and n * (total // w) < 256:
                            break
                        return _ONE, threads, w, threads // w, r, 1, hw
        fit = [w for w in chunks if w * v // cg <= 1024]
        if fit:
            w = next((w for w in fit if w >= 16), fit[-1])
            rows, r = 512 // w, 2 if bwd else 8
            # (64 pixels a thread at most: sums in 32 bits; and every block of the second pass joins all S ranges)
            pps = rows * r * (max(1, min(n * _cdiv(hw, rows * r) * (total // w) // 1024, 32)) if bwd else 1)
            if hw <= 2048 * pps:
                return _TWO, 512, w, rows, r, _cdiv(hw, pps), pps
    for want in (32, 16, 1) if n * c >= 8192 else (1,):
        for threads, r in ((256, 4), (512, 16)):
            for w in range(cg, min(c, threads) + 1, cg):
                if c % w == 0 and (w >= want or w == c) and hw <= threads // w * r:
                    return _LONE, threads, w, threads // w, r, 1, hw
    return None


def _gn(x, groups, spans, vecs, grads, bwd, a, eps):
    """spans: of x, residual, dy, y (the mask), y (the output), dx, dresidual; grads: the addresses of dgamma and dbeta."""
    n, h, w, c = x.shape
    f32 = x.dtype is _F32
    (ax, sx, _), (ar, sr, _), (ad, sd, _), (am, sm, _), (ay, sy, _), (adx, sdx, _), (adr, sdr, _) = spans
    strides = sx | sr | sd | sm | sy | sdx | sdr
    if strides >= 1 << 18:          # (offsets of a lane in 32 bits)
        v = 0
    else:
        v = 4 if f32 else 8
        if (ax | ar | ad | am | ay | adx | adr | strides * (4 if f32 else 2)) & 15 or c % v:
            v = 1
    key = (n, h * w, c, groups, v, bwd)
    plan = _plans.get(key)
    if plan is None:
        if len(_plans) > 4096:
            _plans.clear()
        plan = _plans[key] = _gn_plan(n, h * w, c, c // groups, v, bwd)
    way, threads, wide, rows, r, s, pps = plan
    if bwd:
        slab = n * s * 2 * c if way == _ANY or grads[0] or grads[1] else 0
        coef = 0 if way & 1 else 2 * n * groups * (s if way == _TWO else 1)
    else:
        slab, coef = 0 if way & 1 else n * s * 2 * (groups if way == _TWO else c), 0
    _run(x.device, _gn_launch, x.device, slab, coef, bwd, f32, (ax, ar, ad, am, ay, adx, adr) + vecs,
         grads + (sx, sr, sd, sm, sy, sdx, sdr, n, h * w, c, groups, c // groups, s, pps, a, wide, rows, r, threads, way, eps))


def _gn_launch(stream, device, slab, coef, bwd, f32, head, tail):
    at = 0
    if slab + coef:
        ws = torch.empty(slab + coef, device=device, dtype=_F32)
        at = ws.data_ptr()
    rc = _lib().dpa_group_norm(_GN_PARAMS.pack(*head, at, at + 4 * slab, *tail), bwd, f32, stream)
    if rc:
        name = "group_norm_bwd" if bwd else "group_norm_fwd"
        raise checks.group_norm_overlaps(name) if rc == -1 else native.KernelLaunchError(f"{name}: kernel launch failed with hipError_t {rc}")


def group_norm_fwd(x, gamma, beta, groups, eps, y, mean, rstd, act="none", residual=None):
    a, xs, ys, rs, vecs = checks.group_norm_fwd(x, gamma, beta, groups, y, mean, rstd, act, residual)
    if x.shape[0]:
        o = checks.NOTHING
        _gn(x, groups, (xs, rs, o, o, ys, o, o), tuple(vecs), (0, 0), 0, a, eps)
    return y


def group_norm_bwd(dy, x, gamma, beta, groups, mean, rstd, dx, dgamma=None, dbeta=None, act="none", y=None, residual=None,
                   dresidual=None):
    a, xs, dys, dxs, ys, rs, drs, vecs = checks.group_norm_bwd(dy, x, gamma, beta, groups, mean, rstd, dx, dgamma, dbeta, act, y,
                                                               residual, dresidual)
    if x.shape[0] == 0:
        for t in (dgamma, dbeta):
            if t is not None:
                t.zero_()
        return dx
    _gn(x, groups, (xs, rs, dys, ys, checks.NOTHING, dxs, drs), tuple(vecs[:4]), tuple(vecs[4:]), 1, a, 0.0)
    return dx


# ----------------------------------------------------------------------------------------- linear products
_FPROP, _DGRAD, _WGRAD = 0, 1, 2          # csrc/hip/linear.h


def _plan(rows, cols, k, f32):
    """(tile of lin_tile, splits of the reduction).  The largest tile that still fills the chip: 256 x 256 runs one block on
    each of the 256 CUs, 128 x 128 two (or one with four steps in LDS), 64 x 64 two.  Measured on both sides, us:
      256 x 256 below K = 384 pays more for its epilogue than it saves (2909 x 6280 x 192: 29.1, 128 x 128 23.2; 10382 x 5456
        x 480: 84.2, 90.2); fp32 walks over K six times and has no such bound;
      128 x 128 from 140 tiles on (1433 x 1872 x 2640, 180 tiles: 31.2, 64 x 64 37.6; 715 x 560 x 1504, 30 tiles: 20.4, 11.7);
        two blocks a CU above 256 tiles (6306 x 1112 x 736: 21.3, one 25.8), four steps in LDS below (2048^3: 25.4, 30.0);
      fp32 in tiles of 128 x 128 has one block a CU, so the last round has to be well filled (688 x 5688 x 888, 270 tiles: 91.9,
        64 x 64 82.3), and a long reduction is split over it (976 x 744 x 5741: 84 in five, 64 x 64 125 whole and 123 in two);
        up to 512 elements a part 64 x 64 in one round needs no split and no launch to join it (1021 x 1000 x 2048: 44.0, 128 x
        128 in four 45.8; 900 x 700 x 1600: 37.9, 51.7 in three);
      a split costs a pass over its partial products and pays from 512 elements a part on (3119 x 280 x 624: 7.9 whole, 14.6
        in two; a weight gradient of 784 x 184 x 4670: 14.7 in six, 28.7 whole, of 792 x 1424 x 6161 in 128 x 128: 34.7 in six, 55.4
        in whole 64 x 64),
        in fp32 with few tiles from 128 on (176 x 248 x 571: 13.4 in four, 15.7 whole), as long as every part has a CU of its own: two
        blocks share one's LDS traffic (256 x 1000 x 2048, 64 tiles: 28.2 in four, 30.5 in eight; 900 x 900 x 1400, 225 tiles:
        44.0 whole, 52.5 in two; 700 x 700 x 2048, 121 tiles: 37.0 in two, 40.3 in four)."""
    if _cdiv(rows, 256) * _cdiv(cols, 256) >= 200 and (f32 or k >= 384):
        return 0, 1
    t128, t64 = _cdiv(rows, 128) * _cdiv(cols, 128), _cdiv(rows, 64) * _cdiv(cols, 64)
    if f32:
        if t128 >= 160 * _cdiv(t128, 256):
            return 4, 1
        if 40 <= t128 <= 128 and k >= 1500 and (t64 > 256 or k > 512 * (256 // t128)):
            return 4, min(256 // t128, k // 512)
        return 5, max(1, min(256 // t64, k // (128 if t64 < 64 else 384), 16))
    if k >= 4096 and 32 <= t128 < 200:
        return 1, min(512 // t128, k // 768, 16)
    if t128 >= 140:
        return (1 if t128 > 256 else 2), 1
    return 3, max(1, min(512 // t64, k // 512, 16))


def _linear(stream, epi, t_a, a, t_b, b, rows, cols, k, vec, act=0, out=checks.NOTHING, bias=0, bias_vec=0, addend=checks.NOTHING,
            pre=checks.NOTHING, preact=checks.NOTHING, db=0, accumulate=0):
    """The plan, the workspace and the launch of a product: matrices as the checks return them."""
    f32 = t_a.dtype is _F32
    es = 4 if f32 else 2
    (src_a, src_lda, _), (src_b, src_ldb, _) = a, b
    (a_rows, a_cols), (b_rows, b_cols) = t_a.shape, t_b.shape
    ok_a, ok_b = not (src_a | src_lda * es) & 15, not (src_b | src_ldb * es) & 15
    at_a, lda, at_b, ldb = src_a, src_lda, src_b, src_ldb
    parts = 3 if f32 else 1
    need = ld_a = ld_b = a_part = b_part = pack_a = pack_b = ws = sums = db_out = db_slab = takers = db_splits = 0
    if epi == _FPROP and rows <= (64 if f32 else 32) and cols < 1 << 27 and ok_a and ok_b and not (k * es) & 15:
        # (a launch has fewer than 2^32 threads, 32 for a column; 32 rows x 4096 x 4096 in bf16: 15.0 us, in 64 x 64 tiles 18.8; 64 rows: 21.6 and 19.7.
        # fp32, 64 rows: 47.9 and 56.8)
        tile, splits = -1, 1
    else:
        tile, splits = _plan(rows, cols, k, f32)
        # the DMA takes bf16 rows of a multiple of 8 elements at 16-byte addresses as they are; anything else is packed
        if f32 or not ok_a or a_cols & 7:
            ld_a = lda = (a_cols + 7) & ~7
            a_part = a_rows * lda
            pack_a, need = 1, parts * a_part * 2 + 15 & ~15
        if f32 or not ok_b or b_cols & 7:
            ld_b = ldb = (b_cols + 7) & ~7
            b_part = b_rows * ldb
            pack_b, need = need + 1, need + (parts * b_part * 2 + 15 & ~15)
        steps = _cdiv(k, 32 if tile >= 4 else 64) * (6 if f32 and tile < 4 else 1)
        if splits > 1:
            splits = _cdiv(steps, _cdiv(steps, splits))          # no range is empty
        if splits > 1:
            ws, need = need + 1, need + (splits * rows * cols * 4 + 15 & ~15)
        if db:
            if tile == 0:          # a pass over dy of its own
                db_splits = max(1, min(_cdiv(k, 32), 1024 // _cdiv(rows, 512)))
                db_slab, need = need + 1, need + db_splits * rows * 4
            elif splits == 1 and steps <= 16:
                # one wave makes the sums of a row tile, into db: at most some 100 instructions more, and no launch to join them
                # (500 x 512 x 1000: 8.2 us, joined 10.0; 128 x 64 x 64: 9.9 us a call, 14.3)
                takers, sums = 1, db
            else:          # the 2 waves in each of the tiles of a row take turns
                takers = min(2 * _cdiv(cols, 64 if tile == 3 or tile == 5 else 128), 16)
                db_out, sums, need = db, need + 1, need + splits * takers * rows * 4
    if need:          # (offsets plus one so far)
        base = torch.empty(need, device=t_a.device, dtype=torch.uint8)
        at = base.data_ptr() - 1
        if pack_a:
            at_a = pack_a = at + pack_a
        if pack_b:
            at_b = pack_b = at + pack_b
        if ws:
            ws += at
        if db_out:
            sums += at
        if db_slab:
            db_slab += at
    _lib().dpa_linear(_LIN_CALL.pack(
        at_a, at_b, lda, ldb, a_part, b_part, bias, addend[0], pre[0], out[0], preact[0], ws, sums, db_out,
        addend[1], pre[1], out[1], preact[1], src_a, src_b, src_lda, src_ldb, rows, cols, k, splits, accumulate, act, vec,
        bias_vec, takers, pack_a, pack_b, db, db_slab,
        a_rows, a_cols, b_rows, b_cols, ld_a, ld_b, ok_a, ok_b, db_splits, epi, tile, f32), stream)


def linear_fprop(x, w, y, bias=None, act="none", addend=None, preact=None):
    a, xs, ws, ys, ads, zs, b = checks.linear_fprop(x, w, y, bias, act, addend, preact)
    m, k = x.shape
    if m:
        n = w.shape[0]
        vec = not (n & 7 or (ys[0] | ads[0] | zs[0] | (ys[1] | ads[1] | zs[1]) * y.element_size()) & 15)
        _run(x.device, _linear, _FPROP, x, xs, w, ws, m, n, k, vec, a, ys, b, not (n & 7 or b & 15), ads, checks.NOTHING, zs)
    return y


def linear_dgrad(dy, w, dx, act="none", preact=None, addend=None):
    a, dys, ws, dxs, zs, ads = checks.linear_dgrad(dy, w, dx, act, preact, addend)
    m, n = dy.shape
    if m:
        k = w.shape[1]
        vec = not (k & 7 or (dxs[0] | ads[0] | zs[0] | (dxs[1] | ads[1] | zs[1]) * dx.element_size()) & 15)
        _run(dy.device, _linear, _DGRAD, dy, dys, w, ws, m, k, n, vec, a, dxs, 0, 0, ads, zs)
    return dx


def linear_wgrad(dy, x, dw, db=None, accumulate=False):
    dys, xs, dws, b = checks.linear_wgrad(dy, x, dw, db)
    m, n = dy.shape
    if m == 0:
        if not accumulate:
            dw.zero_()
            if db is not None:
                db.zero_()
        return dw
    k = x.shape[1]
    vec = not (k & 7 or (dws[0] | dws[1] * 4) & 15)
    _run(dy.device, _linear, _WGRAD, dy, dys, x, xs, n, k, m, vec, out=dws, db=b, accumulate=int(accumulate))
    return dw


# ----------------------------------------------------------------------------------------- AdamW
def adamw_step(p, g, m, v, p16, hyper, groups, group_ids, lo=0, hi=None):
    n = p.numel()
    hi, at = checks.adamw("adamw_step", p, g, p16, hyper, groups, group_ids, lo, hi, (("m", m, _F32, n), ("v", v, _F32, n)))
    _run(p.device, _adamw, at, groups.shape[0], lo, hi)


def _adamw(stream, at, rows, lo, hi):
    p, g, p16, h, gr, ids, m, v = at
    b = 4 * lo
    _lib().dpa_adamw_step(p + b, g + b, m + b, v + b, p16 and p16 + 2 * lo, h, gr, rows, ids + lo // 64, hi - lo, stream)


def adamw8_step(p, g, m, v, m_scale, v_scale, p16, hyper, groups, group_ids, seed, lo=0, hi=None):
    n = p.numel()
    hi, at = checks.adamw("adamw8_step", p, g, p16, hyper, groups, group_ids, lo, hi,
                          (("m", m, torch.float8_e4m3fn, n), ("v", v, torch.float8_e5m2, n), ("m_scale", m_scale, _F32, n // 64),
                           ("v_scale", v_scale, _F32, n // 64)))
    _run(p.device, _adamw8, at, groups.shape[0], seed & 0xFFFFFFFF, lo, hi)


def _adamw8(stream, at, rows, seed, lo, hi):
    p, g, p16, h, gr, ids, m, v, ms, vs = at
    b, s = 4 * lo, lo // 16
    _lib().dpa_adamw8_step(p + b, g + b, m + lo, v + lo, ms + s, vs + s, p16 and p16 + 2 * lo, h, gr, rows, ids + lo // 64, seed, lo,
                           hi - lo, stream)
