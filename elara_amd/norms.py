"""Root-mean-square norm with the residual's addition, in the input's type or in fp8 with scales, and its backward.  No
counterpart in the reference.

    rms_norm(x, weight, eps=1e-6, residual=None) -> Norm              y = h rstd weight, h = x + residual
    rms_norm_fp8(x, weight, eps=1e-6, residual=None, group=0) -> NormFp8    y as e4m3 values and float32 scales
    rms_norm_backward(dy, h, weight, rstd, dh=None) -> (dx, dweight)
    rms_norm_backward_int8(dy, h, weight, rstd, dh=None) -> (dx, dweight)   the same with h kept in 8 bits (int8.Int8Rows)

They run the HIP kernels behind elr_rms_norm, elr_rms_norm_backward and elr_rms_norm_backward_int8 (elara_amd/csrc/norms.hip) on torch's current
stream: one launch forward (each row is read and written once; rows of more than 4,096 16-byte vectors are read again), two
backward (one where the rows are few).  Neither registers with autograd: results are detached.
"""
from typing import NamedTuple

import torch

from . import _lib, int8

FP8 = torch.float8_e4m3fn
GROUPS = (32, 64, 128, 256)


class Norm(NamedTuple):
    y: torch.Tensor        # x's type and shape
    h: torch.Tensor        # x + residual in the residual's type; x itself without a residual
    rstd: torch.Tensor     # float32, x's shape without the last dimension


class NormFp8(NamedTuple):
    y: torch.Tensor        # float8_e4m3fn, x's shape: the output divided by its scale
    scale: torch.Tensor    # float32 [..., 1], or [..., D / group]
    h: torch.Tensor
    rstd: torch.Tensor


def _rows(t, name, dtypes):
    """t [..., D] as [n, D] rows a fixed stride apart (a copy only where the strides allow nothing else)."""
    if not (t.is_cuda and t.dtype in dtypes and t.dim() >= 1 and t.shape[-1] >= 1):
        raise RuntimeError(f'{name} must be a cuda tensor [..., D] of {" or ".join(map(str, dtypes))}, got '
                           f'{tuple(t.shape)} {t.dtype} {t.device}')
    x = t if t.dim() == 2 else t.reshape(t.numel() // t.shape[-1], t.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _ld(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _weight(w, x):
    if w is None:
        return None, _lib.ETYPE[x.dtype]
    if not (w.is_cuda and w.device == x.device and w.dtype in (x.dtype, torch.float32) and w.shape == x.shape[-1:]):
        raise RuntimeError(f'weight must be a cuda {x.dtype} or float32 tensor of shape ({x.shape[-1]},) on {x.device}')
    return w.contiguous(), _lib.ETYPE[w.dtype]


def _norm(x, weight, eps, residual, fp8, group):
    r = (_lib._host or _lib.host()).norm(x, weight, eps, residual, int(fp8), group)
    if r != _lib.NOT_TAKEN:
        _lib.check(r[0], 'elr_rms_norm')
        return r[1:]
    xr = _rows(x, 'x', tuple(_lib.ETYPE))
    n, D = xr.shape
    dev, dt = x.device, x.dtype
    w, wt = _weight(weight, x)
    r, rt, h = None, _lib.ETYPE[dt], x
    if residual is not None:
        if residual.shape != x.shape or residual.device != dev:
            raise RuntimeError(f'residual must have shape {tuple(x.shape)} on {dev}')
        r = _rows(residual, 'residual', (dt, torch.float32))
        rt = _lib.ETYPE[r.dtype]
        h = torch.empty(x.shape, dtype=r.dtype, device=dev)
    lead = x.shape[:-1]
    y = torch.empty(x.shape, dtype=FP8 if fp8 else dt, device=dev)
    rstd = torch.empty(lead, dtype=torch.float32, device=dev)
    scale = torch.empty(lead + (D // group if group else 1,), dtype=torch.float32, device=dev) if fp8 else None
    if n:
        with _lib.on_device(dev):
            rc = _lib.lib().elr_rms_norm(
                xr.data_ptr(), _lib.ETYPE[dt], n, D, _ld(xr), _lib.ptr(r), rt, _ld(r) if r is not None else D, _lib.ptr(w),
                wt, eps, y.data_ptr(), int(fp8), group, _lib.ptr(scale), h.data_ptr() if r is not None else None,
                rstd.data_ptr(), _lib.raw_stream(dev))
        _lib.check(rc, 'elr_rms_norm')
    return y, scale, h, rstd


def rms_norm(x, weight, eps=1e-6, residual=None):
    """x [..., D] cuda float32/float16/bfloat16 (any row stride); weight [D] of x's type or float32, None for ones;
    residual of x's shape, in x's type or float32.  Sums are float32; the norm is taken of the unrounded x + residual, and
    y and h are rounded once."""
    y, _, h, rstd = _norm(x, weight, eps, residual, False, 0)
    return Norm(y, h, rstd)


def rms_norm_fp8(x, weight, eps=1e-6, residual=None, group=0):
    """rms_norm with y in float8_e4m3fn: y / scale, rounded to nearest even, scale = max|y| / 448 (1 where that
    rounds to 0) over each row (group=0) or each group of 32, 64, 128 or 256 columns."""
    group = int(group)
    if group and (group not in GROUPS or x.dim() < 1 or x.shape[-1] % group):
        raise RuntimeError(f'group must be 0 or one of {GROUPS} that divides D, got {group}')
    return NormFp8(*_norm(x, weight, eps, residual, True, group))


def rms_norm_backward(dy, h, weight, rstd, dh=None, need_dweight=True):
    """dy: y's gradient, in x's type; h, rstd: the forward's; dh (h's type and shape, or None): the gradient that arrives
    on the residual stream.  Returns (dx, dweight): dx in h's type, the gradient of x and of the residual alike (dh added);
    dweight float32 [D], summed in an order that depends on the sizes alone (None with need_dweight=False)."""
    r = (_lib._host or _lib.host()).norm_back(dy, h, weight, rstd, dh, int(need_dweight))
    if r != _lib.NOT_TAKEN:
        _lib.check(r[0], 'elr_rms_norm_backward')
        return r[1:]
    dyr = _rows(dy, 'dy', tuple(_lib.ETYPE))
    if h.shape != dy.shape or h.device != dy.device:
        raise RuntimeError(f'h must have shape {tuple(dy.shape)} on {dy.device}')
    hr = _rows(h, 'h', (dy.dtype, torch.float32))
    n, D = dyr.shape
    dev = dy.device
    w, wt = _weight(weight, dy)
    if not (rstd.is_cuda and rstd.device == dev and rstd.dtype == torch.float32 and rstd.shape == dy.shape[:-1]):
        raise RuntimeError(f'rstd must be a cuda float32 tensor of shape {tuple(dy.shape[:-1])} on {dev}')
    rstd = rstd.contiguous()
    dhr = None
    if dh is not None:
        if dh.shape != h.shape or dh.dtype != h.dtype or dh.device != dev:
            raise RuntimeError(f'dh must be a {h.dtype} tensor of shape {tuple(h.shape)} on {dev}')
        dhr = _rows(dh, 'dh', (h.dtype,))
    L = _lib.lib()
    dx = torch.empty(h.shape, dtype=h.dtype, device=dev)
    dw = scratch = None
    nbytes = 0
    if need_dweight:
        dw = torch.empty(D, dtype=torch.float32, device=dev)
        nbytes = L.elr_rms_norm_backward_scratch_bytes(n, D, _lib.ETYPE[dy.dtype])
        scratch = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
    if n or need_dweight:
        with _lib.on_device(dev):
            rc = L.elr_rms_norm_backward(
                dyr.data_ptr(), _lib.ETYPE[dy.dtype], n, D, _ld(dyr), hr.data_ptr(), _lib.ETYPE[h.dtype], _ld(hr),
                _lib.ptr(dhr), _ld(dhr) if dhr is not None else D, _lib.ptr(w), wt, rstd.data_ptr(), dx.data_ptr(),
                _lib.ptr(dw), _lib.ptr(scratch), nbytes, _lib.raw_stream(dev))
        _lib.check(rc, 'elr_rms_norm_backward')
    return dx, dw


def rms_norm_backward_int8(dy, h, weight, rstd, dh=None, need_dweight=True):
    """rms_norm_backward with h as int8.Int8Rows of dy's shape, as int8.quantize kept it (any group); rstd: the forward's, of the
    unrounded h.  dh: dy's shape, in dy's type or float32, or None.  dx has dh's type, dy's without dh."""
    r = (_lib._host or _lib.host()).norm_back_int8(dy, *h, weight, rstd, dh, int(need_dweight))
    if r != _lib.NOT_TAKEN:
        _lib.check(r[0], 'elr_rms_norm_backward_int8')
        return r[1:]
    dyr = _rows(dy, 'dy', tuple(_lib.ETYPE))
    q, q_ld, scale, group = int8.parts(h, 'h')
    if h.q.shape != dy.shape or q.device != dy.device:
        raise RuntimeError(f'h.q must have shape {tuple(dy.shape)} on {dy.device}')
    n, D = dyr.shape
    dev = dy.device
    w, wt = _weight(weight, dy)
    if not (rstd.is_cuda and rstd.device == dev and rstd.dtype == torch.float32 and rstd.shape == dy.shape[:-1]):
        raise RuntimeError(f'rstd must be a cuda float32 tensor of shape {tuple(dy.shape[:-1])} on {dev}')
    rstd = rstd.contiguous()
    dhr, xt = None, dy.dtype
    if dh is not None:
        if dh.shape != dy.shape or dh.device != dev:
            raise RuntimeError(f'dh must have shape {tuple(dy.shape)} on {dev}')
        dhr, xt = _rows(dh, 'dh', (dy.dtype, torch.float32)), dh.dtype
    L = _lib.lib()
    dx = torch.empty(dy.shape, dtype=xt, device=dev)
    dw = scratch = None
    nbytes = 0
    if need_dweight:
        dw = torch.empty(D, dtype=torch.float32, device=dev)
        nbytes = L.elr_rms_norm_backward_scratch_bytes(n, D, _lib.ETYPE[dy.dtype])
        scratch = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
    if n or need_dweight:
        with _lib.on_device(dev):
            rc = L.elr_rms_norm_backward_int8(
                dyr.data_ptr(), _lib.ETYPE[dy.dtype], n, D, _ld(dyr), q.data_ptr(), q_ld, group, scale.data_ptr(),
                _lib.ptr(dhr), _lib.ETYPE[xt], _ld(dhr) if dhr is not None else D, _lib.ptr(w), wt, rstd.data_ptr(),
                dx.data_ptr(), _lib.ptr(dw), _lib.ptr(scratch), nbytes, _lib.raw_stream(dev))
        _lib.check(rc, 'elr_rms_norm_backward_int8')
    return dx, dw
