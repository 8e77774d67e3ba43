"""Rows in 8-bit integers with scales: quantizing and widening them, their product with a weight in 8-bit integers, and a linear
layer's weight gradient from its input kept in 8 bits.  No counterpart in the reference.

    quantize(x, group=0, pow2=False) -> Int8Rows       int8 values, a scale for each row or each group of columns
    dequantize(rows, dtype) -> Tensor                  q scale
    linear(x, w, dtype) -> Tensor                      x w^T for Int8Rows x (tokens) and w (output channels)
    weight_grad(dy, x, transposed=False) -> Tensor     dy^T x for Int8Rows x: the gradient of a weight that x met

Serving: the weight is quantized once, each batch by quantize before linear.  Training: an activation that the backward pass needs
is kept as quantize(x, group=128, pow2=True), half or a quarter of its bytes, and handed to weight_grad here or to
norms.rms_norm_backward_int8; dequantize gives it back to anything else.

They run the HIP kernels behind elr_quantize_int8, elr_dequantize_int8, elr_int8_linear and elr_int8_weight_grad
(elara_amd/csrc/quant.hip, int8_linear.hip, int8_grad.hip) on torch's current stream, without a host synchronisation.  None
registers with autograd: results are detached.
"""
from typing import NamedTuple

import torch

from . import _lib

GROUPS = (32, 64, 128, 256)
K_MOST = (1 << 17) - 1     # columns of a product: its int32 sums hold so many


class Int8Rows(NamedTuple):
    q: torch.Tensor        # int8 [..., D]
    scale: torch.Tensor    # float32 [..., 1], or [..., ceil(D / group)]; the values are q * scale
    group: int             # columns of a scale, 0 for the whole row


def _rows(t, name, dtypes):
    """t [..., D] as [n, D] rows a fixed stride apart (a copy only where the strides allow nothing else)."""
    if not (t.is_cuda and t.dtype in dtypes and t.dim() >= 1 and t.shape[-1] >= 1):
        raise RuntimeError(f'{name} must be a cuda tensor [..., D] of {" or ".join(map(str, dtypes))}, got '
                           f'{tuple(t.shape)} {t.dtype} {t.device}')
    x = t if t.dim() == 2 else t.reshape(t.numel() // t.shape[-1], t.shape[-1])
    return x if (x.stride(1) == 1 and x.stride(0) >= 0) or x.shape[1] == 1 else x.contiguous()


def _ld(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _group(group):
    group = int(group)
    if group and group not in GROUPS:
        raise RuntimeError(f'group must be 0 or one of {GROUPS}, got {group}')
    return group


def parts(rows, name):
    """(q as [n, D] rows, its stride in bytes, contiguous scales, group) of checked Int8Rows."""
    q, scale, group = rows
    group = _group(group)
    x = _rows(q, f'{name}.q', (torch.int8,))
    shape = q.shape[:-1] + (-(-q.shape[-1] // group) if group else 1,)
    if not (scale.is_cuda and scale.device == q.device and scale.dtype == torch.float32 and scale.shape == shape):
        raise RuntimeError(f'{name}.scale must be a cuda float32 tensor of shape {tuple(shape)} on {q.device}')
    return x, _ld(x), scale.contiguous(), group


def quantize(x, group=0, pow2=False):
    """x [..., D] cuda float32/float16/bfloat16 (any row stride) -> Int8Rows.  Over each row (group=0) or each group of 32, 64, 128
    or 256 columns (the last one shorter where that does not divide D): scale = max|x| / 127 (1 where that is 0), or with pow2 the
    smallest power of two that is no less (2^-126 at least); q = x / scale rounded to nearest even.  A power of two costs up to one of
    the 7 bits and makes q * scale exact in bfloat16 and float32, but for the largest values, which can come back infinite
    (float16 from 65,024 on, the others from 127 * 2^121).  A NaN or infinity makes its row or group NaN."""
    r = (_lib._host or _lib.host()).quantize(x, group, int(pow2))
    if r != _lib.NOT_TAKEN:
        _lib.check(r[0], 'elr_quantize_int8')
        return Int8Rows(r[1], r[2], group)
    group = _group(group)
    xr = _rows(x, 'x', tuple(_lib.ETYPE))
    n, D = xr.shape
    dev = x.device
    q = torch.empty(x.shape, dtype=torch.int8, device=dev)
    scale = torch.empty(x.shape[:-1] + (-(-D // group) if group else 1,), dtype=torch.float32, device=dev)
    if n:
        with _lib.on_device(dev):
            rc = _lib.lib().elr_quantize_int8(xr.data_ptr(), _lib.ETYPE[x.dtype], n, D, _ld(xr), group, int(bool(pow2)),
                                              q.data_ptr(), scale.data_ptr(), _lib.raw_stream(dev))
        _lib.check(rc, 'elr_quantize_int8')
    return Int8Rows(q, scale, group)


def dequantize(rows, dtype=torch.bfloat16):
    """q * scale in float32, rounded to dtype (float32, float16 or bfloat16), in q's shape."""
    r = (_lib._host or _lib.host()).dequantize(*rows, _lib.ETYPE.get(dtype, -1))
    if r != _lib.NOT_TAKEN:
        _lib.check(r[0], 'elr_dequantize_int8')
        return r[1]
    q, ld, scale, group = parts(rows, 'rows')
    if dtype not in _lib.ETYPE:
        raise RuntimeError(f'dtype must be one of {tuple(_lib.ETYPE)}, got {dtype}')
    n, D = q.shape
    x = torch.empty(rows.q.shape, dtype=dtype, device=q.device)
    if n:
        with _lib.on_device(q.device):
            rc = _lib.lib().elr_dequantize_int8(q.data_ptr(), n, D, ld, group, scale.data_ptr(), x.data_ptr(),
                                                _lib.ETYPE[dtype], _lib.raw_stream(q.device))
        _lib.check(rc, 'elr_dequantize_int8')
    return x


def linear(x, w, dtype=torch.bfloat16):
    """x: Int8Rows [..., K], a scale for each token; w: Int8Rows [N, K], a scale for each output channel (group=0 both).  Returns
    [..., N] of dtype: sum_k x.q w.q, exact, times x.scale, times w.scale, rounded once to fp32 at each of these steps (infinite
    where one passes its range) and then to dtype.  K is at most 131,071."""
    r = (_lib._host or _lib.host()).linear(*x, *w, _lib.ETYPE.get(dtype, -1))
    if r != _lib.NOT_TAKEN:
        _lib.check(r[0], 'elr_int8_linear')
        return r[1]
    xq, x_ld, xs, xg = parts(x, 'x')
    wq, w_ld, ws, wg = parts(w, 'w')
    if w.q.dim() != 2 or wq.shape[1] != xq.shape[1] or wq.device != xq.device:
        raise RuntimeError(f'w.q must have shape (N, {xq.shape[1]}) on {xq.device}, got {tuple(w.q.shape)} {w.q.device}')
    if xg or wg:
        raise RuntimeError('linear takes one scale for each row of x and w (group=0)')
    if dtype not in _lib.ETYPE:
        raise RuntimeError(f'dtype must be one of {tuple(_lib.ETYPE)}, got {dtype}')
    n, K = xq.shape
    N = wq.shape[0]
    if K > K_MOST:
        raise RuntimeError(f'K must be at most {K_MOST}, got {K}')
    dev = xq.device
    y = torch.empty(x.q.shape[:-1] + (N,), dtype=dtype, device=dev)
    if n and N:
        with _lib.on_device(dev):
            rc = _lib.lib().elr_int8_linear(xq.data_ptr(), n, K, x_ld, xs.data_ptr(), wq.data_ptr(), N, w_ld, ws.data_ptr(),
                                            y.data_ptr(), _lib.ETYPE[dtype], _lib.raw_stream(dev))
        _lib.check(rc, 'elr_int8_linear')
    return y


def weight_grad(dy, x, transposed=False):
    """dy [..., N] cuda float32/float16/bfloat16 (any row stride): the gradient of x W^T; x: Int8Rows [..., K], the layer's input
    as it was kept (scales by row or by group).  Returns dy^T x, float32 [N, K], or [K, N] with transposed (the gradient of a weight
    that multiplies from the right).  dy is not rounded; x is q * scale in bfloat16, exact where the scales are powers of two
    (pow2=True), else rounded: by 2^-8 of each value at most, no more than quantizing took off it.  Sums are float32 in an order that
    depends on the sizes alone.  An infinity in dy leaves NaN or infinities in its row of dy^T x."""
    r = (_lib._host or _lib.host()).weight_grad(dy, *x, int(transposed))
    if r != _lib.NOT_TAKEN:
        _lib.check(r[0], 'elr_int8_weight_grad')
        return r[1]
    dyr = _rows(dy, 'dy', tuple(_lib.ETYPE))
    q, ld, scale, group = parts(x, 'x')
    if x.q.shape[:-1] != dy.shape[:-1] or q.device != dy.device:
        raise RuntimeError(f'x.q must have shape {tuple(dy.shape[:-1])} + (K,) on {dy.device}')
    n, N = dyr.shape
    K = q.shape[1]
    dev, L = dy.device, _lib.lib()
    dw = torch.empty((K, N) if transposed else (N, K), dtype=torch.float32, device=dev)
    nbytes = L.elr_int8_weight_grad_scratch_bytes(n, N, K, _lib.ETYPE[dy.dtype])
    scratch = torch.empty(nbytes // 4, dtype=torch.float32, device=dev) if nbytes else None
    with _lib.on_device(dev):
        rc = L.elr_int8_weight_grad(dyr.data_ptr(), _lib.ETYPE[dy.dtype], n, N, _ld(dyr), q.data_ptr(), K, ld, group,
                                    scale.data_ptr(), dw.data_ptr(), int(bool(transposed)), _lib.ptr(scratch), nbytes,
                                    _lib.raw_stream(dev))
    _lib.check(rc, 'elr_int8_weight_grad')
    return dw
