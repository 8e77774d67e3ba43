"""The global norm of many gradients, and clipping by it, before the row-sparse and the dense Adam.  No counterpart in the
reference, whose step updates unclipped.

    grad_norm(grads, norm_type=2.0) -> norm                              float32 scalar on the GPU
    clip_grad_norm(grads, max_norm, norm_type=2.0, eps=1e-6, out=None) -> norm   grads scaled by min(1, max_norm / (norm + eps))

They run the HIP kernels behind elr_grad_norm and elr_clip_grad_norm (elara_amd/csrc/gradnorm.hip) on torch's current
stream, without a host synchronisation: two launches for up to 136 tensors that are each one run of memory, of up to 16 MB
together, a third beyond that, two more for each further 136 and for each tensor that is not one run (an element a thread
there: 2 to 4 times the time).  A batch's summed row gradients (dedup.embedding_dense_backward, dedup.segment_sum_plan) are one
of the tensors; the sums that ElaraStep takes within its native step are not reachable, so only a loop over the row ops (or the
host-planned step's plan and update) can clip.  Gradients are written without bumping their version.
"""
import math

import torch

from . import _lib

_KINDS = {1.0: 1, 2.0: 2, math.inf: 0}


def _two_strides(t, o):
    """(rows, cols, ld, cs, out_ld, out_cs) of t's elements and o's in the same order, neighbouring dimensions merged."""
    dims = []
    for d in sorted(range(t.dim()), key=lambda i: (-t.stride(i), -o.stride(i), -t.shape[i])):
        if t.shape[d] == 1:
            continue
        ts, os = t.stride(d), o.stride(d)
        if dims and dims[-1][1] == ts * t.shape[d] and dims[-1][2] == os * t.shape[d]:
            dims[-1] = (dims[-1][0] * t.shape[d], ts, os)
        else:
            dims.append((t.shape[d], ts, os))
    while len(dims) < 2:
        dims.insert(0, (1, 0, 0))
    if len(dims) > 2:
        raise RuntimeError(f'a gradient of shape {tuple(t.shape)} and strides {t.stride()} does not reduce to two strides')
    (rows, ld, old), (cols, cs, ocs) = dims
    return rows, cols, ld, cs, old, ocs


def _describe(grads, out):
    grads = list(grads)
    if not grads:
        raise RuntimeError('grads must hold at least one tensor')
    outs = grads if out is None else list(out)
    if len(outs) != len(grads):
        raise RuntimeError(f'out must hold {len(grads)} tensors, got {len(outs)}')
    dev = getattr(grads[0], 'device', None)
    arr = (_lib.Grad * len(grads))()
    for i, (t, o) in enumerate(zip(grads, outs)):
        if not (isinstance(t, torch.Tensor) and isinstance(o, torch.Tensor)):
            raise RuntimeError(f'gradient {i} and its output must be tensors, got {type(t).__name__}, {type(o).__name__}')
        if not (t.is_cuda and t.device == dev and t.dtype in _lib.ETYPE and t.layout == torch.strided):
            raise RuntimeError(f'gradient {i} must be a cuda float32, float16 or bfloat16 tensor on {dev}, got {t.dtype} '
                               f'{t.device}')
        if o is not t and not (o.is_cuda and o.device == dev and o.dtype in (t.dtype, torch.float32)
                               and o.shape == t.shape and o.layout == torch.strided):
            raise RuntimeError(f'out {i} must be a cuda {t.dtype} or float32 tensor of shape {tuple(t.shape)} on {dev}')
        n = t.numel()
        if t.is_contiguous() and (o is t or o.is_contiguous()):
            shape = (1, n, n, 1, n, 1)
        else:
            shape = _two_strides(t, o) if n else (0, 0, 0, 0, 0, 0)
        arr[i] = (t.data_ptr(), o.data_ptr(), *shape, _lib.ETYPE[t.dtype], _lib.ETYPE[o.dtype])
    return grads, outs, dev, arr


def _kind(norm_type):
    try:
        return _KINDS[float(norm_type)]
    except (KeyError, TypeError, ValueError):
        raise RuntimeError(f'norm_type must be 1, 2 or inf, got {norm_type!r}') from None


def _run(grads, out, kind, clip):
    r = (_lib._host or _lib.host()).clip(grads, out, kind, *(clip or (None, None)))
    if r != _lib.NOT_TAKEN:
        _lib.check(r[0], 'elr_clip_grad_norm' if clip else 'elr_grad_norm')
        return r[1]
    grads, outs, dev, arr = _describe(grads, out)
    if clip:
        _check_outputs(grads, outs)
    L = _lib.lib()
    n = len(arr)
    nbytes = L.elr_grad_norm_scratch_bytes(arr, n)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    scratch = torch.empty(max(nbytes, 8) // 8, dtype=torch.float64, device=dev)
    with _lib.on_device(dev):
        if clip:
            rc = L.elr_clip_grad_norm(arr, n, kind, *clip, norm.data_ptr(), scratch.data_ptr(), nbytes,
                                      _lib.raw_stream(dev))
        else:
            rc = L.elr_grad_norm(arr, n, kind, norm.data_ptr(), scratch.data_ptr(), nbytes, _lib.raw_stream(dev))
    _lib.check(rc, 'elr_clip_grad_norm' if clip else 'elr_grad_norm')
    return norm


def _same_places(t, o):
    """Whether o is t's memory, element by element."""
    return t.data_ptr() == o.data_ptr() and t.dtype == o.dtype and all(
        a == b for n, a, b in zip(t.shape, t.stride(), o.stride()) if n > 1)


def _check_outputs(grads, outs):
    """Each element is read and scaled once: an output may be its own gradient, and shares no memory with anything else."""
    spans = []                                     # (first byte, end, is an output, number, tensor)
    for i, (t, o) in enumerate(zip(grads, outs)):
        if not t.numel():
            continue
        if _lib.overlaps_itself(o):
            raise RuntimeError(f'output {i} overlaps itself or another: each element is scaled once')
        for x, out in ((o, True),) if o is t or _same_places(t, o) else ((o, True), (t, False)):
            end = x.data_ptr() + x.element_size() * (1 + sum((n - 1) * st for n, st in zip(x.shape, x.stride())))
            spans.append((x.data_ptr(), end, out, i, x))
    spans.sort(key=lambda s: s[:2])
    open_ = []                                     # those that reach to where the next begins
    for s in spans:
        open_ = [q for q in open_ if q[1] > s[0]]
        for q in open_:
            if (q[2] or s[2]) and _lib.overlap(q[4], s[4]):
                if q[2] and s[2]:
                    raise RuntimeError(f'output {q[3]} overlaps itself or another: each element is scaled once')
                o, t = (q, s) if q[2] else (s, q)
                raise RuntimeError(f'output {o[3]} overlaps gradient {t[3]}, in another place or order than its own')
        open_.append(s)


def grad_norm(grads, norm_type=2.0):
    """(sum |g|^p)^(1/p) over every element of every tensor of grads (p = norm_type: 1, 2 or inf), as a float32 scalar on
    the GPU.  grads: cuda float32, float16 or bfloat16 tensors of one device, of any shapes and of strides that reduce to
    two.  Summed in float64; the order of the additions depends on the sizes, strides and alignments alone."""
    return _run(grads, None, _kind(norm_type), None)


def clip_grad_norm(grads, max_norm, norm_type=2.0, eps=1e-6, out=None):
    """Scales grads so that their global norm is at most max_norm, and returns the norm before that (grad_norm's).
    In place, or into out: a list of tensors of grads' shapes, each of its gradient's type or float32 (16-bit gradients
    straight into the float32 rows that gpu_adam reads).  An output may be its own gradient, and shares no memory with another
    output or gradient.  In place a norm of at most max_norm costs no write.  A NaN makes the norm and every gradient NaN; an
    infinite norm scales by 0, unless max_norm is infinite too, which never scales; gradients of nothing but 0 stay."""
    max_norm = float(max_norm)
    if not (max_norm >= 0.0 and eps >= 0.0):
        raise RuntimeError(f'max_norm and eps must be at least 0, got {max_norm} and {eps}')
    return _run(grads, out, _kind(norm_type), (max_norm, float(eps)))
