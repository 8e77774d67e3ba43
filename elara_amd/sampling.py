"""A token for each row of logits, drawn with temperature, top-k, top-p and min-p from given uniform numbers: the answer of a model
whose likeliest ids logprobs.token_logprobs lists.  No counterpart in the reference.

    sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> Sample    the ids and their log probabilities

It runs the HIP kernel behind elr_sample_tokens (elara_amd/csrc/sampling.hip) on torch's current stream: one launch, no workspace, no
host synchronisation.  The numbers are the caller's (torch.rand with a generator of its own), so a draw can be repeated; the same
inputs give the same ids on every call.
"""
import operator
from typing import NamedTuple

import torch

from . import _lib
from .logprobs import _ld, _logits2d


class Sample(NamedTuple):
    token: torch.Tensor      # int64, u's shape
    logprob: torch.Tensor    # float32, u's shape: the token's log probability among the kept ones


def _setting(v, u, name, dtypes, low, high):
    """(value, None) for a number in [low, high] (a whole one for integer types), (0, tensor) for one value a row."""
    if torch.is_tensor(v):
        if not (v.is_cuda and v.device == u.device and v.dtype in dtypes and v.shape == u.shape):
            raise RuntimeError(f'{name} must be a number or a cuda {" or ".join(map(str, dtypes))} tensor of shape '
                               f'{tuple(u.shape)} on {u.device}')
        return 0, v.contiguous()
    try:
        v = float(v) if dtypes == (torch.float32,) else operator.index(v)
    except (TypeError, ValueError):
        raise RuntimeError(f'{name} must be {"a number" if dtypes == (torch.float32,) else "a whole number"}, got {v!r}') from None
    if not low <= v <= high:
        raise RuntimeError(f'{name} must lie in [{low}, {high}], got {v}')
    return v, None


def sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """logits [..., V] cuda float32/float16/bfloat16 (any row stride); u float32 [...] in [0, 1), a number for each row.  Each setting
    is a number, or a tensor of u's shape with one for each row (float32; top_k int32 or int64).  With e = exp((x - max) / temperature)
    and the order of larger logits first, ties by the lower id:

      top_k   keeps the first so many of the order (0, or V and more: all);
      top_p   of these, those before which in the order less than top_p of their mass lies (1: all; the first always stays);
      min_p   of these, those with e >= min_p, i.e. at least that share of the largest probability (0: all).

    The token is the first kept id, by rising id, at which the running sum of e exceeds u times the whole; logprob is log(e / whole).
    temperature = 0 takes the first of the order, with logprob 0.  Sums are exact and the same for every launch; an e below
    2^-(s + 1) of the largest, s = min(51, 62 - ceil(log2 V)), is never drawn (2^-46 at V = 131,072).  -inf marks banned ids: a row
    of nothing else has token -1 and logprob -inf.  A row with a NaN or +inf, and one whose temperature (in a tensor) is negative or NaN or whose u is NaN, has token -1 and logprob NaN; other
    per-row settings out of range count as the nearest in it, a NaN as no limit."""
    r = (_lib._host or _lib.host()).sample(logits, u, temperature, top_k, top_p, min_p)
    if r != _lib.NOT_TAKEN:
        _lib.check(r[0], 'elr_sample_tokens')
        return Sample(r[1], r[2])
    x = _logits2d(logits, 'logits')
    if not (u.is_cuda and u.device == logits.device and u.dtype == torch.float32 and u.shape == logits.shape[:-1]):
        raise RuntimeError(f'u must be a cuda float32 tensor of shape {tuple(logits.shape[:-1])} on {logits.device}')
    n, V = x.shape
    dev = logits.device
    temp, temps = _setting(temperature, u, 'temperature', (torch.float32,), 0.0, torch.finfo(torch.float64).max)
    k, ks = _setting(top_k, u, 'top_k', (torch.int32, torch.int64), 0, (1 << 63) - 1)
    p, ps = _setting(top_p, u, 'top_p', (torch.float32,), 0.0, 1.0)
    mp, mps = _setting(min_p, u, 'min_p', (torch.float32,), 0.0, 1.0)
    un = u.contiguous()
    token = torch.empty(u.shape, dtype=torch.int64, device=dev)
    logprob = torch.empty(u.shape, dtype=torch.float32, device=dev)
    if n:
        with _lib.on_device(dev):
            rc = _lib.lib().elr_sample_tokens(
                x.data_ptr(), _lib.ETYPE[x.dtype], n, V, _ld(x), un.data_ptr(), temp, _lib.ptr(temps), k, _lib.ptr(ks),
                int(ks is not None and ks.dtype == torch.int64), p, _lib.ptr(ps), mp, _lib.ptr(mps), token.data_ptr(),
                logprob.data_ptr(), _lib.raw_stream(dev))
        _lib.check(rc, 'elr_sample_tokens')
    return Sample(token, logprob)
