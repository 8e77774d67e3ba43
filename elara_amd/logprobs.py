"""Log probabilities of given tokens over rows of logits: the loss of a model that predicts one of V ids, with its
gradient, and the scores of the same model when it serves.  No counterpart in the reference (its models end in a
sigmoid, srm2/models.py).

    token_logprobs(logits, tokens, k=0) -> TokenLogprobs     log probability of each row's token, log-sum-exp, entropy,
                                                             and the k likeliest ids
    token_logprobs_backward(logits, tokens, lse, entropy, d_logprob, d_entropy=None, d_lse=None, out=None)
                                                             the gradient to the logits

Both run the HIP kernels behind elr_token_logprobs and elr_token_logprobs_backward (elara_amd/csrc/logprobs.hip) on torch's
current stream, without a host synchronisation.  The row is read once, and with k a few of its places again (all of it where the
large logits crowd).  Neither registers with autograd: results are detached, and what is written into `out` bumps no version.
"""
from typing import NamedTuple, Optional

import torch

from . import _lib

TOPK_MAX = 32   # ELR_TOPK_MAX


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                    # float32, tokens' shape
    lse: torch.Tensor                        # float32, tokens' shape
    entropy: torch.Tensor                    # float32, tokens' shape, in nats
    top_logprob: Optional[torch.Tensor]      # float32, tokens' shape + (k,); None with k = 0
    top_id: Optional[torch.Tensor]           # int64, tokens' shape + (k,)


def _logits2d(t, name):
    """t [..., V] as [n, V] rows a fixed stride apart (a copy only where the strides allow nothing else)."""
    if not (t.is_cuda and t.dtype in _lib.ETYPE and t.dim() >= 1 and t.shape[-1] >= 1):
        raise RuntimeError(f'{name} must be a cuda float32, float16 or bfloat16 tensor [..., V], got {tuple(t.shape)} '
                           f'{t.dtype} {t.device}')
    x = t if t.dim() == 2 else t.reshape(t.numel() // t.shape[-1], t.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _ld(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _tokens(tokens, logits):
    if not (tokens.is_cuda and tokens.device == logits.device and tokens.dtype in (torch.int32, torch.int64)):
        raise RuntimeError(f'tokens must be a cuda int32/int64 tensor on {logits.device}')
    if tokens.shape != logits.shape[:-1]:
        raise RuntimeError(f'tokens must have shape {tuple(logits.shape[:-1])}, got {tuple(tokens.shape)}')
    return tokens.contiguous()


def token_logprobs(logits, tokens, k=0, check=False):
    """logits [..., V] cuda float32/float16/bfloat16 (any row stride), tokens int32/int64 [...]: one id per row.  All
    arithmetic is float32.  A token outside [0, V) marks a row without one (padding, a masked position): its logprob is 0;
    check=True raises IndexError for a token >= V first, at the cost of a host synchronisation.  A row of nothing but -inf
    has logprob and lse -inf and entropy 0.  k (at most 32 and at most V): that many largest logits' ids, larger first and
    ties by the lower id, with their log probabilities."""
    if not check:
        r = (_lib._host or _lib.host()).logprobs(logits, tokens, k)
        if r != _lib.NOT_TAKEN:
            _lib.check(r[0], 'elr_token_logprobs')
            return TokenLogprobs(*r[1:])
    x = _logits2d(logits, 'logits')
    tok = _tokens(tokens, logits)
    n, V = x.shape
    k = int(k)
    if not 0 <= k <= min(V, TOPK_MAX):
        raise RuntimeError(f'k must lie in [0, min(V, {TOPK_MAX})], got {k} with V = {V}')
    if check and n and int(tok.max()) >= V:
        raise IndexError(f'tokens out of range: {int(tok.max())} not below {V}')
    dev, shape = logits.device, tokens.shape
    L = _lib.lib()
    nbytes = L.elr_token_logprobs_scratch_bytes(n, V, k)
    sums = torch.empty((3,) + shape, dtype=torch.float32, device=dev)
    top_lp = torch.empty(shape + (k,), dtype=torch.float32, device=dev) if k else None
    top_id = torch.empty(shape + (k,), dtype=torch.int64, device=dev) if k else None
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    logprob, lse, entropy = sums.unbind(0)
    if n:
        with _lib.on_device(dev):
            rc = L.elr_token_logprobs(x.data_ptr(), _lib.ETYPE[x.dtype], n, V, _ld(x), tok.data_ptr(),
                                      int(tok.dtype == torch.int64), k, logprob.data_ptr(), lse.data_ptr(),
                                      entropy.data_ptr(), _lib.ptr(top_lp), _lib.ptr(top_id), _lib.ptr(scratch), nbytes,
                                      _lib.raw_stream(dev))
        _lib.check(rc, 'elr_token_logprobs')
    return TokenLogprobs(logprob, lse, entropy, top_lp, top_id)


def _per_row(t, like, name):
    if t is None:
        return None
    if not (t.is_cuda and t.device == like.device and t.dtype == torch.float32 and t.shape == like.shape):
        raise RuntimeError(f'{name} must be a cuda float32 tensor of shape {tuple(like.shape)} on {like.device}')
    return t.contiguous()


def token_logprobs_backward(logits, tokens, lse, entropy, d_logprob, d_entropy=None, d_lse=None, out=None):
    """The gradient to the logits of sum(d_logprob * logprob + d_entropy * entropy + d_lse * lse), in the logits' type and
    shape.  lse and entropy are token_logprobs' (entropy may be None without d_entropy); d_* are float32 of tokens' shape,
    None for zero.  Rows without a token get nothing from d_logprob; rows of nothing but -inf, or nothing but
    float32's or bfloat16's lowest value, get 0.  Where |lse| is 256 or more (a large offset common to the row) lse's last
    digits no longer tell p, and the row's sum is taken again (a slower pass over it).  out: where to write it, a
    tensor of the logits' shape and type whose rows lie apart by a fixed stride; the logits themselves are allowed, and are
    then overwritten, but no other memory of theirs."""
    r = (_lib._host or _lib.host()).logprobs_back(logits, tokens, lse, entropy, d_logprob, d_entropy, d_lse, out)
    if r != _lib.NOT_TAKEN:
        _lib.check(r[0], 'elr_token_logprobs_backward')
        return r[1]
    x = _logits2d(logits, 'logits')
    tok = _tokens(tokens, logits)
    n, V = x.shape
    lse = _per_row(lse, tok, 'lse')
    if lse is None:
        raise RuntimeError('lse is needed')
    d_logprob, d_entropy, d_lse = (_per_row(t, tok, m) for t, m in ((d_logprob, 'd_logprob'), (d_entropy, 'd_entropy'),
                                                                   (d_lse, 'd_lse')))
    entropy = _per_row(entropy, tok, 'entropy') if d_entropy is not None else None
    if d_entropy is not None and entropy is None:
        raise RuntimeError('entropy is needed for d_entropy')
    dev = logits.device
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    elif not (out.is_cuda and out.device == dev and out.dtype == logits.dtype and out.shape == logits.shape):
        raise RuntimeError(f'out must be a cuda {logits.dtype} tensor of shape {tuple(logits.shape)} on {dev}')
    if n == 0:
        return out
    o = out if out.dim() == 2 else out.view(n, V)      # (view raises where no fixed row stride exists)
    if (V > 1 and o.stride(1) != 1) or (n > 1 and o.stride(0) < V):
        raise RuntimeError('out must have contiguous rows that do not overlap')
    if (o.data_ptr(), _ld(o)) != (x.data_ptr(), _ld(x)) and _lib.overlap(o, x):
        raise RuntimeError('out must be the logits themselves or share no memory with them')
    with _lib.on_device(dev):
        rc = _lib.lib().elr_token_logprobs_backward(
            x.data_ptr(), _lib.ETYPE[x.dtype], n, V, _ld(x), tok.data_ptr(), int(tok.dtype == torch.int64), _lib.ptr(lse),
            _lib.ptr(entropy), _lib.ptr(d_logprob), _lib.ptr(d_entropy), _lib.ptr(d_lse), o.data_ptr(), _ld(o),
            _lib.raw_stream(dev))
    _lib.check(rc, 'elr_token_logprobs_backward')
    return out
