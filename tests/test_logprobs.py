"""Token log probabilities and their gradient (elara_amd.logprobs) against the definition in 64 bits.  No counterpart in the
reference.

Bounds, with u = 2^-24: an exponential's argument x - m is rounded once and scaled once (2 |x - m| u) and the instruction
adds 2 u; weighted by the exponential itself, |x - m| averages at most log V.  A thread adds at most V / 64 + 32 terms in a
row, and about 16 partial sums are joined, so log s is within (V / 64 + 2 log V + 64) u.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from elara_amd import _lib

U = 2.0 ** -24
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TINY = {torch.float32: 1e-38, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float('inf')


def _lp():
    from elara_amd import logprobs
    return logprobs


def ref_forward(x, tok, k):
    """x [n, V] float64 numpy, tok [n]: (logprob, lse, entropy, top_logprob, top_id) from the definition."""
    n, V = x.shape
    with np.errstate(all='ignore'):
        m = x.max(1, keepdims=True)
        m0 = np.where(m == -np.inf, 0.0, m)
        s = np.exp(x - m0).sum(1, keepdims=True)
        lse = np.where(s == 0, -np.inf, m0 + np.log(s))
        logp = np.where(s == 0, -np.inf, (x - m0) - np.log(s))
        p = np.exp(logp)
        ent = -np.where(p == 0, 0.0, p * logp).sum(1)
        has = (tok >= 0) & (tok < V)
        lp = np.where(has, logp[np.arange(n), np.where(has, tok, 0)], 0.0)
        key = np.where(np.isnan(x), -np.inf, x) + 0.0
        ids = np.argsort(-key, axis=1, kind='stable')[:, :k]
        top = np.take_along_axis(np.where(np.isnan(lse), np.nan, logp), ids, 1)
    return lp, lse[:, 0], ent, top, ids


def ref_backward(x, tok, g, h, z):
    n, V = x.shape
    lp, lse, ent, _, _ = ref_forward(x, tok, 0)
    with np.errstate(all='ignore'):
        m0 = np.where(x.max(1) == -np.inf, 0.0, x.max(1))[:, None]
        logp = (x - m0) - np.log(np.exp(x - m0).sum(1, keepdims=True))
        p = np.where(lse[:, None] == -np.inf, 0.0, np.exp(logp))
        plogp = np.where(p == 0, 0.0, p * logp)
        has = ((tok >= 0) & (tok < V))[:, None]
        hit = (np.arange(V)[None] == tok[:, None]) & has
        d = np.where(has, g[:, None], 0.0) * (hit - p) + z[:, None] * p - h[:, None] * (plogp + p * ent[:, None])
    return np.where(lse[:, None] < -2.0 ** 100, 0.0, d), p, logp, lse, ent     # nothing left by the mask: no gradient


def _same_special(got, ref):
    """Infinite and NaN places are the same; returns the finite places."""
    fin = np.isfinite(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(got[~fin & ~np.isnan(ref)], ref[~fin & ~np.isnan(ref)])
    return fin


def check_forward(x, tok, k, **kw):
    r = _lp().token_logprobs(x, tok, k=k, **kw)
    V = x.shape[-1]
    n = x.numel() // V
    xs, ts = x.double().reshape(n, V).cpu().numpy(), tok.reshape(-1).cpu().numpy().astype(np.int64)
    lp, lse, ent, top, ids = ref_forward(xs, ts, k)
    e = (V / 64 + 2 * math.log(V) + 64) * U
    for got, ref, name in ((r.logprob, lp, 'logprob'), (r.lse, lse, 'lse'), (r.entropy, ent, 'entropy'),
                           (r.top_logprob, top, 'top')):
        if got is None:
            assert k == 0
            continue
        assert got.dtype == torch.float32 and got.shape == tok.shape + ((k,) if name == 'top' else ())
        a = got.double().cpu().numpy().reshape(ref.shape)
        fin = _same_special(a, ref)
        size = np.abs(ref) + (2 + ent if name == 'entropy' else 0) * 0
        bound = (e * (2 + np.abs(ref)) if name == 'entropy' else e) + 4 * U * size
        assert np.all(np.abs(a[fin] - ref[fin]) <= bound[fin]), (name, np.abs(a[fin] - ref[fin]).max())
    if k:
        assert r.top_id.dtype == torch.int64
        assert np.array_equal(r.top_id.cpu().numpy().reshape(n, k), ids)
    return r


def check_backward(x, tok, g, h, z, out=None, special=False):
    V, n = x.shape[-1], x.numel() // x.shape[-1]
    f = _lp().token_logprobs(x, tok)
    xs, ts = x.double().reshape(n, V).cpu().numpy(), tok.reshape(-1).cpu().numpy().astype(np.int64)
    zero = np.zeros(n)
    gs, hs, zs = (zero if t is None else t.double().reshape(-1).cpu().numpy() for t in (g, h, z))
    ref, p, logp, lse, ent = ref_backward(xs, ts, gs, hs, zs)
    d = _lp().token_logprobs_backward(x, tok, f.lse, f.entropy if h is not None else None, g, h, z, out=out)
    assert d.dtype == x.dtype and d.shape == x.shape
    a = d.double().reshape(n, V).cpu().numpy()
    with np.errstate(all='ignore'):
        lp0 = np.where(p == 0, 0.0, np.abs(logp))
        l0 = np.where(np.isfinite(lse), np.abs(lse), 0.0)[:, None]
        e = (V / 64 + 2 * math.log(V) + 64) * U                  # of lse and, times 2 + ent, of the entropy
        mag = p * (np.abs(gs) + np.abs(zs) + np.abs(hs) * ent)[:, None] + p * np.abs(hs)[:, None] * lp0
        bound = mag * (e + (2 * lp0 + 2 * l0 + 16) * U) + p * np.abs(hs)[:, None] * e * (3 + ent[:, None])
        bound = bound + HALF_ULP[x.dtype] * (np.abs(ref) + bound) + 4 * U * np.abs(ref) + TINY[x.dtype] + 1e-37
    fin = _same_special(a, ref) if special else np.isfinite(ref)
    assert fin.all() or special
    assert np.all(np.abs(a - ref)[fin] <= bound[fin]), (np.abs(a - ref) - bound)[fin].max()
    return d


def _randn(dev, seed, *shape, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dev)


SIZES = [(1, 1, 1), (3, 2, 2), (5, 3, 0), (4, 63, 5), (2, 64, 32), (9, 65, 20), (130, 100, 3), (7, 255, 32), (6, 513, 1),
         (5, 1000, 20), (3, 1023, 32), (4, 2047, 5), (3, 2049, 32), (2, 4097, 20), (1, 8193, 8), (1, 16384, 32),
         (2, 40_001, 20), (1, 131_075, 32), (1200, 9001, 4), (70, 20_000, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,V,k', SIZES)
def test_forward(dev, n, V, k, dtype):
    x = _randn(dev, n * V + k, n, V).to(dtype)
    tok = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(1)).to(dev)
    if n > 2:
        tok[1] = -100
        tok[2] = V          # no id either
    check_forward(x, tok, k)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,V', [(1, 1), (3, 2), (4, 63), (5, 513), (9, 1000), (3, 2049), (2, 8195), (1, 40_001), (600, 300)])
@pytest.mark.parametrize('parts', ['g', 'h', 'gh', 'ghz'])
def test_backward(dev, n, V, dtype, parts):
    x = _randn(dev, n * V, n, V).to(dtype)
    tok = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(2)).to(dev)
    if n > 2:
        tok[1] = -1
        tok[2] = V + 7
    g, h, z = (_randn(dev, j, n, scale=1.0) if c in parts else None for j, c in enumerate('ghz'))
    check_backward(x, tok, g, h, z)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('V', [50, 700, 9000, 40_000])
def test_masked_rows(dev, V, dtype):
    """-inf and the type's lowest value in masked places, rows left with few ids or none, and their gradients."""
    low = torch.finfo(dtype).min
    x = _randn(dev, V, 9, V).to(dtype)
    x[0, V // 3:] = -INF
    x[1] = -INF                                 # nothing left
    x[2] = low
    x[2, V // 2] = 1.0                          # one id left, the others at the lowest value
    x[3] = -INF
    x[3, V - 1] = -3.0                          # one id left
    x[4] = low                                  # nothing left: uniform, but no gradient in float32 and bfloat16
    x[5, ::2] = low
    x[6, 5:] = -INF
    x[7] = torch.finfo(dtype).max               # uniform, at the largest value
    tok = torch.tensor([0, 3, V // 2, V - 1, 7, 1, 20, 2, 4], device=dev)
    check_forward(x, tok, 32)
    r = _lp().token_logprobs(x, tok, k=4)
    assert r.lse[1] == -INF and r.logprob[1] == -INF and r.entropy[1] == 0 and r.logprob[6] == -INF
    assert r.top_id[1].tolist() == [0, 1, 2, 3]
    g, h = _randn(dev, 3, 9, scale=1.0), _randn(dev, 4, 9, scale=1.0)
    d = check_backward(x, tok, g, h, None)
    assert not d[1].any() and torch.isfinite(d).all()


def check_offset_backward(x, tok, g, h, z, out=None):
    """check_backward with lse's own rounding taken no further than |lse| = 256: a row's common offset costs nothing."""
    n, V = x.shape
    f = _lp().token_logprobs(x, tok)
    xs, ts = x.double().cpu().numpy(), tok.cpu().numpy().astype(np.int64)
    gs, hs, zs = (t.double().cpu().numpy() for t in (g, h, z))
    ref, p, logp, lse, ent = ref_backward(xs, ts, gs, hs, zs)
    d = _lp().token_logprobs_backward(x, tok, f.lse, f.entropy, g, h, z, out=out)
    a = d.double().cpu().numpy()
    lp0, l0 = np.where(p == 0, 0.0, np.abs(logp)), np.minimum(np.abs(lse), 256.0)[:, None]
    e = (V / 64 + 2 * math.log(V) + 64) * U
    mag = p * (np.abs(gs) + np.abs(zs) + np.abs(hs) * ent)[:, None] + p * np.abs(hs)[:, None] * lp0
    bound = mag * (e + (2 * lp0 + 2 * l0 + 16) * U) + p * np.abs(hs)[:, None] * e * (3 + ent[:, None])
    bound = bound + HALF_ULP[x.dtype] * (np.abs(ref) + bound) + 4 * U * np.abs(ref) + TINY[x.dtype] + 1e-37
    assert np.all(np.abs(a - ref) <= bound), (np.abs(a - ref) - bound).max(1)
    return d


OFFSETS = {torch.float32: (-1e30, -1e9, -65_504.0, -255.0, 300.0, 1e6, 1e20), torch.bfloat16: (-1e30, -1e9, -3e4, 255.0, 300.0, 1e6),
           torch.float16: (-65_504.0, -65_000.0, -300.0, 260.0, 2e4, 65_504.0)}


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('V', [1, 2, 63, 300, 513, 1025, 4000, 9001, 40_003])
def test_backward_of_rows_with_an_offset(dev, V, dtype):
    """Rows of a large common offset, of which lse keeps few digits of log V or none: rows that a mask of -1e9 or the like left
    nothing of (alike in every place), and spread ones; with and without a token, in place, unaligned and over row strides."""
    low, rows = torch.finfo(dtype).min, []
    for i, c in enumerate(OFFSETS[dtype]):
        flat = torch.full((V,), c)
        near = (c + torch.randn(V, generator=torch.Generator().manual_seed(V + i)) * 2.5).clamp(low, -low)
        some = torch.where(torch.arange(V) % 3 == 0, near, torch.tensor(low))      # two of three masked
        rows += [flat, flat, near, near, some]
    x = torch.stack(rows).to(dtype).to(dev)
    n = x.shape[0]
    tok = (torch.arange(n) * 7 % V).to(dev)
    tok[::5] = -1                                                                  # one of each flat pair is ignored
    g, h, z = (_randn(dev, j, n, scale=1.0) for j in range(3))
    want = check_offset_backward(x, tok, g, h, z)
    y = x.clone()
    assert torch.equal(check_offset_backward(y, tok, g, h, z, out=y), want)
    buf = torch.zeros(n, V + 13, dtype=dtype, device=dev)
    buf[:, 5:5 + V] = x
    want = check_offset_backward(buf[:, 5:5 + V], tok, g, h, z, out=torch.empty_like(buf)[:, 5:5 + V])
    got = check_offset_backward(buf[:, 5:5 + V], tok, g, h, z, out=buf[:, 5:5 + V])      # (the order of sums goes by alignment)
    assert torch.equal(got, want) and not buf[:, :5].any() and not buf[:, 5 + V:].any()


@pytest.mark.gpu
@pytest.mark.parametrize('offset', [0.0, 1000.0])
def test_backward_with_the_lse_of_more_logits(dev, offset):
    """An lse over a wider row than these logits (here twice as many) is used as it is; it errs by its rounding, at most
    1013 * 2^-24 of p, beside the forward's and the exponential's bounds."""
    lp = _lp()
    V = 5000
    x = _randn(dev, 1, 6, 2 * V) + offset
    tok = torch.full((6,), -1, device=dev)
    f = lp.token_logprobs(x, tok)
    z = torch.ones(6, device=dev)
    d = torch.cat([lp.token_logprobs_backward(x[:, :V], tok, f.lse, None, None, d_lse=z),
                   lp.token_logprobs_backward(x[:, V:], tok, f.lse, None, None, d_lse=z)], 1).double()
    ref = torch.softmax(x.double(), -1)
    e = (2 * V / 64 + 2 * math.log(2 * V) + 64) * U
    assert bool(((d - ref).abs() <= ref * (e + (2 * 30 + 2 * 1013 + 16) * U) + 1e-37).all())


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('V', [100, 3000, 50_000])
def test_nan_and_inf(dev, V, dtype):
    x = _randn(dev, V, 5, V).to(dtype)
    x[0, 17] = float('nan')
    x[1, 0] = INF
    x[2] = -INF
    x[2, 4] = float('nan')
    x[3] = float('nan')
    tok = torch.tensor([1, 0, 4, 2, 3], device=dev)
    r = check_forward(x, tok, 10)
    assert torch.isnan(r.lse[:4]).all() and torch.isnan(r.logprob[:4]).all() and torch.isfinite(r.lse[4])
    f = _lp().token_logprobs(x, tok)
    one = torch.ones(5, device=dev)
    d = _lp().token_logprobs_backward(x, tok, f.lse, f.entropy, one, one, one)
    assert torch.isnan(d[:4]).all() and torch.isfinite(d[4]).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('V', [64, 1500, 8191, 40_000, 140_000])
@pytest.mark.parametrize('kind', ['zeros', 'ascending', 'descending', 'steps', 'negative', 'signed zeros', 'few values',
                                  'one thread', 'close'])
def test_top_order(dev, V, dtype, kind):
    """Rows whose candidates crowd: equal values, sorted rows, rows whose large elements all belong to a few threads."""
    i = torch.arange(V, dtype=torch.float32)
    x = {'zeros': i * 0, 'ascending': i * 2.0 ** -12, 'descending': -i * 2.0 ** -12, 'steps': torch.floor(i / 777) * 0.5,
         'negative': -1.5 - (i % 3), 'signed zeros': torch.where(i % 2 == 0, -0.0, 0.0),
         'few values': ((i * 7919) % 5) * 0.25, 'one thread': torch.where((i / 8).floor() % 256 < 12, 5.0 + (i % 64) / 64, -9.0),
         'close': 3.0 + ((i * 7919) % V) * 2.0 ** -22}[kind].to(dtype).to(dev)[None].repeat(2, 1)
    tok = torch.tensor([0, V - 1], device=dev)
    check_forward(x, tok, 32)
    check_forward(x, tok, 1)


@pytest.mark.gpu
def test_layouts(dev):
    """Padded vocabularies, broadcast rows, transposed logits, leading dimensions, unaligned bases, int32 tokens."""
    lp = _lp()
    base = _randn(dev, 1, 6, 1031).to(torch.bfloat16)
    tok = torch.tensor([0, 5, 1000, 7, 999, 3], device=dev)
    check_forward(base[:, 3:1004], tok, 7)                              # rows 1031 apart, base not 4-byte aligned
    check_forward(base[:1, :1001].expand(6, 1001), tok, 7)              # stride 0
    check_forward(base[:, :1001].t().contiguous().t(), tok, 7)          # last stride not 1
    check_forward(base[:, :1002].reshape(2, 3, 1002), tok.view(2, 3).to(torch.int32), 5)
    check_forward(base[::2, :1001], tok[::2], 5)                        # strided tokens
    one = torch.ones(6, device=dev)
    check_backward(base[:, 3:1004], tok, one, one, one)
    x = base[:, 1:1001]
    buf = torch.full((6, 1100), 7.0, dtype=torch.bfloat16, device=dev)
    d = check_backward(x, tok, one, None, None, out=buf[:, 5:1005])     # rows apart by another stride
    assert d.data_ptr() == buf[:, 5:1005].data_ptr() and (buf[:, :5] == 7).all() and (buf[:, 1005:] == 7).all()
    want = check_backward(x, tok, one, None, None)
    f = lp.token_logprobs(x, tok)
    y = base.clone()
    got = lp.token_logprobs_backward(y[:, 1:1001], tok, f.lse, None, one, out=y[:, 1:1001])    # over the logits
    assert torch.equal(got, want) and torch.equal(y[:, 1001:], base[:, 1001:]) and torch.equal(y[:, 0], base[:, 0])
    e = lp.token_logprobs(base[:0, :10], tok[:0], k=2)
    assert e.logprob.shape == (0,) and e.top_id.shape == (0, 2)
    assert lp.token_logprobs_backward(base[:0, :10], tok[:0], e.lse, None, e.lse).shape == (0, 10)


@pytest.mark.gpu
@pytest.mark.parametrize('V', [40, 3000])
def test_gradient_against_differences(dev, V):
    """A directional derivative of the forward kernel itself.  The central difference of step s errs by s^2 / 6 times the
    third derivative (at most 8 * sum |v|^3-like terms, below 40 here) and by the forward's error over s."""
    lp = _lp()
    n, s = 6, 2.0 ** -6
    x = _randn(dev, V, n, V, scale=1.0)
    v = _randn(dev, V + 1, n, V, scale=1.0).clamp(-1, 1)
    tok = torch.arange(n, device=dev) * 5
    g, h, z = (_randn(dev, j, n, scale=1.0).clamp(-1, 1) for j in range(3))

    def f(y):
        r = lp.token_logprobs(y, tok)
        return (g.double() * r.logprob.double() + h.double() * r.entropy.double() + z.double() * r.lse.double())
    r = lp.token_logprobs(x, tok)
    d = lp.token_logprobs_backward(x, tok, r.lse, r.entropy, g, h, z)
    dot = (d.double() * v.double()).sum(1)
    diff = (f(x + s * v) - f(x - s * v)) / (2 * s)
    err = (V / 64 + 2 * math.log(V) + 64) * U * 40 / s + 40 * s * s / 6
    assert float((dot - diff).abs().max()) < err


@pytest.mark.gpu
@pytest.mark.parametrize('V', [40, 3000])
@pytest.mark.parametrize('part', ['logprob', 'entropy', 'lse'])
def test_each_gradient_along_its_own_sign(dev, V, part):
    """One output at a time, along the signs of its reference gradient: the derivative is that gradient's 1-norm, more than ten
    times what the difference may err by, so a term that is missing, halved or turned round fails.  With |v| <= 1 the third
    derivatives are sums of cumulants of v and x: at most 8 for logprob and lse, 2 * 8 + 32 E|x - E x| < 80 for the entropy.
    The forward's error is e (2 + entropy) + 4 u |f| (|f| < 13) at each end, the ends' rounding 4.5 u of each logit."""
    lp = _lp()
    n, s = 6, 2.0 ** -6
    x = _randn(dev, V, n, V, scale=1.0)
    tok = torch.arange(n, device=dev) * 5
    ones, none = torch.ones(n, device=dev), np.zeros(n)
    which = [part == p for p in ('logprob', 'entropy', 'lse')]
    ref = ref_backward(x.double().cpu().numpy(), tok.cpu().numpy(), *(none + w for w in which))[0]
    v = torch.from_numpy(np.sign(ref)).float().to(dev)
    r = lp.token_logprobs(x, tok)
    d = lp.token_logprobs_backward(x, tok, r.lse, r.entropy, *(ones if w else None for w in which))

    def f(y):
        return getattr(lp.token_logprobs(y, tok), part).double()
    dot = (d.double() * v.double()).sum(1)
    diff = (f(x + s * v) - f(x - s * v)) / (2 * s)
    e = (V / 64 + 2 * math.log(V) + 64) * U
    err = (e * (2 + math.log(V)) + 4 * 13 * U + 2 * 4.5 * U) / s + 80 * s * s / 6
    assert float((dot - diff).abs().max()) < err
    assert float(diff.abs().min()) > 10 * err


@pytest.mark.gpu
def test_offsets_beyond_32_bits(dev):
    """The last rows of 2.2 * 10^9 logits: element offsets past 2^31, byte offsets past 2^32."""
    lp = _lp()
    n, V = 17_001, 131_072
    x = torch.zeros(n, V, dtype=torch.bfloat16, device=dev)
    x[-2:] = _randn(dev, 3, 2, V).to(torch.bfloat16)
    tok = torch.full((n,), -1, device=dev)
    tok[-2:] = torch.tensor([5, V - 1], device=dev)
    r = lp.token_logprobs(x, tok, k=3)
    want = check_forward(x[-2:].contiguous(), tok[-2:], 3)
    assert torch.equal(r.top_id[-2:], want.top_id)
    assert float((r.lse[-2:] - want.lse).abs().max()) < 1e-4    # the same row split differently: twice the bound
    one = torch.ones(n, device=dev)
    d = lp.token_logprobs_backward(x, tok, r.lse, None, one, out=x)
    assert abs(float(d[-1].double().sum())) < 2.0 ** -8 and float(d[-1, V - 1]) > 0 and not d[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize('k', [0, 2])
def test_more_rows_than_a_launch(dev, k):
    """33,554,437 rows of three logits: several launches forward and backward, the same bits as the rows by themselves."""
    lp = _lp()
    n = (1 << 25) + 5
    x = _randn(dev, 1, 1 << 16, 3).to(torch.bfloat16).repeat((1 << 9) + 1, 1)[:n]
    tok = torch.arange(n, device=dev, dtype=torch.int32) % 3
    r = lp.token_logprobs(x, tok, k=k)
    one = torch.ones(n, device=dev)
    d = lp.token_logprobs_backward(x, tok, r.lse, None, one)
    for a in (0, (1 << 22) - 2, 1 << 24, n - 7):
        s = slice(a, a + 7)
        want = lp.token_logprobs(x[s].clone(), tok[s].clone(), k=k)
        assert all(torch.equal(p[s], q) for p, q in zip(r, want) if p is not None)
        assert torch.equal(d[s], lp.token_logprobs_backward(x[s].clone(), tok[s].clone(), want.lse, None, one[s].clone()))

@pytest.mark.gpu
def test_streams_and_graph(dev):
    """The same results on a side stream, and from every replay of a captured graph on changed logits."""
    lp = _lp()
    x = _randn(dev, 1, 3, 50_000).to(torch.bfloat16)
    tok = torch.tensor([3, 4, 49_999], device=dev)
    one = torch.ones(3, device=dev)

    def both():
        r = lp.token_logprobs(x, tok, k=9)
        return [*r, lp.token_logprobs_backward(x, tok, r.lse, r.entropy, one, one)]
    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for seed in range(4):
        x.copy_(_randn(dev, 10 + seed, 3, 50_000))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, both())), seed


@pytest.mark.gpu
def test_with_and_without_host_module(dev, monkeypatch):
    """The native argument checks and the Python ones make the same call."""
    lp = _lp()
    x = _randn(dev, 1, 2, 5, 3001).to(torch.bfloat16)
    tok = torch.randint(0, 3001, (2, 5), generator=torch.Generator().manual_seed(1)).to(dev)
    one = torch.ones(2, 5, device=dev)

    def run():
        r = lp.token_logprobs(x, tok, k=3)
        none = lp.token_logprobs(x, tok.to(torch.int32))
        assert none.top_id is None and none.top_logprob is None
        out = torch.empty_like(x)
        assert lp.token_logprobs_backward(x, tok, r.lse, None, one, out=out) is out
        return [*r, none.logprob, out, lp.token_logprobs_backward(x, tok, r.lse, r.entropy, one, one, one)]
    want = run()
    calls = []
    monkeypatch.setattr(_lib, '_host', _lib._NoHost)
    monkeypatch.setattr(_lib, 'check', lambda rc, what, f=_lib.check: (calls.append(what), f(rc, what)))
    got = run()
    assert len(calls) == 4 and all(a.shape == b.shape and torch.equal(a, b) for a, b in zip(got, want))

@pytest.mark.gpu
def test_refusals(dev):
    lp = _lp()
    x = torch.zeros(4, 50, device=dev)
    tok = torch.zeros(4, dtype=torch.int64, device=dev)
    f = lp.token_logprobs(x, tok)
    for bad in (lambda: lp.token_logprobs(x.cpu(), tok), lambda: lp.token_logprobs(x.double(), tok),
                lambda: lp.token_logprobs(x, tok.cpu()), lambda: lp.token_logprobs(x, tok.float()),
                lambda: lp.token_logprobs(x, tok[:3]), lambda: lp.token_logprobs(x, tok, k=33),
                lambda: lp.token_logprobs(x, tok, k=-1), lambda: lp.token_logprobs(x[:, :5], tok, k=6),
                lambda: lp.token_logprobs(x[:, :0], tok),
                lambda: lp.token_logprobs_backward(x, tok, None, None, f.lse),
                lambda: lp.token_logprobs_backward(x, tok, f.lse.double(), None, f.lse),
                lambda: lp.token_logprobs_backward(x, tok, f.lse, None, f.lse, d_entropy=f.lse),
                lambda: lp.token_logprobs_backward(x, tok, f.lse, None, f.lse[:3]),
                lambda: lp.token_logprobs_backward(x, tok, f.lse, None, f.lse, out=x.half()),
                lambda: lp.token_logprobs_backward(x, tok, f.lse, None, f.lse, out=x[:1].expand(4, 50)),
                lambda: lp.token_logprobs_backward(x, tok, f.lse, None, f.lse, out=torch.zeros(50, 4, device=dev).t())):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(IndexError):
        lp.token_logprobs(x, tok + 50, check=True)
    lp.token_logprobs(x, tok - 100, check=True)


@pytest.mark.gpu
@pytest.mark.parametrize('native', [True, False])
def test_out_that_overlaps_the_logits(dev, monkeypatch, native):
    """Refused unless it is the logits themselves; other columns of the same rows, or the memory of logits that were copied
    for their strides, are taken."""
    lp = _lp()
    if not native:
        monkeypatch.setattr(_lib, '_host', _lib._NoHost)
    flat = _randn(dev, 1, 1100)
    keep = flat.clone()
    x, tok = flat[:1000].view(10, 100), torch.arange(10, device=dev)
    r = lp.token_logprobs(x, tok)
    one = torch.ones(10, device=dev)
    wide = flat[:1080].view(10, 108)
    for logits, out in ((x, flat[4:1004].view(10, 100)), (x, flat[100:].view(10, 100)), (wide[:, :100], wide[:, 8:]),
                        (wide[:, :100], wide[:, 1:101]), (x[:1].expand(10, 100), x), (x, flat[:1080].view(10, 108)[:, :100])):
        with pytest.raises(RuntimeError, match='out must be'):
            lp.token_logprobs_backward(logits, tok, r.lse, None, one, out=out)
        assert torch.equal(flat, keep)
    half = flat[:1000].view(5, 200)
    f = lp.token_logprobs(half[:, :100], tok[:5])
    want = lp.token_logprobs_backward(half[:, :100].contiguous(), tok[:5], f.lse, None, one[:5])
    got = lp.token_logprobs_backward(half[:, :100], tok[:5], f.lse, None, one[:5], out=half[:, 100:])
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-7) and torch.equal(half[:, :100], keep[:1000].view(5, 200)[:, :100])
    sq = flat[:900].view(30, 30)
    f = lp.token_logprobs(sq.t(), tok[0].expand(30))
    want = lp.token_logprobs_backward(sq.t().contiguous(), tok[0].expand(30), f.lse, None, one[0].expand(30))
    assert torch.equal(lp.token_logprobs_backward(sq.t(), tok[0].expand(30), f.lse, None, one[0].expand(30), out=sq), want)


def test_cabi_refusals():
    """Arguments that the library refuses on the host (none of these calls reaches the GPU)."""
    L = _lib.lib()
    p = ctypes.c_void_p(256)

    def fwd(x=p, type=0, n=4, V=100, ld=100, tok=p, k=2, a=p, b=p, c=p, d=p, e=p, s=None, sb=0):
        return L.elr_token_logprobs(x, type, n, V, ld, tok, 1, k, a, b, c, d, e, s, sb, None)

    def bwd(x=p, type=0, n=4, V=100, ld=100, tok=p, lse=p, ent=None, g=p, h=None, z=None, out=p, old=100):
        return L.elr_token_logprobs_backward(x, type, n, V, ld, tok, 1, lse, ent, g, h, z, out, old, None)
    assert fwd(n=0, x=None) == 0 and bwd(n=0, x=None) == 0
    for rc in (fwd(x=None), fwd(type=3), fwd(n=-1), fwd(V=0), fwd(ld=-1), fwd(tok=None), fwd(k=-1), fwd(k=101), fwd(a=None),
               fwd(b=None), fwd(c=None), fwd(d=None), fwd(e=None), fwd(x=ctypes.c_void_p(258)),
               bwd(x=None), bwd(type=-1), bwd(lse=None), bwd(out=None), bwd(old=99), bwd(h=p), bwd(tok=None),
               bwd(out=ctypes.c_void_p(257), type=2)):
        assert rc == -1
    assert fwd(V=1000, ld=1000, k=33) == -2 and fwd(V=(1 << 30) + 1) == -2
    need = L.elr_token_logprobs_scratch_bytes(1, 131_072, 20)
    assert need > 0 and L.elr_token_logprobs_scratch_bytes(100_000, 131_072, 20) == 0
    assert L.elr_token_logprobs_scratch_bytes(1, 0, 0) == -1 and L.elr_token_logprobs_scratch_bytes(1, 50, 33) == -1
    assert fwd(n=1, V=131_072, ld=131_072, k=20) == -3
    assert fwd(n=1, V=131_072, ld=131_072, k=20, s=p, sb=need - 1) == -3
    assert fwd(n=1, V=131_072, ld=131_072, k=20, s=ctypes.c_void_p(260), sb=need) == -3


def test_python_refuses_host_tensors():
    lp = _lp()
    with pytest.raises(RuntimeError, match='logits must be a cuda'):
        lp.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match='logits must be a cuda'):
        lp.token_logprobs_backward(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64), None, None, None)
