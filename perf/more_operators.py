"""Operators in 8-bit integers and the draw of a token, measured through the framework's entry points.

Kinds of case (the field "kind"):
  sample     sampling.sample_tokens: a token for each row of logits by temperature, top-k, top-p and min-p from a given
             uniform number, and its log probability in the distribution that it was drawn from
  linear     int8.linear: the product of int8 rows with an int8 weight, a scale for each token and each channel
  ckpt       int8.quantize and int8.dequantize: an activation kept in 8 bits by the forward pass and widened again
  norm_back  norms.rms_norm_backward_int8: the RMS norm's backward pass from its input kept in 8 bits
  wgrad      int8.weight_grad: a linear layer's weight gradient from its input kept in 8 bits

Sizes: the widths, batches and vocabularies of the examples and of perf/operators.py, and generic model widths.  The plain
forms below compute in 32 bits and round once at the end (the draw in 64: a cumulative sum next to its border); exact()
computes in 64 bits.
"""
import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
ESIZE = {'f32': 4, 'bf16': 2, 'f16': 2}
EPS = 1e-6
NEG = float('-inf')


def listed():
    return [
        # serving: one user's next item out of 131,072, drawn from the 50 likeliest
        dict(name='sample_next', kind='sample', n=1, V=131_072, dtype='bf16', temperature=0.8, top_k=50, top_p=0.95, min_p=0.0,
             per_row=False, masked=0.0),
        # a large batch of requests, each with settings of its own, some ids banned by -inf
        dict(name='sample_batch', kind='sample', n=4_096, V=32_768, dtype='bf16', temperature=1.0, top_k=40, top_p=0.9,
             min_p=0.05, per_row=True, masked=0.1),
        # rollouts of a training run: the model's own distribution over an odd number of items, logits in fp32
        dict(name='sample_items', kind='sample', n=301, V=50_021, dtype='f32', temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
             per_row=False, masked=0.0),
        # serving: four tokens through a wide layer
        dict(name='linear_token', kind='linear', n=4, K=4_096, N=16_384, dtype='bf16'),
        # scoring: a small odd batch against an odd number of items, a width that is no multiple of 16
        dict(name='linear_items', kind='linear', n=301, K=1_000, N=20_011, dtype='f32'),
        # a prompt's tokens through a wide layer
        dict(name='linear_prompt', kind='linear', n=8_192, K=4_096, N=16_384, dtype='bf16'),
        # a training batch's activation, kept with a scale for each 128 columns
        dict(name='ckpt_train', kind='ckpt', n=16_384, D=4_096, dtype='bf16', group=128, pow2=True),
        # the same of a small odd batch in fp32, one scale a row
        dict(name='ckpt_odd', kind='ckpt', n=5_001, D=1_000, dtype='f32', group=0, pow2=False),
        # the norm's backward of the training batch, with the gradient that arrives on the residual stream
        dict(name='norm_back_train', kind='norm_back', n=16_384, D=4_096, dtype='bf16', group=128, residual=True),
        # the same of the next-item example's default step (64 sessions of 32 items)
        dict(name='norm_back_small', kind='norm_back', n=2_048, D=256, dtype='bf16', group=0, residual=False),
        # the weight gradient of the training batch
        dict(name='wgrad_train', kind='wgrad', n=16_384, N=4_096, K=4_096, dtype='bf16', group=128, transposed=False),
        # the same of a small odd layer with fp32 gradients, into a weight that multiplies from the right
        dict(name='wgrad_odd', kind='wgrad', n=5_001, N=500, K=1_000, dtype='f32', group=0, transposed=True),
    ]


def _logu(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _width(rng, lo, hi):
    """A layer's width: a multiple of 64 for the most part, else any."""
    d = _logu(rng, lo, hi)
    return max(64, d // 64 * 64) if rng.random() < 0.7 else d


def draw(rng):
    kind = rng.choice(('sample', 'sample', 'sample', 'linear', 'linear', 'ckpt', 'norm_back', 'wgrad', 'wgrad'))
    dtype = rng.choice(('bf16', 'bf16', 'f16', 'f32'))
    if kind == 'sample':
        V = _logu(rng, 100, 262_144)
        n = _logu(rng, 1, max(1, min(8_192, (1 << 26) // V)))
        return dict(kind=kind, n=n, V=V, dtype=dtype, temperature=rng.choice((0.5, 0.8, 1.0, 1.3)),
                    top_k=rng.choice((0, 0, 5, 50, 1_000)), top_p=rng.choice((0.5, 0.9, 0.95, 1.0)),
                    min_p=rng.choice((0.0, 0.0, 0.05)), per_row=rng.random() < 0.5, masked=rng.choice((0.0, 0.1, 0.9)))
    if kind == 'linear':
        K, N = _width(rng, 64, 8_192), _width(rng, 64, 65_536)
        n = _logu(rng, 1, max(1, min(8_192, (1 << 38) // (K * N))))
        return dict(kind=kind, n=n, K=K, N=N, dtype=dtype)
    if kind == 'wgrad':
        K, N = _width(rng, 64, 4_096), _width(rng, 64, 4_096)
        n = _logu(rng, 1, max(1, min(16_384, (1 << 36) // (K * N))))
        return dict(kind=kind, n=n, N=N, K=K, dtype=dtype, group=rng.choice((0, 32, 64, 128, 256)),
                    transposed=rng.random() < 0.5)
    D = _width(rng, 64, 8_192)
    n = _logu(rng, 1, max(1, min(200_000, (1 << 25) // D)))
    c = dict(kind=kind, n=n, D=D, dtype=dtype, group=rng.choice((0, 32, 64, 128, 256)))
    if kind == 'ckpt':
        return dict(c, pow2=rng.random() < 0.7)
    return dict(c, residual=rng.random() < 0.7)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device='cuda', dtype=torch.float32)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device='cuda', dtype=torch.float32)


def _groups(x, group):
    """x [n, D] as [n, groups, columns], the last group filled up with zeros."""
    n, D = x.shape
    g = group or D
    m = -(-D // g)
    if m * g != D:
        x = torch.nn.functional.pad(x, (0, m * g - D))
    return x.view(n, m, g)


def _plain_quantize(x, group, pow2):
    """int8 values and fp32 scales of x [n, D]: scale = max|x| / 127 (1 where that is 0), or the smallest power of two that is
    no less; q = x / scale rounded to the nearest, ties to even (the quotient in 64 bits: 32 would round it to a tie first)."""
    grp = _groups(x.float(), group)
    amax = grp.abs().amax(-1, keepdim=True)
    if pow2:
        m, e = torch.frexp(amax)
        scale = torch.ldexp(torch.ones_like(amax), (e - torch.where(m <= 127 / 128, 7, 6)).clamp(min=-126))
        scale = torch.where(amax > 0, scale, 1.0)
    else:
        scale = amax / torch.full_like(amax, 127.0)
        scale = torch.where(scale > 0, scale, 1.0)
    q = (grp.double() / scale.double()).round().clamp(-127, 127).to(torch.int8)
    return q.view(x.shape[0], -1)[:, :x.shape[1]].contiguous(), scale[..., 0].contiguous()


def _plain_widen(q, scale, group, dtype=torch.float32):
    grp = _groups(q.float(), group) * scale[..., None]
    return grp.view(q.shape[0], -1)[:, :q.shape[1]].to(dtype)


def _logits(c, g):
    """Logits of about the spread that a trained model gives, the row's own offset added; some ids banned, one row of
    a masked batch left without any."""
    n, V = c['n'], c['V']
    x = (_randn(g, n, V).mul_(2.5).add_(_randn(g, n, 1))).to(TYPES[c['dtype']])
    if c['masked']:
        x.masked_fill_(_rand(g, n, V) < c['masked'], NEG)
        if n > 8:
            x[n // 2] = NEG
    return x


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device='cuda').manual_seed(int(seed))
    kind, t, n = c['kind'], TYPES[c['dtype']], c['n']
    if kind == 'sample':
        c['logits'], c['u'] = _logits(c, g), _rand(g, n)
        c['set'] = {k: c[k] for k in ('temperature', 'top_k', 'top_p', 'min_p')}
        if c['per_row']:                    # requests with settings around the case's, some greedy, some unrestricted
            pick = _rand(g, n)
            temp = c['temperature'] * (0.5 + _rand(g, n))
            k = (c['top_k'] * (0.5 + _rand(g, n))).to(torch.int32)
            c['set'] = dict(temperature=torch.where(pick < 0.1, 0.0, temp), top_k=torch.where(pick > 0.8, 0, k),
                            top_p=torch.where(pick > 0.9, 1.0, c['top_p'] * (0.5 + 0.5 * _rand(g, n))),
                            min_p=c['min_p'] * _rand(g, n))
    elif kind == 'linear':
        c['xq'], c['xs'] = _plain_quantize(_randn(g, n, c['K']), 0, False)
        c['wq'], c['ws'] = _plain_quantize(_randn(g, c['N'], c['K']).mul_(c['K'] ** -0.5), 0, False)
    elif kind == 'ckpt':
        c['x'] = _randn(g, n, c['D']).mul_(1.0 + 3.0 * _rand(g, 1, c['D'])).to(t)
    elif kind == 'norm_back':
        h = _randn(g, n, c['D']).mul_(2.0)
        c['hq'], c['hs'] = _plain_quantize(h, c['group'], True)
        c['rstd'] = (h.double().square().mean(-1) + EPS).rsqrt().float()
        c['w'] = (1.0 + 0.1 * _randn(g, c['D'])).to(t)
        c['dy'] = _randn(g, n, c['D']).mul_(1e-3).to(t)
        c['dh'] = _randn(g, n, c['D']).mul_(1e-3).to(t) if c['residual'] else None
    else:
        c['xq'], c['xs'] = _plain_quantize(_randn(g, n, c['K']), c['group'], True)
        c['dy'] = _randn(g, n, c['N']).mul_(1e-3).to(t)
    return c


def _column(v, x):
    """A setting as fp64 [n, 1] beside x [n, V]."""
    v = v if torch.is_tensor(v) else torch.full((x.shape[0],), v, dtype=torch.float64, device=x.device)
    return v.double()[:, None]


def _plain_sample(c, rows):
    x, u = c['logits'][rows].double(), c['u'][rows].double()[:, None]
    n, V = x.shape
    s = {k: _column(v[rows] if torch.is_tensor(v) else v, x) for k, v in c['set'].items()}
    top = x.amax(-1, keepdim=True)
    empty = top == NEG
    d = x - torch.where(empty, 0.0, top)
    greedy = s['temperature'] == 0
    e = torch.where(greedy, (d == 0).double(), (d / torch.where(greedy, 1.0, s['temperature'])).exp())
    order = x.sort(dim=-1, descending=True, stable=True).indices   # larger first, ties by the lower id
    se = e.gather(1, order)
    rank = torch.arange(V, device=x.device)
    k = torch.where(greedy, 1.0, s['top_k'])
    se = torch.where((k <= 0) | (rank < k), se, 0.0)
    total = se.sum(-1, keepdim=True)
    before = se.cumsum(-1) - se
    keep = (se > 0) & ((rank == 0) | (s['top_p'] >= 1) | (before < s['top_p'] * total)) & (se >= s['min_p'])
    w = torch.zeros_like(e).scatter_(1, order, torch.where(keep, se, 0.0))
    cum = w.cumsum(-1)
    t = u * cum[:, -1:]
    token = (cum <= t).sum(-1).clamp(max=V - 1)
    own_w = w.gather(1, token[:, None])[:, 0]
    logprob = (own_w / cum[:, -1]).log()
    none = empty[:, 0]
    return dict(token=torch.where(none, -1, token), logprob=torch.where(none, NEG, logprob).float())


def _plain_norm_back(c):
    h, dy, rstd = _plain_widen(c['hq'], c['hs'], c['group']), c['dy'].float(), c['rstd'][:, None]
    xh, u = h * rstd, dy * c['w'].float()
    dx = rstd * (u - xh * (u * xh).mean(-1, keepdim=True))
    if c['dh'] is not None:
        dx = dx + c['dh'].float()
    return dict(dx=dx.to(c['dy'].dtype), dw=(dy * xh).sum(0))


def _join(parts):
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _slices(n, step):
    return [slice(a, min(a + step, n)) for a in range(0, n, step)]


def _own(c):
    from elara_amd import int8, norms, sampling
    kind = c['kind']
    if kind == 'sample':
        r = sampling.sample_tokens(c['logits'], c['u'], **c['set'])
        return dict(token=r.token, logprob=r.logprob)
    if kind == 'linear':
        return dict(y=int8.linear(int8.Int8Rows(c['xq'], c['xs'], 0), int8.Int8Rows(c['wq'], c['ws'], 0),
                                  dtype=TYPES[c['dtype']]))
    if kind == 'ckpt':
        kept = int8.quantize(c['x'], group=c['group'], pow2=c['pow2'])
        return dict(scale=kept.scale, x=int8.dequantize(kept, dtype=c['x'].dtype))
    if kind == 'norm_back':
        dx, dw = norms.rms_norm_backward_int8(c['dy'], int8.Int8Rows(c['hq'], c['hs'], c['group']), c['w'], c['rstd'],
                                              dh=c['dh'])
        return dict(dx=dx, dw=dw)
    return dict(dw=int8.weight_grad(c['dy'], int8.Int8Rows(c['xq'], c['xs'], c['group']), transposed=c['transposed']))


def run(state):
    c, kind = state, state['kind']
    if own:
        return _own(c)
    if kind == 'sample':
        return _join([_plain_sample(c, s) for s in _slices(c['n'], max(1, (1 << 26) // c['V']))])
    if kind == 'linear':
        y = (c['xq'].float() @ c['wq'].float().t()) * c['xs'] * c['ws'].t()
        return dict(y=y.to(TYPES[c['dtype']]))
    if kind == 'ckpt':
        q, scale = _plain_quantize(c['x'], c['group'], c['pow2'])
        return dict(scale=scale, x=_plain_widen(q, scale, c['group'], c['x'].dtype))
    if kind == 'norm_back':
        return _plain_norm_back(c)
    dw = c['dy'].float().t() @ _plain_widen(c['xq'], c['xs'], c['group'])
    return dict(dw=dw.t().contiguous() if c['transposed'] else dw)


def _scales(c, width):
    return -(-c[width] // c['group']) if c['group'] else 1


def work(case):
    c, kind, n = case, case['kind'], case['n']
    es = ESIZE[c['dtype']]
    if kind == 'sample':
        return dict(bytes=n * c['V'] * es + n * (4 + 12 + (16 if c['per_row'] else 0)), flops=8 * n * c['V'])
    if kind == 'linear':
        return dict(bytes=(n + c['N']) * (c['K'] + 4) + n * c['N'] * es, flops=2 * n * c['N'] * c['K'])
    if kind == 'ckpt':
        nd = n * c['D']
        return dict(bytes=2 * nd * (es + 1) + 8 * n * _scales(c, 'D'), flops=4 * nd)
    if kind == 'norm_back':
        nd = n * c['D']
        return dict(bytes=nd * (1 + es * (3 if c['residual'] else 2)) + 4 * n * (1 + _scales(c, 'D')) + c['D'] * (es + 4),
                    flops=12 * nd)
    return dict(bytes=n * (c['N'] * es + c['K'] + 4 * _scales(c, 'K')) + 4 * c['N'] * c['K'], flops=2 * n * c['N'] * c['K'])


def exact(case, seed):
    c, kind, n = prepare(case, seed), case['kind'], case['n']
    if kind == 'sample':
        return _join([_exact_sample(c, s) for s in _slices(n, max(1, (1 << 25) // c['V']))])
    if kind == 'linear':
        w = c['wq'].double() * c['ws'].double()
        return dict(y=torch.cat([(c['xq'][s].double() * c['xs'][s].double()) @ w.t() for s in _slices(n, 2_048)]))
    if kind == 'ckpt':
        x, out, scales = c['x'].double(), [], []
        for cols in x.split(c['group'] or c['D'], dim=1):
            top = cols.abs().max(1, keepdim=True).values
            s = top / 127
            s = torch.exp2(torch.ceil(torch.log2(s))) if c['pow2'] else s.float().double()    # a scale is held in fp32
            s = torch.where(s > 0, s, 1.0)
            out.append(torch.round(cols / s) * s)
            scales.append(s)
        return dict(scale=torch.cat(scales, 1), x=torch.cat(out, 1))
    each = c['group'] or (c['K'] if kind == 'wgrad' else c['D'])
    q, s = (c['xq'], c['xs']) if kind == 'wgrad' else (c['hq'], c['hs'])
    x = q.double() * s.double().repeat_interleave(each, 1)[:, :q.shape[1]]
    if kind == 'wgrad':
        dw = torch.einsum('ik,in->kn', x, c['dy'].double())
        return dict(dw=dw if c['transposed'] else dw.t())
    rstd, dy, w = c['rstd'].double()[:, None], c['dy'].double(), c['w'].double()
    dot = (dy * w * x).sum(-1, keepdim=True)
    dx = dy * w * rstd - x * (rstd ** 3 * dot / c['D'])
    dw = (dy * x * rstd).sum(0)
    return dict(dx=dx if c['dh'] is None else dx + c['dh'].double(), dw=dw)


def _exact_sample(c, rows):
    x, u = c['logits'][rows].double(), c['u'][rows].double()
    n, V = x.shape
    s = {k: (v[rows].double() if torch.is_tensor(v) else torch.full((n,), float(v), dtype=torch.float64, device=x.device))
         for k, v in c['set'].items()}
    some = x.max(1).values > NEG
    x[~some] = 0.0
    hot = s['temperature'] > 0
    xs, ids = torch.sort(x, dim=1, descending=True, stable=True)
    logp = torch.log_softmax(xs / torch.where(hot, s['temperature'], 1.0)[:, None], 1)
    at = torch.arange(V, device=x.device)[None]
    in_k = at < torch.where(hot, torch.where(s['top_k'] > 0, s['top_k'], V), 1)[:, None]
    p = logp.exp() * in_k
    p = p / p.sum(1, keepdim=True)
    ahead = torch.cat([torch.zeros(n, 1, dtype=torch.float64, device=x.device), p.cumsum(1)[:, :-1]], 1)
    limit = torch.where(s['top_p'] < 1, s['top_p'], float('inf'))[:, None]
    near = logp - logp[:, :1] >= torch.log(s['min_p'])[:, None]
    p = p * (((ahead < limit) | (at == 0)) & near)
    by_id = torch.empty_like(p).scatter_(1, ids, p)
    cdf = by_id.cumsum(1)
    token = torch.searchsorted(cdf, (u * cdf[:, -1])[:, None], right=True)[:, 0].clamp(max=V - 1)
    logprob = by_id[torch.arange(n, device=x.device), token].log() - cdf[:, -1].log()
    return dict(token=torch.where(some, token, -1), logprob=torch.where(some, logprob, NEG))
