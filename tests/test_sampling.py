"""Drawing tokens (elara_amd.sampling) against the definition in 64 bits.  No counterpart in the reference.

The drawn ids have to be equal.  The kernel's weights are e rounded to a multiple of 2^-s with V 2^s < 2^63, s <= 51, so a sum of V of them
is within V 2^-s-1 of its own beside a whole sum of at least 1: 2^-26 for the largest V here (2^18, s = 43).  (fp64 exponentials are within
2^-45.)  The tests place u no nearer than 2^-25 of the whole to a border.  A log probability is within 2^-24 of itself (its rounding to
fp32) and 2^-25.
"""
import ctypes
import math

import pytest
import torch

from elara_amd import _lib

TYPES = [torch.float32, torch.float16, torch.bfloat16]
NEG = float('-inf')


def _sp():
    from elara_amd import sampling
    return sampling


def _row(x, temperature, top_k, top_p, min_p):
    """(kept ids by rising id, their weights) of one row in 64 bits, on the CPU."""
    x = x.double()
    V = x.numel()
    m = float(x.max())
    order = torch.sort(x, descending=True, stable=True).indices
    if temperature == 0:
        return order[:1], torch.ones(1, dtype=torch.float64)
    e = torch.exp((x - m) / temperature)
    kept = order[:top_k] if 0 < top_k < V else order
    w = e[kept]
    before = torch.cat([torch.zeros(1, dtype=torch.float64), w.cumsum(0)[:-1]])
    if top_p < 1:
        on = before < top_p * w.sum()
        on[0] = True
        kept = kept[on]
    if min_p > 0:
        kept = kept[(x[kept] - m >= math.log(min_p) * temperature)]
    kept = kept.sort().values
    return kept, e[kept]


def _value(v, i):
    return v[i].item() if torch.is_tensor(v) else v


def check(dev, x, u=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, view=lambda t: t, seed=0):
    """Each row drawn with u (or several drawn at random), kept away from borders."""
    sp = _sp()
    n = x.shape[0]
    if u is None:
        u = torch.rand(n, generator=torch.Generator().manual_seed(seed))
    tokens, logps, clear = [], [], []
    for i in range(n):
        if bool((x[i] == NEG).all()):
            tokens.append(-1), logps.append(NEG), clear.append(True)
            continue
        ids, w = _row(x[i], *(_value(v, i) for v in (temperature, top_k, top_p, min_p)))
        cum = w.cumsum(0)
        t = float(u[i].double()) * float(cum[-1])
        at = min(int((cum <= t).sum()), len(ids) - 1)
        clear.append(float((cum - t).abs().min()) > 2.0 ** -25 * float(cum[-1]) or len(ids) == 1)
        tokens.append(int(ids[at])), logps.append(float((w[at] / cum[-1]).log()))
    up = lambda v: v.to(dev) if torch.is_tensor(v) else v  # noqa: E731
    r = sp.sample_tokens(view(x.to(dev)), u.to(dev), temperature=up(temperature), top_k=up(top_k), top_p=up(top_p), min_p=up(min_p))
    assert r.token.dtype == torch.int64 and r.logprob.dtype == torch.float32 and r.token.shape == r.logprob.shape == (n,)
    clear = torch.tensor(clear)
    assert float(clear.double().mean()) > 0.9
    tok, ref = torch.tensor(tokens), torch.tensor(logps, dtype=torch.float64)
    assert torch.equal(r.token.cpu()[clear], tok[clear]), (r.token.cpu()[clear] != tok[clear]).nonzero()[:5]
    got = r.logprob.cpu().double()
    same = got == ref
    assert bool((same | ((got - ref).abs() <= 2.0 ** -24 * ref.abs() + 2.0 ** -25))[clear].all())
    return r


def _logits(seed, n, V, dtype, spread=2.5, masked=0.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, V, generator=g) * spread + torch.randn(n, 1, generator=g)).to(dtype)
    if masked:
        x[torch.rand(n, V, generator=g) < masked] = NEG
    return x


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=5), dict(top_k=50), dict(top_p=0.9), dict(top_p=0.3),
            dict(min_p=0.1), dict(top_k=40, top_p=0.9, min_p=0.05, temperature=0.8), dict(temperature=0.0),
            dict(temperature=1.5, top_p=0.99), dict(top_k=1000, top_p=0.5), dict(top_p=0.0), dict(min_p=1.0)]
WIDTHS = [1, 2, 7, 63, 64, 65, 100, 255, 500, 1000, 1024, 2049, 4096, 5000, 16_384, 20_001, 50_021, 131_072, 262_147]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('V', WIDTHS)
def test_settings(dev, V, dtype):
    n = 2 if V > 60_000 else 3 if V > 5000 else 9
    for i, s in enumerate(SETTINGS):
        check(dev, _logits(V + i, n, V, dtype, masked=(0, 0.3)[i % 2] if V > 2 else 0), seed=i, **s)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('V', [3, 40, 300, 2500])
def test_every_token_is_reached(dev, V, dtype):
    """u in the middle of each kept token's part of the mass draws that token, and each just inside both its ends."""
    sp = _sp()
    x = _logits(V, 1, V, dtype, spread=1.0)
    for s in (dict(), dict(top_k=17), dict(top_p=0.8, temperature=2.0), dict(min_p=0.3), dict(top_k=30, top_p=0.6, min_p=0.05)):
        full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, **{}) | s
        ids, w = _row(x[0], **full)
        cum = w.cumsum(0) / w.sum()
        lo = torch.cat([torch.zeros(1, dtype=torch.float64), cum[:-1]])
        for f in (0.1, 0.5, 0.9):
            u = (lo + f * (cum - lo)).float()
            r = sp.sample_tokens(x.expand(len(ids), V).contiguous().to(dev), u.to(dev), **s)
            assert torch.equal(r.token.cpu(), ids)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_ties_go_to_the_lowest_ids(dev, dtype):
    for V in (70, 1000, 5000, 40_000):
        x = torch.zeros(6, V, dtype=dtype)
        x[:, V // 2:] = -0.0                                  # equal to +0
        x[1, ::7] = 1.0
        x[2, V - 3:] = 2.0
        x[3] = torch.finfo(dtype).min                         # a finite mask everywhere: uniform
        x[4, 5:] = NEG
        x[5, : V - 1] = NEG
        for s in (dict(top_k=9), dict(top_k=V - 1), dict(top_p=0.25), dict(top_p=0.7, top_k=20), dict(), dict(temperature=0.0),
                  dict(min_p=0.5)):
            for seed in range(3):
                check(dev, x, seed=seed, **s)


@pytest.mark.gpu
def test_many_rows_with_ties_at_the_threshold(dev):
    """Searches that follow one another in a block (for the ties of a threshold, then for the token), over thousands of rows."""
    sp = _sp()
    n, V = 6000, 20_000
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randint(0, 12, (n, V), generator=g, device=dev).bfloat16()
    u = torch.rand(n, generator=g, device=dev)
    first = (x == x.amax(-1, keepdim=True)).int().argmax(-1)
    assert torch.equal(sp.sample_tokens(x, u, temperature=0.0).token, first)
    assert torch.equal(sp.sample_tokens(x, u, top_k=1).token, first)
    for k in (40, 300):                                       # the first k ids with the largest value, alike in weight
        at = torch.nonzero(x == 11)[:, 1].split((x == 11).sum(-1).tolist())
        want = torch.stack([a[min(int(k * float(v)), k - 1)] for a, v in zip(at, u.double().tolist())])
        assert torch.equal(sp.sample_tokens(x, u, top_k=k).token, want)


def _nucleus(x, u, top_p, min_p):
    """(ids, log probabilities, whether u and top_p lie clear of every border) of all rows by top_p and min_p, in 64 bits on x's
    device."""
    x = x.double()
    m = x.amax(-1, keepdim=True)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    e = (x - m).exp()
    w = e.gather(1, order)
    total, before = w.sum(-1, keepdim=True), w.cumsum(-1) - w
    on = before < top_p * total
    on[:, 0] = True
    clear = (before - top_p * total).abs().amin(-1) > 2.0 ** -25 * total[:, 0]
    if min_p > 0:
        on &= x.gather(1, order) - m >= math.log(min_p)
    kept = torch.zeros_like(e).scatter_(1, order, torch.where(on, w, 0.0))
    cum = kept.cumsum(-1)
    t = u.double()[:, None] * cum[:, -1:]
    clear &= (cum - t).abs().amin(-1) > 2.0 ** -25 * cum[:, -1]
    token = (cum <= t).sum(-1).clamp(max=x.shape[1] - 1)
    return token, (kept.gather(1, token[:, None])[:, 0] / cum[:, -1]).log(), clear


@pytest.mark.gpu
@pytest.mark.parametrize('n,V,top_k,dtype', [(3000, 5000, 1000, torch.bfloat16), (3000, 3000, 600, torch.float32),
                                             (2000, 20_000, 4000, torch.bfloat16), (300, 20_000, 4000, torch.float16),
                                             (600, 40_000, 9000, torch.bfloat16), (200, 50_000, 9000, torch.bfloat16),
                                             (40, 140_000, 30_000, torch.bfloat16), (300, 150_000, 40_000, torch.float32)])
def test_fewer_finite_ids_than_top_k(dev, n, V, top_k, dtype):
    """Most ids banned, so that top_k (more than a bound's candidates) reaches past the last finite id and top_p has to look for
    its place after a search that found none: in blocks of 4, 8 and 16 waves."""
    sp = _sp()
    g = torch.Generator(device=dev).manual_seed(V + n)
    x = (torch.randn(n, V, generator=g, device=dev) * 2).to(dtype)
    x.masked_fill_(torch.rand(n, V, generator=g, device=dev) < 0.9, NEG)
    assert int((x > NEG).sum(-1).max()) < top_k < V
    u = torch.rand(n, generator=g, device=dev)
    for top_p, min_p in ((0.9, 0.0), (0.5, 0.0), (0.95, 1e-3)):
        token, logp, clear = _nucleus(x, u, top_p, min_p)
        assert float(clear.double().mean()) > 0.9
        for k in (top_k, torch.full((n,), top_k, dtype=torch.int32, device=dev)):
            for _ in range(3):
                r = sp.sample_tokens(x, u, top_k=k, top_p=top_p, min_p=min_p)
                assert torch.equal(r.token[clear], token[clear])
                off = (r.logprob.double() - logp).abs()
                assert bool((off <= 2.0 ** -24 * logp.abs() + 2.0 ** -25)[clear].all())


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('V', [50, 777, 4096, 33_000])
def test_settings_by_row(dev, V, dtype):
    n = 40 if V < 5000 else 12
    g = torch.Generator().manual_seed(V)
    x = _logits(V, n, V, dtype, masked=0.1)
    x[3] = NEG
    temp = torch.rand(n, generator=g) * 1.5
    temp[1] = 0
    k = torch.randint(0, V + 20, (n,), generator=g)
    p, mp = torch.rand(n, generator=g), torch.rand(n, generator=g) * 0.2
    p[5] = 1.0
    for kt in (torch.int32, torch.int64):
        check(dev, x, temperature=temp, top_k=k.to(kt), top_p=p, min_p=mp)
    check(dev, x, top_k=k, seed=1)
    check(dev, x, temperature=temp, top_p=0.8, seed=2)
    check(dev, x, top_p=p, seed=3)


@pytest.mark.gpu
def test_flat_and_steep_rows(dev):
    """Where the mass lies with many ids alike, with one, with a few far from the rest, or beyond what 64 bits resolve."""
    for V in (300, 9000, 60_000):
        g = torch.Generator().manual_seed(V)
        flat = torch.randn(4, V, generator=g) * 1e-3
        steep = torch.randn(4, V, generator=g) * 200
        few = torch.full((4, V), -30.0)
        few[:, ::V // 5] = torch.randn(4, len(range(0, V, V // 5)), generator=g)
        for x in (flat, steep, few):
            for s in (dict(), dict(top_p=0.9), dict(top_k=100, top_p=0.95), dict(temperature=0.05), dict(temperature=100.0, top_p=0.5)):
                check(dev, x, **s)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_smallest_temperatures(dev, dtype):
    """Temperatures whose reciprocal fp64 does not hold, or just holds: the ids of the largest logit share the mass, nothing else
    has any.  What the outputs' memory held before is no answer."""
    sp = _sp()
    for V in (1, 5, 900, 5000, 40_000):
        x = _logits(V, 6, V, dtype)
        if V > 4:
            x[2:, V // 3] = x[2:, V - 2] = 100.0              # two of the largest
            x[4, :] = -1.0                                    # all of them
            x[5] = 0.0
            x[5, 3] = torch.finfo(dtype).tiny                 # a neighbour
        u = torch.tensor([0.1, 0.9, 0.25, 0.75, 0.6, 0.4])
        ids = [torch.nonzero(r == r.max())[:, 0] for r in x]
        for s in (dict(), dict(top_k=5), dict(top_k=700), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=400, top_p=1.0, min_p=0.5)):
            for T in (5e-324, 1e-310, 5e-309, 8e-309, 1e-300):
                old = torch.full((6,), 777, device=dev), torch.full((6,), 777.0, device=dev)      # the memory of the outputs to come
                del old
                r = sp.sample_tokens(x.to(dev), u.to(dev), temperature=T, **s)
                for i in range(6):
                    kept = ids[i][:s['top_k']] if 0 < s.get('top_k', 0) < V else ids[i]
                    if 'top_p' in s and s['top_p'] < 1:       # the first whose mass before is less than the part
                        kept = kept[torch.arange(len(kept)).double() < s['top_p'] * len(kept)]
                    assert int(r.token[i]) == int(kept[int(float(u[i].double()) * len(kept))]), (V, s, T, i)
                    assert abs(float(r.logprob[i]) + math.log(len(kept))) <= 2.0 ** -24 * math.log(len(kept)) + 2.0 ** -25


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_rows_without_an_answer(dev, dtype):
    sp = _sp()
    for V in (5, 900, 50_000):
        x = _logits(1, 6, V, dtype)
        x[0] = NEG
        x[1, 2] = float('nan')
        x[2, V - 1] = float('inf')
        u = torch.full((6,), 0.5)
        u[3] = float('nan')
        temp = torch.ones(6)
        temp[4] = -1.0
        for s in (dict(), dict(top_k=3, top_p=0.5)):
            r = sp.sample_tokens(x.to(dev), u.to(dev), temperature=temp.to(dev), **s)
            assert r.token[:5].tolist() == [-1] * 5 and int(r.token[5]) >= 0
            assert float(r.logprob[0]) == NEG and torch.isnan(r.logprob[1:5]).all()
        r = sp.sample_tokens(x.to(dev), torch.full((6,), 0.5, device=dev), temperature=torch.full((6,), float('nan'), device=dev))
        assert r.token.tolist() == [-1] * 6


@pytest.mark.gpu
def test_settings_out_of_range_by_row(dev):
    sp = _sp()
    x = _logits(3, 8, 500, torch.float32).to(dev)
    u = torch.rand(8, device=dev)
    f = lambda v, t=torch.float32: torch.full((8,), v, dtype=t, device=dev)  # noqa: E731
    base = sp.sample_tokens(x, u)
    for s in (dict(top_k=f(-4, torch.int32)), dict(top_k=f(10_000, torch.int64)), dict(top_p=f(1.7)), dict(top_p=f(float('nan'))),
              dict(min_p=f(-1.0)), dict(min_p=f(float('nan')))):
        r = sp.sample_tokens(x, u, **s)
        assert torch.equal(r.token, base.token) and torch.equal(r.logprob, base.logprob), s
    top = x.argmax(-1)
    assert torch.equal(sp.sample_tokens(x, u, top_p=f(-0.5)).token, top)
    assert torch.equal(sp.sample_tokens(x, u, min_p=f(3.0)).token, top)
    last = sp.sample_tokens(x, f(1.0), top_k=5)
    assert torch.equal(last.token, x.topk(5).indices.max(-1).values)
    first = sp.sample_tokens(x, f(-0.5), top_k=5)
    assert torch.equal(first.token, x.topk(5).indices.min(-1).values)


@pytest.mark.gpu
def test_strides_shapes_and_empty(dev):
    sp = _sp()
    x = _logits(5, 12, 1001, torch.bfloat16)
    for view in (lambda t: torch.cat([t, t], 1)[:, :1001], lambda t: torch.cat([t[:, :1], t], 1)[:, 1:],
                 lambda t: t.t().contiguous().t()):
        check(dev, x, view=view, top_p=0.9)
    a, u = x.to(dev), torch.rand(12, device=dev)
    base = sp.sample_tokens(a, u, top_k=20)
    r = sp.sample_tokens(a.view(3, 4, 1001), u.view(3, 4), top_k=20)
    assert r.token.shape == (3, 4) and torch.equal(r.token.view(-1), base.token)
    r = sp.sample_tokens(a.view(3, 4, 1001), u.view(3, 4), top_k=torch.full((3, 4), 20, device=dev))
    assert torch.equal(r.token.view(-1), base.token)
    one = sp.sample_tokens(a[2], u[2], top_k=20)
    assert one.token.shape == () and int(one.token) == int(base.token[2])
    r = sp.sample_tokens(a[:1].expand(12, 1001), u)
    assert torch.equal(r.token, sp.sample_tokens(a[:1].expand(12, 1001).contiguous(), u).token)
    assert sp.sample_tokens(a[:0], u[:0]).token.shape == (0,)
    uu = torch.rand(24, device=dev)
    assert torch.equal(sp.sample_tokens(a, uu[::2]).token, sp.sample_tokens(a, uu[::2].contiguous()).token)


@pytest.mark.gpu
def test_numbers_of_other_types(dev):
    import numpy as np
    sp = _sp()
    x, u = _logits(8, 5, 700, torch.float32).to(dev), torch.rand(5, device=dev)
    a = sp.sample_tokens(x, u, temperature=0.5, top_k=9, top_p=0.75, min_p=0.25)
    b = sp.sample_tokens(x, u, temperature=np.float32(0.5), top_k=np.int32(9), top_p=np.float64(0.75), min_p=np.float16(0.25))
    assert torch.equal(a.token, b.token) and torch.equal(a.logprob, b.logprob)


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """Calls in flight together share nothing."""
    sp = _sp()
    xs = [_logits(20 + i, 300, 9000, torch.bfloat16).to(dev) for i in range(2)]
    u = torch.rand(300, device=dev)
    alone = [sp.sample_tokens(x, u, top_k=1000, top_p=0.9).token for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(sp.sample_tokens(xs[i], u, top_k=1000, top_p=0.9).token)
    torch.cuda.synchronize()
    assert all(torch.equal(t, alone[i]) for i in range(2) for t in got[i])


@pytest.mark.gpu
def test_streams_graphs_and_repeats(dev):
    sp = _sp()
    x = [_logits(7 + i, 20, 6000, torch.float16).to(dev) for i in range(2)]
    u = torch.rand(20, device=dev)
    call = lambda t: sp.sample_tokens(t, u, temperature=0.9, top_k=200, top_p=0.9, min_p=0.01)  # noqa: E731
    eager = [call(t) for t in x]
    assert all(torch.equal(call(x[0]).token, eager[0].token) for _ in range(4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(x[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.token, eager[0].token) and torch.equal(got.logprob, eager[0].logprob)
    ins, graphs, outs = [t.clone() for t in x], [], []
    for t in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(t))
        graphs.append(g)
    for turn in range(3):
        for i, g in enumerate(graphs):
            ins[i].copy_(x[(i + turn) % 2])
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i].token, eager[(i + turn) % 2].token)
            assert torch.equal(outs[i].logprob, eager[(i + turn) % 2].logprob)
            call(x[0])


@pytest.mark.gpu
def test_shares_of_many_draws(dev):
    """Equally spaced numbers draw each id in proportion to its probability, to within one draw at each end."""
    sp = _sp()
    n, V = 20_000, 40
    x = _logits(9, 1, V, torch.float32, spread=1.0)
    u = (torch.arange(n) + 0.5) / n
    r = sp.sample_tokens(x.expand(n, V).to(dev), u.to(dev))
    share = torch.bincount(r.token.cpu(), minlength=V).double()
    p = torch.softmax(x[0].double(), 0)
    assert float((share - p * n).abs().max()) <= 1.0 + n * 2.0 ** -23


@pytest.mark.gpu
def test_many_rows(dev):
    sp = _sp()
    x = torch.randn(2_200_000, 5, device=dev)
    u = torch.rand(2_200_000, device=dev)
    r = sp.sample_tokens(x, u, top_k=3)
    pick = torch.cat([torch.arange(0, 2_200_000, 99_991), torch.tensor([2_097_151, 2_097_152, 2_199_999])])
    one = sp.sample_tokens(x[pick.to(dev)], u[pick.to(dev)], top_k=3)
    assert torch.equal(one.token, r.token[pick.to(dev)]) and bool((r.token >= 0).all())
    check(dev, x[pick.to(dev)].cpu(), u=u[pick.to(dev)].cpu(), top_k=3)


def test_refusals_of_the_c_entry_point():
    L = _lib.lib()
    p = ctypes.c_void_p(256)

    def call(x=p, type=0, n=1, V=8, ld=8, u=p, t=1.0, k=0, tp=1.0, mp=0.0, token=p):
        return L.elr_sample_tokens(x, type, n, V, ld, u, t, None, k, None, 0, tp, None, mp, None, token, p, None)
    assert call(n=-1) == -1 and call(V=0) == -1 and call(ld=-1) == -1 and call(type=4) == -1
    assert call(V=(1 << 30) + 1) == -2
    for t in (-0.5, float('nan'), float('inf')):
        assert call(t=t) == -1
    assert call(k=-1) == -1 and call(tp=1.5) == -1 and call(tp=float('nan')) == -1 and call(mp=-0.1) == -1 and call(mp=2.0) == -1
    assert call(x=None) == -1 and call(u=None) == -1 and call(token=None) == -1 and call(x=ctypes.c_void_p(257)) == -1
    assert call(n=0, x=None, u=None, token=None) == 0


def test_refusals_of_cpu_tensors():
    with pytest.raises(RuntimeError, match='cuda'):
        _sp().sample_tokens(torch.zeros(2, 5), torch.zeros(2))


@pytest.mark.gpu
def test_refusals(dev):
    sp = _sp()
    x, u = torch.randn(3, 50, device=dev), torch.rand(3, device=dev)
    bad = [lambda: sp.sample_tokens(x.double(), u), lambda: sp.sample_tokens(x, u.double()), lambda: sp.sample_tokens(x, u[:2]),
           lambda: sp.sample_tokens(x, u.cpu()), lambda: sp.sample_tokens(x, u, temperature=-1.0),
           lambda: sp.sample_tokens(x, u, temperature=float('nan')), lambda: sp.sample_tokens(x, u, temperature=float('inf')),
           lambda: sp.sample_tokens(x, u, top_k=-1), lambda: sp.sample_tokens(x, u, top_p=1.1),
           lambda: sp.sample_tokens(x, u, top_p=-0.1), lambda: sp.sample_tokens(x, u, min_p=1.5),
           lambda: sp.sample_tokens(x, u, top_k=5.5), lambda: sp.sample_tokens(x, u, temperature='hot'),
           lambda: sp.sample_tokens(x, u, temperature=u.double()), lambda: sp.sample_tokens(x, u, top_k=u),
           lambda: sp.sample_tokens(x, u, top_p=u[:1]), lambda: sp.sample_tokens(x, u, min_p=u.cpu())]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f'call {i} was taken')
