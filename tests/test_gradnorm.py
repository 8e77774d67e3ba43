"""The global gradient norm and clipping (elara_amd.gradnorm) against the definition in 64 bits.  No counterpart in the
reference.

Bounds, with u = 2^-24: the sums are fp64, so the norm is within one rounding (2 u with the square root's); the scale adds
two roundings and the product one, so an output is within 8 u before its own rounding.
"""
import ctypes
import math
import random
import threading

import pytest
import torch

from elara_amd import _lib

U = 2.0 ** -24
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-37}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = math.inf


def _gn():
    from elara_amd import gradnorm
    return gradnorm


def _randn(dev, seed, *shape, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dev)


def ref_norm(grads, p):
    flat = torch.cat([g.double().reshape(-1) for g in grads]) if grads else torch.zeros(0)
    a = flat.abs()
    if p == INF:
        return float(a.max()) if a.numel() else 0.0
    return float((a ** p).sum() ** (1 / p))


def check(grads, p=2.0, max_norm=None, out=None, eps=1e-6):
    gn = _gn()
    N = ref_norm(grads, p)
    n = gn.grad_norm(grads, p)
    assert n.dtype == torch.float32 and n.dim() == 0 and abs(float(n) - N) <= 2 * U * N
    if max_norm is None:
        return
    before = [g.clone() for g in grads]
    c = min(1.0, max_norm / (N + eps))
    m = gn.clip_grad_norm(grads, max_norm, p, eps, out=out)
    assert float(m) == float(n)
    for b, g, o in zip(before, grads, out if out is not None else grads):
        want = b.double() * c
        d = (o.double() - want).abs()
        bound = (8 * U + HALF_ULP[o.dtype] * (1 + 8 * U)) * want.abs() + TINY[o.dtype]
        assert bool((d <= bound).all())
        if out is not None and o is not g:
            assert torch.equal(g, b)


SHAPES = [(1,), (3,), (8,), (255,), (4096,), (4097,), (33, 65), (8191,), (2, 3, 5), (0,), (0, 7), (100_003,), (300, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize('p', [1.0, 2.0, INF])
@pytest.mark.parametrize('dtype', TYPES + ['mixed'])
@pytest.mark.parametrize('out', [None, 'same', 'f32'])
def test_clip(dev, dtype, p, out):
    grads = [_randn(dev, i, *s, scale=0.1).to(TYPES[i % 3] if dtype == 'mixed' else dtype) for i, s in enumerate(SHAPES)]
    N = ref_norm(grads, p)
    for max_norm in (0.3 * N, 2 * N, 0.0):
        outs = None if out is None else [torch.full_like(g, 7.0, dtype=None if out == 'same' else torch.float32) for g in grads]
        check([g.clone() for g in grads] if out is None else grads, p, max_norm, outs)


@pytest.mark.gpu
@pytest.mark.parametrize('count', [1, 135, 136, 137, 143, 144, 145, 289, 700])
def test_many_tensors(dev, count):
    """More tensors than one launch takes, in one unaligned buffer; nothing between them is touched."""
    sizes = [1 + (i * 37) % 501 for i in range(count)]
    buf = _randn(dev, 1, sum(sizes) + count + 1, scale=0.1).to(torch.bfloat16)
    before = buf.clone()
    at, grads, gaps = 1, [], [0]
    for s in sizes:
        grads.append(buf[at:at + s])
        gaps.append(at + s)
        at += s + 1
    check(grads, 2.0, 0.5)
    assert torch.equal(buf[gaps], before[gaps])


@pytest.mark.gpu
@pytest.mark.parametrize('n', [1, 4095, 4096, 8192, 8193, 5_000_000, 33_554_433])
def test_sizes(dev, n):
    g = _randn(dev, n % 97, min(n, 1 << 20)).repeat(-(-n // min(n, 1 << 20)))[:n].contiguous()
    check([g], 2.0, 1.0)
    check([g.to(torch.bfloat16)], 2.0, 1.0, [torch.empty(n, device=dev)])


@pytest.mark.gpu
def test_strides(dev):
    """Slices of rows, columns, every other element, transposed and permuted tensors, in place and into another layout."""
    base = _randn(dev, 1, 60, 80, 6, scale=0.1)
    views = [base[:, :, 0], base[:, 3:40, 1], base[::2, ::3, 2].t(), base[5, :, 3], base[:, 7, 4], base[:, :, 5].t()]
    keep = base.clone()
    check(views, 2.0, 1.0)
    touched = torch.zeros_like(base, dtype=torch.bool)
    for v in (touched[:, :, 0], touched[:, 3:40, 1], touched[::2, ::3, 2], touched[5, :, 3], touched[:, 7, 4], touched[:, :, 5]):
        v.fill_(True)
    assert torch.equal(base[~touched], keep[~touched]) and not torch.equal(base[touched], keep[touched])
    g = _randn(dev, 2, 40, 50)
    check([g], 2.0, 1.0, [torch.empty(50, 40, device=dev).t()])
    check([g.t()], 2.0, 1.0, [torch.empty(50, 40, device=dev)])
    check([g.expand(3, 40, 50)[:, :5, :1].to(torch.bfloat16)], 1.0, 1.0)
    assert abs(float(_gn().grad_norm([g[:1].expand(7, 50)])) - ref_norm([g[:1].expand(7, 50)], 2.0)) < 1e-5
    check([_randn(dev, 3, 6, 7, 8).permute(2, 0, 1)], 2.0, 1.0)          # dense, permuted: one run of memory
    check([torch.tensor(3.0, device=dev)], 2.0, 1.0)                     # no dimension


@pytest.mark.gpu
def test_extremes(dev):
    """Squares that overflow or vanish in fp32, infinities and NaN, nothing at all."""
    gn = _gn()
    big, small = torch.full((1000,), 1e30, device=dev), torch.full((1000,), 1e-30, device=dev)
    check([big], 2.0, 1.0)
    check([small], 2.0, 1e-35, eps=0.0)
    for bad, want in ((float('nan'), math.isnan), (float('inf'), math.isinf)):
        for p in (1.0, 2.0, INF):
            g = torch.ones(5000, device=dev)
            g[4321] = bad
            assert want(float(gn.grad_norm([g], p)))
            h = torch.ones(100, device=dev, dtype=torch.float16)
            n = gn.clip_grad_norm([h, g], 1.0, p)
            assert want(float(n))
            if math.isnan(bad):
                assert torch.isnan(h).all() and torch.isnan(g).all()
            else:                                                # scaled by 0
                assert not h.any() and torch.isnan(g[4321]) and not g[:4321].any()
    e = torch.zeros(0, device=dev)
    assert float(gn.grad_norm([e])) == 0 and float(gn.clip_grad_norm([e, e], 1.0)) == 0
    z = torch.zeros(10, device=dev)
    assert float(gn.clip_grad_norm([z], 1.0)) == 0 and not z.any()


@pytest.mark.gpu
def test_unclipped_is_untouched(dev):
    """A norm of at most max_norm leaves the bits as they are (also signed zeros), in place and into another buffer."""
    g = _randn(dev, 1, 10_001)
    g[5] = -0.0
    keep = g.clone()
    _gn().clip_grad_norm([g], 1e6)
    assert torch.equal(g.view(torch.int32), keep.view(torch.int32))
    o = torch.empty_like(g)
    _gn().clip_grad_norm([g], 1e6, out=[o])
    assert torch.equal(o.view(torch.int32), keep.view(torch.int32))


@pytest.mark.gpu
def test_more_than_2_31_elements(dev):
    n = (1 << 31) + 70_001
    g = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    g[-3:] = 2.0
    g[5] = 2.0
    assert float(_gn().clip_grad_norm([g], 1.0)) == 4.0
    assert g[-3:].tolist() == [0.5] * 3 and float(g[5]) == 0.5 and not g[6:-3].any()


@pytest.mark.gpu
def test_streams_graph_and_repeats(dev):
    gn = _gn()
    grads = [_randn(dev, i, 3000, 77 + i).to(TYPES[i % 3]) for i in range(5)]
    outs = [torch.empty_like(g, dtype=torch.float32) for g in grads]

    def run():
        n = gn.clip_grad_norm(grads, 1.0, out=outs)
        return [n.clone(), *(o.clone() for o in outs)]
    want = run()
    assert all(torch.equal(a, b) for a, b in zip(run(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = gn.clip_grad_norm(grads, 1.0, out=outs)
    for seed in range(4):
        for g in grads:
            g.copy_(_randn(dev, 10 + seed, *g.shape))
        graph.replay()
        torch.cuda.synchronize()
        held = [n.clone(), *(o.clone() for o in outs)]
        assert all(torch.equal(a, b) for a, b in zip(held, run())), seed


@pytest.mark.gpu
def test_with_and_without_host_module(dev, monkeypatch):
    """The native argument checks and the Python ones make the same call."""
    gn = _gn()
    grads = [_randn(dev, i, 300, 7 + i).to(TYPES[i % 3]) for i in range(5)] + [torch.zeros(0, device=dev)]

    def run():
        g = [t.clone() for t in grads]
        outs = tuple(torch.empty_like(t, dtype=torch.float32) for t in grads)
        return [gn.grad_norm(g, INF), gn.clip_grad_norm(g, 1.0, out=outs), *outs, gn.clip_grad_norm(g, 0.5, 1.0), *g]
    want = run()
    calls = []
    monkeypatch.setattr(_lib, '_host', _lib._NoHost)
    monkeypatch.setattr(_lib, 'check', lambda rc, what, f=_lib.check: (calls.append(what), f(rc, what)))
    got = run()
    assert len(calls) == 3 and all(a.shape == b.shape and torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError):
        gn.clip_grad_norm([grads[0], grads[0]], 1.0)

@pytest.mark.gpu
def test_refusals(dev):
    gn = _gn()
    g = torch.zeros(6, 8, device=dev)
    for bad in (lambda: gn.grad_norm([]), lambda: gn.grad_norm([g.cpu()]), lambda: gn.grad_norm([g.double()]),
                lambda: gn.grad_norm([g, g.cpu()]), lambda: gn.grad_norm([g], 3.0), lambda: gn.grad_norm([g], 'x'),
                lambda: gn.clip_grad_norm([g], -1.0), lambda: gn.clip_grad_norm([g], float('nan')),
                lambda: gn.clip_grad_norm([g], 1.0, eps=-1.0), lambda: gn.grad_norm([g, None]), lambda: gn.grad_norm([None]),
                lambda: gn.clip_grad_norm([g, g], 1.0), lambda: gn.clip_grad_norm([g[:1].expand(6, 8)], 1.0),
                lambda: gn.clip_grad_norm([g], 1.0, out=[]), lambda: gn.clip_grad_norm([g], 1.0, out=[g.half()]),
                lambda: gn.clip_grad_norm([g], 1.0, out=[g[:5]]),
                lambda: gn.clip_grad_norm([g, g.clone()], 1.0, out=[torch.zeros_like(g)] * 2),
                lambda: gn.grad_norm([torch.zeros(6, 7, 8, device=dev)[:4, :5, :6]])):
        with pytest.raises(RuntimeError):
            bad()


def test_cabi_refusals():
    L = _lib.lib()
    p, q = 256, 1024

    def arr(**kw):
        g = _lib.Grad(p, q, 1, 100, 100, 1, 100, 1, 0, 0)
        for k, v in kw.items():
            setattr(g, k, v)
        return (_lib.Grad * 1)(g)

    def clip(a, n=1, kind=2, norm=ctypes.c_void_p(256), s=ctypes.c_void_p(256), sb=8):
        return L.elr_clip_grad_norm(a, n, kind, 1.0, 1e-6, norm, s, sb, None)
    for a in (arr(data=None), arr(out=None), arr(rows=-1), arr(cols=-1), arr(type=3), arr(out_type=7), arr(data=258),
              arr(out=1026), arr(rows=1 << 40, cols=1 << 40), arr(type=2, out=p)):
        assert clip(a, sb=1 << 20) == -1
    assert clip(arr(), n=-1) == -1 and clip(None) == -1 and clip(arr(), norm=None, sb=1 << 20) == -1
    for m, eps in ((-1.0, 0.0), (float('nan'), 0.0), (1.0, -1.0), (1.0, float('nan'))):
        assert L.elr_clip_grad_norm(arr(), 1, 2, m, eps, ctypes.c_void_p(256), ctypes.c_void_p(256), 1 << 20, None) == -1
    assert clip(arr(out_type=2), sb=1 << 20) == -2 and clip(arr(), kind=3, sb=1 << 20) == -2
    assert clip(arr(), sb=7) == -3 and clip(arr(), s=None, sb=1 << 20) == -3
    assert clip(arr(), s=ctypes.c_void_p(260), sb=1 << 20) == -3
    assert L.elr_grad_norm_scratch_bytes(arr(type=9), 1) == -1
    # partial sums: one per chunk, and never many more than the chip can use
    assert 16 <= L.elr_grad_norm_scratch_bytes(arr(), 1) <= 64
    assert L.elr_grad_norm_scratch_bytes(arr(cols=1 << 34, ld=1 << 34, out_ld=1 << 34), 1) <= 8 * (8192 + 64)


def test_python_refuses_host_tensors():
    gn = _gn()
    with pytest.raises(RuntimeError, match='must be a cuda'):
        gn.grad_norm([torch.zeros(3)])
    with pytest.raises(RuntimeError, match='must be a cuda'):
        gn.clip_grad_norm([torch.zeros(3)], 1.0)


def _bytes_of(t):
    idx = torch.zeros(t.shape, dtype=torch.int64)
    for d, (n, s) in enumerate(zip(t.shape, t.stride())):
        idx = idx + (torch.arange(n) * s).view([-1 if e == d else 1 for e in range(t.dim())])
    return [t.data_ptr() + int(i) * t.element_size() + b for i in idx.reshape(-1) for b in range(t.element_size())]


def test_overlap_is_exact():
    """_lib.overlap and overlaps_itself against the sets of bytes, on random views of one buffer."""
    rng = random.Random(3)
    buf = torch.zeros(700)
    found = [0, 0, 0, 0]
    for _ in range(1500):
        views = []
        for _ in range(2):
            dt = rng.choice((torch.float32, torch.bfloat16))
            base = buf.view(dt)
            shape = [rng.randint(1, 4) for _ in range(rng.randint(0, 3))]
            stride = [rng.choice((0, 1, 2, 3, 4, 6, 8, 12, 24, 25)) for _ in shape]
            views.append(base.as_strided(shape, stride, rng.randint(0, 60)))
        sets = [_bytes_of(v) for v in views]
        assert _lib.overlap(*views) == _lib.overlap(*views[::-1]) == bool(set(sets[0]) & set(sets[1]))
        own = len(set(sets[0])) < len(sets[0])
        assert _lib.overlaps_itself(views[0]) == own
        found[bool(set(sets[0]) & set(sets[1]))] += 1
        found[2 + own] += 1
    assert min(found) > 100
    rows = torch.zeros(1 << 20, 96)                                     # told apart without a list of their rows
    assert not _lib.overlap(rows[:, :32], rows[:, 32:]) and not _lib.overlap(rows[:, ::2], rows[:, 1::2])
    assert _lib.overlap(rows[:, :33], rows[:, 32:])


def test_outputs_that_overlap():
    gn = _gn()
    flat = torch.zeros(300)
    a, b = flat[:100], flat[100:200]
    m = flat[:240].view(20, 12)
    for grads, outs in (([a, b], [b, a]),                               # swapped
                        ([flat[:200], flat[64:264]], None),             # at an offset
                        ([a], [flat[1:101]]), ([a, flat[50:60]], [torch.zeros(100), a[:10]]),
                        ([m], [flat[:240].view(12, 20).t()]),           # in place in another order
                        ([m[:, :7], m[:, 6:]], None), ([m, m[3]], None), ([flat.as_strided((5, 5), (2, 1))], None),
                        ([torch.zeros(100), b], [b, a])):
        with pytest.raises(RuntimeError, match='overlaps'):
            gn._check_outputs(grads, grads if outs is None else outs)
    for grads, outs in (([a, b], None), ([a, a], [b, flat[200:]]), ([m[:, :7], m[:, 7:]], None), ([m[::2], m[1::2]], None),
                        ([m[:, ::3].t(), m[:, 1::3], m[:, 2::3]], None), ([a, b], [a, flat[200:]]), ([a], [a.view(100)]),
                        ([a.bfloat16()[:50], a], [a[:50].clone(), b]),
                        ([flat[:0], flat[:0]], None), ([m.t(), m], [m.clone().t(), torch.zeros(20, 12)])):
        gn._check_outputs(grads, grads if outs is None else outs)


@pytest.mark.gpu
@pytest.mark.parametrize('native', [True, False])
def test_overlapping_outputs_are_refused(dev, monkeypatch, native):
    """Both host paths refuse outputs that share memory, and run nothing."""
    gn = _gn()
    if not native:
        monkeypatch.setattr(_lib, '_host', _lib._NoHost)
    flat = _randn(dev, 1, 300)
    keep = flat.clone()
    a, b, half = flat[:100], flat[100:200], flat[:100].view(torch.bfloat16)[:100]
    for grads, outs in (([a, b], [b, a]), ([flat, flat[64:]], None), ([flat[64:], flat], None), ([a], [flat[1:101]]),
                        ([a, b], [b, torch.zeros_like(b)]), ([half], [a]), ([a, flat[40:60]], [a, torch.zeros(20, device=dev)])):
        with pytest.raises(RuntimeError, match='overlaps'):
            gn.clip_grad_norm(grads, 1.0, out=outs)
        assert torch.equal(flat, keep)
    m = flat[:240].view(20, 12)
    check([m[:, :7], m[:, 7:]], 2.0, 1.0)
    check([a.clone(), b], 2.0, 1.0, [torch.empty_like(a), b])
    x = flat[:100].clone()
    check([x, x], 2.0, 1.0, [torch.empty_like(x), torch.empty_like(x)])


@pytest.mark.gpu
def test_a_list_changed_by_another_thread(dev):
    """A call works on the tensors that its list held when it began, and keeps them: their norm is that of one whole list."""
    gn = _gn()
    lists = [[torch.full((5000 + i,), v, device=dev) for i in range(40)] for v in (1.0, 2.0)]
    norms = {float(gn.grad_norm(x)) for x in lists}
    torch.cuda.synchronize()
    shared, stop = list(lists[0]), threading.Event()

    def change():
        v = 0
        while not stop.is_set():
            v = 1 - v
            shared[:] = [t.clone() for t in lists[v]]
    worker = threading.Thread(target=change)
    worker.start()
    try:
        got = [gn.grad_norm(shared) for _ in range(200)]
    finally:
        stop.set()
        worker.join()
    assert {float(x) for x in got} <= norms and len(norms) == 2


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n', [10, 5_000_000])
@pytest.mark.parametrize('out', [False, True])
def test_nothing_to_scale(dev, dtype, n, out):
    """0 / 0 and inf / inf: gradients of nothing but zeros with max_norm = eps = 0, and an infinite norm without a bound."""
    gn = _gn()
    for max_norm, eps in ((0.0, 0.0), (1.0, 0.0), (INF, 0.0)):
        g = torch.zeros(n, dtype=dtype, device=dev)
        o = torch.full((n,), 7.0, device=dev)
        assert float(gn.clip_grad_norm([g], max_norm, eps=eps, out=[o] if out else None)) == 0
        assert not (o if out else g).any()
    for p in (1.0, 2.0, INF):
        g = torch.ones(n, dtype=dtype, device=dev)
        g[-1] = -INF
        o = torch.zeros(n, device=dev)
        assert float(gn.clip_grad_norm([g], INF, p, out=[o] if out else None)) == INF
        assert torch.equal((o if out else g).float(), torch.cat([torch.ones(n - 1, device=dev), g.new_full((1,), -INF).float()]))
        g[0] = float('nan')
        gn.clip_grad_norm([g], INF, p, out=[o] if out else None)
        assert torch.isnan(o if out else g).all()


def test_two_strides_of_broadcast_gradients():
    """A gradient broadcast over three dimensions or more (a sum's) into a dense output is one run of the output's memory."""
    gn = _gn()
    for shape in ((2, 3, 4), (4, 3, 2), (3, 3, 3), (5, 1, 4, 2)):
        t, o = torch.zeros(1).expand(shape), torch.zeros(shape)
        rows, cols, ld, cs, old, ocs = gn._two_strides(t, o)
        assert rows * cols == o.numel() and (ld, cs) == (0, 0)
        assert sorted(i * old + j * ocs for i in range(rows) for j in range(cols)) == list(range(o.numel()))
        p = o.permute(*reversed(range(o.dim())))
        rows, cols, ld, cs, old, ocs = gn._two_strides(t.permute(*reversed(range(o.dim()))), p)
        assert rows * cols == o.numel() and sorted(i * old + j * ocs for i in range(rows) for j in range(cols)) == list(range(o.numel()))


@pytest.mark.gpu
def test_broadcast_gradients(dev):
    for shape in ((2, 3, 4), (4, 3, 2), (7, 5, 6, 3), (30, 40, 50)):
        g = torch.full((1,), 0.5, device=dev)
        check([g.expand(shape)], 2.0, 1.0, [torch.empty(shape, device=dev)])
        check([g.to(torch.bfloat16).expand(shape), _randn(dev, 1, *shape)], 1.0, 1.0,
              [torch.empty(shape, device=dev), torch.empty(shape, device=dev)])
