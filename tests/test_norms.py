"""RMS norm with the residual's addition, fp8 output, and the backward (elara_amd.norms) against the definition in 64 bits.
No counterpart in the reference.

Bounds, with u = 2^-24: a lane adds at most max(64, D / 256) squares in a row and about 12 partial sums are joined, so the
sum of squares is within A = (max(64, D / 256) + 16) u of itself and rstd within A / 2 + 4 u.
"""
import ctypes

import pytest
import torch

from elara_amd import _lib

U = 2.0 ** -24
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-37}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
EPS = 1e-6


def _nm():
    from elara_amd import norms
    return norms


def _adds(D):
    return (max(64, D / 256) + 16) * U


def _randn(dev, seed, *shape, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dev)


def _close(got, ref, bound):
    """Finite places within the bound, the others alike."""
    got = got.double()
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    d = (got - ref).abs()
    assert bool((d[fin] <= bound[fin]).all()), float((d - bound)[fin].max())


def _ref(x, w, r, eps=EPS):
    h = x.double() + (r.double() if r is not None else 0)
    rstd = 1 / torch.sqrt((h * h).mean(-1) + eps)
    y = h * rstd[..., None] * (w.double() if w is not None else 1.0)
    return h, rstd, y


def check(x, w, r, fp8=None, eps=EPS):
    nm = _nm()
    D, dt = x.shape[-1], x.dtype
    h, rstd, y = _ref(x, w, r, eps)
    res = nm.rms_norm(x, w, eps, residual=r) if fp8 is None else nm.rms_norm_fp8(x, w, eps, residual=r, group=fp8)
    rel = _adds(D) + 8 * U
    _close(res.rstd, rstd, rel * rstd)
    if r is not None:
        assert res.h.dtype == r.dtype and res.h.shape == x.shape
        _close(res.h, h, (HALF_ULP[r.dtype] + 2 * U) * h.abs() + TINY[r.dtype])
    else:
        assert res.h is x
    if fp8 is None:
        assert res.y.dtype == dt and res.y.shape == x.shape
        _close(res.y, y, (rel + HALF_ULP[dt] * (1 + rel)) * y.abs() + TINY[dt])
        return res
    assert res.y.dtype == torch.float8_e4m3fn and res.y.shape == x.shape
    grp = y.reshape(x.shape[:-1] + (-1, fp8 or D))
    amax = grp.abs().amax(-1)
    scale = torch.where(amax > 0, amax / 448, 1.0)
    assert res.scale.shape == scale.shape and res.scale.dtype == torch.float32
    _close(res.scale, scale, (rel + 2 * U) * scale)
    # a value is within half a step of e4m3 (2^-4 of itself, 2^-10 where it is subnormal) and the fp32 error before it
    back = res.y.double().reshape(grp.shape) * scale[..., None]
    bound = torch.maximum(grp.abs() * 2.0 ** -4, scale[..., None] * 2.0 ** -10) * (1 + 1e-3) + 4 * rel * grp.abs()
    _close(back, grp, bound)
    return res


def check_back(dy, h, w, dh, rstd=None):
    nm = _nm()
    D, n = h.shape[-1], h.numel() // h.shape[-1]
    if rstd is None:
        rstd = (1 / torch.sqrt((h.double() ** 2).mean(-1) + EPS)).float()
    c, H, G = rstd.double()[..., None], h.double(), dy.double()
    W = w.double() if w is not None else torch.ones(D, dtype=torch.float64, device=h.device)
    xh, u = H * c, G * W
    dot = (u * xh).sum(-1, keepdim=True) / D
    dx = c * (u - xh * dot) + (dh.double() if dh is not None else 0)
    dw = (G * xh).reshape(n, D).sum(0)
    gx, gw = nm.rms_norm_backward(dy, h, w, rstd, dh=dh)
    assert gx.dtype == h.dtype and gx.shape == h.shape and gw.dtype == torch.float32 and gw.shape == (D,)
    a = _adds(D)
    size = c.abs() * (u.abs() + xh.abs() * (u * xh).abs().sum(-1, keepdim=True) / D)
    err = size * (a + 16 * U) + 2 * U * dx.abs()
    _close(gx, dx, err + HALF_ULP[h.dtype] * (dx.abs() + err) + TINY[h.dtype])
    adds = (n / 256 + 700) * U          # rows of one team in a row, then the teams, waves and blocks
    _close(gw, dw, adds * (G * xh).abs().reshape(n, D).sum(0) + 1e-37)
    return gx, gw


DIMS = [1, 2, 3, 7, 8, 31, 64, 100, 127, 128, 200, 255, 256, 500, 512, 513, 1000, 1024, 2048, 2050, 4096, 5120, 8192, 8200,
        16_384, 20_001]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', DIMS)
def test_forward(dev, D, dtype):
    for n, res, wt in ((1, None, dtype), (5, dtype, torch.float32), (67, torch.float32, dtype), (3, dtype, None)):
        x = _randn(dev, D + n, n, D).to(dtype)
        r = _randn(dev, n, n, D, scale=2.0).to(res) if res else None
        w = (1 + 0.1 * _randn(dev, 5, D)).to(wt) if wt else None
        check(x, w, r)
        check(x, w, r, fp8=0)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('group', [32, 64, 128, 256])
@pytest.mark.parametrize('D', [256, 512, 768, 2048, 8192, 16_384, 16_640])
def test_fp8_groups(dev, D, group, dtype):
    for n, res in ((1, dtype), (33, None)):
        x = _randn(dev, D + group, n, D).to(dtype)
        x[:, :group] = 0                                    # a group of nothing: scale 1
        if n > 1:
            x[:, group:2 * group] *= 2.0 ** -10 if D > group else 1.0
        r = torch.zeros_like(x) if res else None
        out = check(x, None, r, fp8=group)
        assert bool((out.scale[:, 0] == 1).all()) and not out.y.view(torch.uint8)[:, :group].any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', DIMS)
def test_backward(dev, D, dtype):
    for n, ht, wt, with_dh in ((1, dtype, dtype, False), (5, dtype, torch.float32, True), (67, torch.float32, dtype, True),
                               (2100 if D <= 1024 else 600, dtype, None, False)):
        h = _randn(dev, D + n, n, D).to(ht)
        dy = _randn(dev, n, n, D, scale=1e-2).to(dtype)
        w = (1 + 0.1 * _randn(dev, 5, D)).to(wt) if wt else None
        dh = _randn(dev, 7, n, D, scale=1e-2).to(ht) if with_dh else None
        check_back(dy, h, w, dh)


@pytest.mark.gpu
def test_special_values(dev):
    nm = _nm()
    for D in (64, 4096, 20_000):
        x = _randn(dev, D, 6, D)
        x[0] = 0                                            # rstd 1 / sqrt(eps), y 0
        x[1, 3] = float('nan')
        x[2, 1] = float('inf')
        x[3] *= 2.0 ** -60
        out = nm.rms_norm(x, None)
        ref = _ref(x, None, None)[2]
        assert torch.equal(torch.isnan(out.y), torch.isnan(ref)) and not out.y[0].any()
        q = nm.rms_norm_fp8(x, None)
        assert torch.isnan(q.scale[1]).all() and torch.isnan(q.y[1].float()).all() and q.scale[0] == 1
        assert torch.isfinite(q.y[3:].float()).all()
        check(x[3:], None, None, fp8=0)


def quotients(x, w, r, rstd, group):
    """(e4m3 bytes, scales) of rstd's row sums by the definition, each fp32 operation rounded once (IEEE, on the CPU)."""
    x, rstd = x.cpu().float(), rstd.cpu()
    h = x + r.cpu().float() if r is not None else x
    y = (h * rstd[:, None]) * (w.cpu().float() if w is not None else 1.0)
    grp = y.view(y.shape[0], -1, group or y.shape[1])
    amax = grp.abs().amax(-1, keepdim=True)
    scale = amax / torch.full_like(amax, 448.0)
    scale = torch.where(scale == 0, 1.0, scale)
    return (grp / scale).clamp(-448.0, 448.0).view_as(y).to(torch.float8_e4m3fn), scale[..., 0]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D,group', [(64, 0), (64, 32), (1000, 0), (2048, 128), (4096, 0), (4096, 256), (20_480, 0), (20_480, 64)])
def test_fp8_is_the_rounded_quotient(dev, D, group, dtype):
    """Every byte is y / scale rounded, and every scale max|y| / 448, also where quotients lie on e4m3's ties: whole numbers
    up to a largest of 448, of which rstd cancels.  A large and a tiny row, whose scales divide otherwise, are among them."""
    n = 400
    x = torch.randint(-447, 448, (n, D), generator=torch.Generator().manual_seed(D + group)).float()
    x[:, ::group or D] = 448.0
    x[0] *= 2.0 ** -120 if dtype != torch.float16 else 1.0
    x[1] = -0.0
    x = x.to(dtype).to(dev)
    w = torch.where(torch.arange(D) % 3 == 0, -1.0, 1.0).to(dev)
    for weight, eps in ((None, EPS), (w, 1.0)):
        q = _nm().rms_norm_fp8(x, weight, eps, group=group)
        y, scale = quotients(x, weight, None, q.rstd, group)
        assert torch.equal(q.scale.cpu(), scale)
        assert torch.equal(q.y.cpu().view(torch.uint8), y.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D,group', [(64, 32), (256, 64), (2048, 128), (20_480, 32), (64, 0), (500, 0), (4096, 0), (20_480, 0)])
def test_fp8_of_values_below_any_scale(dev, D, group, dtype):
    """Groups (or rows) of zeros and one value so small that max|y| / 448 rounds to 0: scale 1, no NaN; beside it the
    values whose scale is a subnormal."""
    x = torch.zeros(6, D)
    if group:
        x[:, group:] = torch.randn(6, D - group, generator=torch.Generator().manual_seed(D))
    x[:, 3] = torch.tensor([1.0, -1.0, 0.0, 1.0, 1.0, 2.0])
    x = x.to(dtype).to(dev)
    w = torch.ones(D, device=dev)
    w[3] = 2.0 ** -136
    q = _nm().rms_norm_fp8(x, w, 1e4, group=group)              # rstd about 1/100: |y| 82 or 164 times 2^-149
    y, scale = quotients(x, w, None, q.rstd, group)
    assert bool((q.scale[:, 0] == 1).all()) and not q.y[:, :group or D].float().any()
    w[3] = 2.0 ** -133
    p = _nm().rms_norm_fp8(x, w, 1.0, group=group)
    z, tiny = quotients(x, w, None, p.rstd, group)
    assert bool((tiny[[0, 1, 3, 4, 5], 0] < 2.0 ** -130).all()) and tiny[2, 0] == 1 and bool((p.scale[:2, 0] > 0).all())
    for a, b, s, t in ((q.y, y, q.scale, scale), (p.y, z, p.scale, tiny)):
        assert torch.isfinite(a.float()).all() and torch.equal(s.cpu(), t)
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
def test_layouts(dev):
    """Row strides, broadcast and transposed rows, unaligned bases, leading dimensions, no rows; in place over dh."""
    nm = _nm()
    base = _randn(dev, 1, 12, 1031).to(torch.bfloat16)
    w = (1 + 0.1 * _randn(dev, 2, 1001)).to(torch.bfloat16)
    x, r = base[:, 3:1004], base[:, 13:1014]
    check(x, w, r)
    check(x, w, r, fp8=0)
    check(base[:1, :1001].expand(12, 1001), w, r)
    check(base[:, :1001].t().contiguous().t(), w, r.t().contiguous().t())
    check(x.reshape(3, 4, 1001), w, r.reshape(3, 4, 1001))
    check(base[0, :1001], w, None)                          # one dimension: rstd is a scalar
    check_back(x, r, w, base[:, 20:1021])
    check_back(base[:, :1001].t().contiguous().t(), r, w, None)
    check_back(x.reshape(3, 4, 1001), r.reshape(3, 4, 1001), w, None)
    e = nm.rms_norm_fp8(base[:0], None, residual=base[:0])
    assert e.y.shape == (0, 1031) and e.scale.shape == (0, 1) and e.h.shape == (0, 1031)
    dx, dw = nm.rms_norm_backward(base[:0], base[:0], None, e.rstd)
    assert dx.shape == (0, 1031) and not dw.any()
    dx, dw = nm.rms_norm_backward(x, r, w, nm.rms_norm(r, w).rstd, need_dweight=False)
    assert dw is None and torch.equal(dx, nm.rms_norm_backward(x, r, w, nm.rms_norm(r, w).rstd)[0])


@pytest.mark.gpu
@pytest.mark.parametrize('D', [48, 4096])
def test_gradient_against_differences(dev, D):
    """Directional derivatives of the forward kernel in x and the weight.  A central difference of step s errs by s^2 / 6
    times the third derivative (below 60 |dy| sqrt(D) here) and by the forward's error over s."""
    nm = _nm()
    n, s = 4, 2.0 ** -7
    x, w = _randn(dev, 1, n, D), 1 + 0.1 * _randn(dev, 2, D)
    v, vw = _randn(dev, 3, n, D).clamp(-1, 1), _randn(dev, 4, D).clamp(-1, 1)
    dy = _randn(dev, 5, n, D).clamp(-1, 1) / D

    def f(a, b):
        return float((nm.rms_norm(a, b).y.double() * dy.double()).sum())
    out = nm.rms_norm(x, w)
    dx, dw = nm.rms_norm_backward(dy, out.h, w, out.rstd)
    err = n * 4 * (_adds(D) + 16 * U) / s + n * 60 * s * s / 6
    assert abs(float((dx.double() * v.double()).sum()) - (f(x + s * v, w) - f(x - s * v, w)) / (2 * s)) < err
    assert abs(float((dw.double() * vw.double()).sum()) - (f(x, w + s * vw) - f(x, w - s * vw)) / (2 * s)) < err


@pytest.mark.gpu
@pytest.mark.parametrize('D', [48, 4096])
def test_gradients_along_their_own_signs(dev, D):
    """Central differences along the signs of the reference gradients, and along x's, where only the term with the row's mean
    keeps the derivative small (dy has a part along x): each is checked against more than ten times what the difference may
    err by.  For |v| <= 1, q = mean h^2 + eps and c = q^(-1/2): |q'| <= 2 (sqrt(q) + s), |q''| <= 2, and the third derivative of
    a row's y is at most (|x| + s) times c's third, plus 3 times its second, of each weight."""
    nm = _nm()
    n, s = 4, 2.0 ** -7
    x, w = _randn(dev, 1, n, D), 1 + 0.1 * _randn(dev, 2, D)
    dy = _randn(dev, 5, n, D) + x
    X, W, G = x.double(), w.double(), dy.double()
    _, c, y = _ref(x, w, None)
    c = c[:, None]
    mean = (G * W * X * c).mean(-1, keepdim=True)
    dx_ref, dw_ref = c * (G * W - X * c * mean), (G * X * c).sum(0)

    def f(a, b):
        return float((nm.rms_norm(a, b).y.double() * G).sum())
    out = nm.rms_norm(x, w)
    dx, dw = (t.double() for t in nm.rms_norm_backward(dy, out.h, w, out.rstd))
    q = (X * X).mean(-1, keepdim=True) + EPS
    low, q1 = (q.sqrt() - s) ** 2, 2 * (q.sqrt() + s)
    c2 = 0.75 * low ** -2.5 * q1 ** 2 + low ** -1.5
    c3 = 15 / 8 * low ** -3.5 * q1 ** 3 + 9 / 2 * low ** -2.5 * q1
    third = float(((G * W).abs() * ((X.abs() + s) * c3 + 3 * c2)).sum())
    err_w = 1.1 * float((G * y).abs().sum()) * (_adds(D) + 12 * U) / s
    err = err_w + third * s * s / 6
    for v in (dx_ref.sign(), X.sign()):
        t = (s * v).float()
        diff = (f(x + t, w) - f(x - t, w)) / (2 * s)
        assert abs(float((dx * v).sum()) - diff) < err
    assert float(dx_ref.abs().sum()) > 10 * err and abs(float((X.sign() * X * c * c * mean).sum())) > 10 * err
    t = (s * dw_ref.sign()).float()
    diff = (f(x, w + t) - f(x, w - t)) / (2 * s)
    assert abs(float((dw * dw_ref.sign()).sum()) - diff) < err_w and diff > 10 * err_w


@pytest.mark.gpu
def test_offsets_beyond_32_bits(dev):
    nm = _nm()
    n, D = 1_050_000, 2048                                  # 2.15 * 10^9 elements
    x = torch.zeros(n, D, dtype=torch.bfloat16, device=dev)
    x[-3:] = _randn(dev, 1, 3, D).to(torch.bfloat16)
    out = nm.rms_norm(x, None)
    assert torch.equal(out.y[-3:], nm.rms_norm(x[-3:].contiguous(), None).y) and not out.y[0].any()
    dx, _ = nm.rms_norm_backward(x, x, None, out.rstd)
    assert torch.equal(dx[-3:], nm.rms_norm_backward(x[-3:].contiguous(), x[-3:].contiguous(), None, out.rstd[-3:])[0])


@pytest.mark.gpu
def test_more_rows_than_a_launch(dev):
    nm = _nm()
    n = (1 << 21) + 9
    x = _randn(dev, 1, 1 << 12, 64).to(torch.bfloat16).repeat((1 << 9) + 1, 1)[:n]
    r = torch.ones_like(x)
    out, q = nm.rms_norm(x, None, residual=r), nm.rms_norm_fp8(x, None, residual=r, group=32)
    for a in (0, (1 << 21) - 3, n - 7):
        s = slice(a, a + 7)
        want = nm.rms_norm(x[s].clone(), None, residual=r[s].clone())
        wq = nm.rms_norm_fp8(x[s].clone(), None, residual=r[s].clone(), group=32)
        assert all(torch.equal(p[s], w) for p, w in zip(out, want))
        assert torch.equal(q.y[s].view(torch.uint8), wq.y.view(torch.uint8)) and torch.equal(q.scale[s], wq.scale)

@pytest.mark.gpu
def test_weight_gradient_of_more_columns_than_a_launch(dev):
    """Rows of 2^27 + 33: the sum of the blocks' weight gradients takes several launches; without rows it is 0."""
    nm = _nm()
    n, D = 4, (1 << 27) + 33
    empty = torch.zeros(0, D, dtype=torch.bfloat16, device=dev)
    dw = nm.rms_norm_backward(empty, empty, None, torch.zeros(0, device=dev))[1]
    assert dw.shape == (D,) and not dw.any()
    i = torch.arange(D, device=dev)
    h = torch.stack([((i + 3 * r) % 251 - 125).to(torch.bfloat16) for r in range(n)])
    dy = torch.stack([((i + r) % 7 - 3).to(torch.bfloat16) for r in range(n)])
    rstd = torch.tensor([0.5, 0.25, 1.0, 2.0], device=dev)               # whole numbers and powers of two: sums are exact
    dw = nm.rms_norm_backward(dy, h, None, rstd)[1]
    for a in range(0, D, 1 << 25):
        s = slice(a, min(D, a + (1 << 25)))
        assert torch.equal(dw[s], (dy[:, s].float() * h[:, s].float() * rstd[:, None]).sum(0))


@pytest.mark.gpu
def test_streams_graph_and_repeats(dev):
    """A side stream and every replay of a graph give the eager bits; so do repeated calls (the weight gradient's order)."""
    nm = _nm()
    x, r = _randn(dev, 1, 3000, 512).to(torch.bfloat16), _randn(dev, 2, 3000, 512).to(torch.bfloat16)
    w = torch.ones(512, dtype=torch.bfloat16, device=dev)

    def all_():
        a = nm.rms_norm(x, w, residual=r)
        q = nm.rms_norm_fp8(x, w, residual=r, group=128)
        return [a.y, a.h, a.rstd, q.y.view(torch.uint8), q.scale, *nm.rms_norm_backward(a.y, a.h, w, a.rstd, dh=x)]
    want = all_()
    assert all(torch.equal(a, b) for a, b in zip(all_(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = all_()
    for seed in range(4):
        x.copy_(_randn(dev, 10 + seed, 3000, 512))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, all_())), seed


@pytest.mark.gpu
def test_with_and_without_host_module(dev, monkeypatch):
    """The native argument checks and the Python ones make the same call."""
    nm = _nm()
    x, r = _randn(dev, 1, 2, 5, 256).to(torch.bfloat16), _randn(dev, 2, 2, 5, 256)
    w = torch.full((256,), 1.5, dtype=torch.bfloat16, device=dev)

    def run():
        a, b = nm.rms_norm(x, w, residual=r), nm.rms_norm(x, None)
        assert b.h is x
        q, p = nm.rms_norm_fp8(x, w, residual=r, group=64), nm.rms_norm_fp8(x, w)
        return [*a, b.y, b.rstd, q.y.view(torch.uint8), *q[1:], p.y.view(torch.uint8), p.scale,
                *nm.rms_norm_backward(x, a.h, w, a.rstd, dh=r), nm.rms_norm_backward(x, x, None, b.rstd, need_dweight=False)[0]]
    want = run()
    calls = []
    monkeypatch.setattr(_lib, '_host', _lib._NoHost)
    monkeypatch.setattr(_lib, 'check', lambda rc, what, f=_lib.check: (calls.append(what), f(rc, what)))
    got = run()
    assert len(calls) == 6 and all(a.shape == b.shape and torch.equal(a, b) for a, b in zip(got, want))

@pytest.mark.gpu
def test_refusals(dev):
    nm = _nm()
    x = torch.zeros(4, 96, dtype=torch.bfloat16, device=dev)
    rstd = torch.ones(4, device=dev)
    for bad in (lambda: nm.rms_norm(x.cpu(), None), lambda: nm.rms_norm(x.double(), None), lambda: nm.rms_norm(x[:, :0], None),
                lambda: nm.rms_norm(x, torch.ones(95, device=dev)), lambda: nm.rms_norm(x, torch.ones(96)),
                lambda: nm.rms_norm(x, torch.ones(96, device=dev).half()), lambda: nm.rms_norm(x, None, residual=x[:3]),
                lambda: nm.rms_norm(x, None, residual=x.half()), lambda: nm.rms_norm_fp8(x, None, group=64),
                lambda: nm.rms_norm_fp8(x, None, group=48), lambda: nm.rms_norm_fp8(x, None, group=-32),
                lambda: nm.rms_norm_backward(x, x.half(), None, rstd), lambda: nm.rms_norm_backward(x, x[:3], None, rstd),
                lambda: nm.rms_norm_backward(x, x, None, rstd[:3]), lambda: nm.rms_norm_backward(x, x, None, rstd.double()),
                lambda: nm.rms_norm_backward(x, x, None, rstd, dh=x.float())):
        with pytest.raises(RuntimeError):
            bad()


def test_cabi_refusals():
    L = _lib.lib()
    p = ctypes.c_void_p(256)

    def fwd(x=p, type=2, n=4, D=128, x_ld=128, r=None, rt=2, r_ld=128, w=p, wt=2, y=p, fp8=0, group=0, scale=None, h=None,
            rstd=p):
        return L.elr_rms_norm(x, type, n, D, x_ld, r, rt, r_ld, w, wt, 1e-6, y, fp8, group, scale, h, rstd, None)

    def bwd(dy=p, type=2, n=4, D=128, ld=128, h=p, ht=2, dh=None, w=p, wt=2, rstd=p, dx=p, dw=p, s=p, sb=1 << 30):
        return L.elr_rms_norm_backward(dy, type, n, D, ld, h, ht, 128, dh, 128, w, wt, rstd, dx, dw, s, sb, None)
    assert fwd(n=0, x=None) == 0 and bwd(n=0, dw=None) == 0
    for rc in (fwd(x=None), fwd(type=5), fwd(n=-1), fwd(D=0), fwd(x_ld=-1), fwd(r=p), fwd(y=None), fwd(rstd=None), fwd(fp8=1),
               fwd(group=128), fwd(fp8=1, scale=p, group=96), fwd(fp8=1, scale=p, group=-32), fwd(x=ctypes.c_void_p(257)),
               bwd(dy=None), bwd(h=None), bwd(rstd=None), bwd(dx=None), bwd(ld=-1), bwd(dx=ctypes.c_void_p(257))):
        assert rc == -1
    for rc in (fwd(rt=1), fwd(wt=1), fwd(type=0, rt=2), fwd(D=1 << 29), fwd(fp8=1, scale=p, group=16), bwd(ht=1),
               bwd(type=0, ht=2)):
        assert rc == -2
    need = L.elr_rms_norm_backward_scratch_bytes(4, 128, 2)
    assert need > 0 and bwd(sb=need - 1) == -3 and bwd(s=None) == -3
    assert L.elr_rms_norm_backward_scratch_bytes(4, 0, 2) == -1 and L.elr_rms_norm_backward_scratch_bytes(4, 8, 9) == -1


def test_python_refuses_host_tensors():
    nm = _nm()
    for f in (lambda: nm.rms_norm(torch.zeros(2, 8), None), lambda: nm.rms_norm_fp8(torch.zeros(2, 8), None),
              lambda: nm.rms_norm_backward(torch.zeros(2, 8), torch.zeros(2, 8), None, torch.ones(2))):
        with pytest.raises(RuntimeError, match='must be a cuda'):
            f()
