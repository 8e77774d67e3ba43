"""Rows in 8-bit integers (elara_amd.int8) and the norm's backward from them, against the definitions in 64 bits.  No counterpart in
the reference.

Bounds, with u = 2^-24 (half a step of fp32).  Quantizing and widening have none: scale and q are equal.  The product's sum is exact,
then come three fp32 roundings (of the sum, times two scales) and the output's own.  The weight gradient's products are exact and its
sums fp32: at most n + 64 additions, each off by at most a whole step (2 u) of a sum that stays below sum |dy x|.  The norm's backward
has the bounds of tests/test_norms.py.
"""
import ctypes

import pytest
import torch

from elara_amd import _lib

U = 2.0 ** -24
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-37}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
GROUPS = [0, 32, 64, 128, 256]
EPS = 1e-6


def _i8():
    from elara_amd import int8
    return int8


def _randn(seed, *shape, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


def _grouped(x, group):
    D = x.shape[-1]
    g = group or D
    m = -(-D // g)
    if m * g != D:
        x = torch.nn.functional.pad(x, (0, m * g - D))
    return x.reshape(x.shape[:-1] + (m, g))


def ref_quantize(x, group, pow2):
    """(q, scale) by the definition, x on the CPU."""
    D = x.shape[-1]
    grp = _grouped(x.double(), group)
    amax = grp.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(amax)
    if pow2:
        m, e = torch.frexp(amax)                                   # amax = m 2^e, m in [0.5, 1)
        s = torch.ldexp(torch.ones_like(amax), torch.where(m <= 127 / 128, e - 7, e - 6).clamp(min=-126))
        s = torch.where(amax > 0, s, 1.0)
    else:
        s = (amax / 127).float().double()
        s = torch.where(s > 0, s, 1.0)
    q = torch.where(bad, 0.0, torch.round(grp / s)).clamp(-127, 127)
    s = torch.where(bad, float('nan'), s)
    return q.reshape(x.shape[:-1] + (-1,))[..., :D].to(torch.int8), s[..., 0].float()


def values(q, scale, group):
    g = _grouped(q.float(), group) * scale[..., None]
    return g.reshape(q.shape[:-1] + (-1,))[..., :q.shape[-1]]


def same(a, b):
    assert a.shape == b.shape and a.dtype == b.dtype
    assert torch.equal(torch.nan_to_num(a.cpu().float(), nan=12345.0), torch.nan_to_num(b.cpu().float(), nan=12345.0))


def check_quantize(dev, x, group, pow2, view=lambda t: t):
    i8 = _i8()
    q, s = ref_quantize(x, group, pow2)
    r = i8.quantize(view(x.to(dev)), group=group, pow2=pow2)
    same(r.scale, s)
    same(r.q, q)
    assert r.group == group
    for t in TYPES:
        same(i8.dequantize(r, dtype=t), values(q, s, group).to(t))
    if pow2 and torch.isfinite(s).all():
        assert torch.equal(i8.dequantize(r, dtype=torch.bfloat16).cpu().double(), values(q, s, group).double())
    return r


DIMS = [1, 3, 16, 31, 33, 64, 100, 128, 200, 257, 500, 513, 1000, 1024, 2048, 4096, 5120, 8200, 20_001, 40_000]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', DIMS)
def test_quantize(dev, D, dtype):
    for n in (1, 7) if D > 5000 else (1, 5, 300):
        x = (_randn(D + n, n, D) * (1 + 50 * torch.rand(n, 1, generator=torch.Generator().manual_seed(n)))).to(dtype)
        for group in GROUPS:
            check_quantize(dev, x, group, True)
            check_quantize(dev, x, group, False)


@pytest.mark.gpu
@pytest.mark.parametrize('pow2', [False, True])
@pytest.mark.parametrize('group', GROUPS)
def test_quantize_special_values(dev, group, pow2):
    for D in (64, 300, 4096, 20_000):
        x = _randn(D, 12, D)
        x[0] = 0
        x[1, 5] = float('nan')
        x[2, 3] = float('inf')
        x[3, D - 1] = float('-inf')
        x[4] *= 1e-42                                       # subnormal, scales among them
        x[5] *= 1e-38
        x[6] = torch.finfo(torch.float32).max
        x[7] = -0.0
        x[8] = 1.4e-45
        x[9] *= 1e30
        x[10] = 127.0 * 2.0 ** -3                           # the power of two itself reaches 127
        x[11, 0] = 127.0 * (1 + 2.0 ** -23)                 # just beyond it
        check_quantize(dev, x, group, pow2)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_quantize_ties_to_even(dev, dtype):
    """Half steps of a scale of 1, 2^-3 and 3 (a scale of max / 127 whose quotients fp32 cannot hold)."""
    for s in (1.0, 0.125, 3.0):
        x = (torch.arange(-127, 127) + 0.5).repeat(2, 1) * s
        x = torch.cat([x, torch.full((2, 1), 127.0 * s)], 1).to(dtype)
        r = check_quantize(dev, x, 0, False)
        if dtype != torch.bfloat16 or s != 3.0:
            assert not (r.q[0, :-1] % 2).any() or dtype == torch.bfloat16
        check_quantize(dev, x, 0, True)
    x = torch.full((1, 4), 127.0 * (1 + 2.0 ** -20))        # quotients a little off a tie
    scale = float((x[0, 0].double() / 127).float())
    x[0, 1:] = torch.tensor([2.5 * scale, 2.5 * scale * (1 + 2.0 ** -23), 2.5 * scale * (1 - 2.0 ** -23)])
    check_quantize(dev, x, 0, False)


@pytest.mark.gpu
def test_quantize_strides_and_shapes(dev):
    i8 = _i8()
    x = _randn(1, 40, 300).bfloat16()
    for view in (lambda t: torch.cat([t, t], 1)[:, :300], lambda t: torch.cat([t, t], 1)[:, 300:],
                 lambda t: t.t().contiguous().t(), lambda t: torch.cat([t[:, :1], t], 1)[:, 1:]):
        check_quantize(dev, x, 64, True, view)
        check_quantize(dev, x, 0, False, view)
    y = x.to(dev)
    r = i8.quantize(y.view(2, 4, 5, 300), group=128, pow2=True)
    assert r.q.shape == (2, 4, 5, 300) and r.scale.shape == (2, 4, 5, 3)
    assert torch.equal(r.q.view(40, 300), i8.quantize(y, group=128, pow2=True).q)
    one = i8.quantize(y[0], group=0)
    assert one.q.shape == (300,) and one.scale.shape == (1,)
    same(i8.quantize(y[:1].expand(7, 300)).q, i8.quantize(y[:1]).q.expand(7, 300).contiguous())
    for shape in ((0, 8), (3, 0, 8)):
        r = i8.quantize(torch.zeros(shape, device=dev))
        assert r.q.shape == shape and i8.dequantize(r).shape == shape
    part = i8.Int8Rows(torch.cat([i8.quantize(y).q] * 2, 1)[:, 300:], i8.quantize(y).scale, 0)
    same(i8.dequantize(part), i8.dequantize(i8.quantize(y)))


@pytest.mark.gpu
def test_many_short_rows(dev):
    """More rows than a launch's blocks would hold one by one, of a width that leaves lanes idle."""
    i8 = _i8()
    x = torch.randn(2_200_000, 5, device=dev)
    r = i8.quantize(x, group=32, pow2=True)
    s = i8.quantize(x)
    pick = torch.tensor([0, 1, 7, 999_999, 2_097_151, 2_097_152, 2_199_999], device=dev)
    q, sc = ref_quantize(x[pick].cpu(), 32, True)
    same(r.q[pick], q)
    same(r.scale[pick], sc)
    q, sc = ref_quantize(x[pick].cpu(), 0, False)
    same(s.q[pick], q)
    same(s.scale[pick], sc)
    same(i8.dequantize(r, torch.float32)[pick], (r.q.float() * r.scale)[pick])


# ---- the product

def _int_rows(seed, n, K, low=-127, high=127):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(low, high + 1, (n, K), generator=g, dtype=torch.int32).to(torch.int8)


def check_linear(dev, xq, wq, dtype, xs=None, ws=None):
    i8 = _i8()
    n, N = xq.shape[0], wq.shape[0]
    xs = torch.rand(n, 1, generator=torch.Generator().manual_seed(n)) * 0.1 + 1e-3 if xs is None else xs
    ws = torch.rand(N, 1, generator=torch.Generator().manual_seed(N + 1)) * 0.02 + 1e-4 if ws is None else ws
    y = i8.linear(i8.Int8Rows(xq.to(dev), xs.to(dev), 0), i8.Int8Rows(wq.to(dev), ws.to(dev), 0), dtype=dtype)
    assert y.shape == (n, N) and y.dtype == dtype
    acc = xq.to(dev).double() @ wq.to(dev).double().t()
    ref = acc * xs.to(dev).double() * ws.to(dev).double().t()
    bound = (3 * U * (1 + 4 * U) + HALF_ULP[dtype] * (1 + 4 * U)) * ref.abs() + TINY[dtype]
    assert bool(((y.double() - ref).abs() <= bound).all()), float(((y.double() - ref).abs() - bound).max())
    return y


SHAPES = [(1, 1, 1), (1, 7, 16), (2, 64, 64), (3, 130, 17), (4, 256, 4096), (5, 33, 100), (8, 1000, 256), (15, 129, 1000),
          (16, 512, 2048), (17, 513, 333), (31, 65, 128), (33, 64, 15), (48, 200, 96), (64, 300, 512), (65, 257, 250),
          (100, 1024, 64), (127, 127, 127), (128, 128, 128), (129, 1000, 1000), (255, 256, 4096), (256, 300, 192),
          (300, 20_011, 100), (513, 515, 1024), (1000, 700, 4097), (2048, 2048, 512), (3000, 4100, 144), (12_001, 1027, 80),
          (4099, 3333, 400)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,N,K', SHAPES)
def test_linear(dev, n, N, K, dtype):
    check_linear(dev, _int_rows(n, n, K), _int_rows(N + 7, N, K), dtype)


@pytest.mark.gpu
def test_linear_places_of_every_product(dev):
    """One value a row at a place of its own: each output is one product, so a misplaced lane or column shows."""
    for n, N, K in ((1, 300, 1024), (16, 272, 512), (64, 300, 320), (200, 260, 384), (300, 520, 1040), (3300, 3900, 272)):
        xq = torch.zeros(n, K, dtype=torch.int8)
        xq[torch.arange(n), (torch.arange(n) * 37 + 5) % K] = (torch.arange(n) % 127 + 1).to(torch.int8)
        check_linear(dev, xq, _int_rows(3, N, K), torch.float32)
        check_linear(dev, _int_rows(4, n, K), torch.eye(N, K, dtype=torch.int8), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_linear_few_tokens_and_many_channels(dev, dtype):
    """Where the size of the tiles changes with the tokens (128 and 129) and with the channels (48,896 and the next)."""
    for n, N in ((33, 48_896), (64, 48_897), (65, 49_152), (128, 48_897), (128, 65_544), (129, 48_896), (129, 48_897)):
        for K in (64, 400):
            check_linear(dev, _int_rows(n, n, K), _int_rows(N, N, K), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_linear_few_steps_of_k(dev, dtype):
    """Fewer steps of K than are started ahead, and as many or a few more, whole and ending inside: what was started past K does
    not reach the outputs.  Every product is 127 x 100, so that a missing or a repeated step shows everywhere."""
    for n, N in ((33, 64), (64, 200), (200, 190), (129, 33_000)):
        for K in (16, 112, 128, 144, 256, 272, 384, 400, 496, 512, 528, 640, 1024):
            y = check_linear(dev, torch.full((n, K), 127, dtype=torch.int8), torch.full((N, K), 100, dtype=torch.int8), dtype,
                             xs=torch.full((n, 1), 2.0 ** -20), ws=torch.ones(N, 1))
            assert bool((y == y[0, 0]).all())


@pytest.mark.gpu
def test_linear_largest_sums(dev):
    """Every product 2^14 at the largest K: the int32 sum is 2^31 - 2^14."""
    K = 131_071
    for n in (1, 5, 40, 200):
        y = check_linear(dev, torch.full((n, K), -128, dtype=torch.int8), torch.full((70, K), -128, dtype=torch.int8), torch.float32,
                         xs=torch.ones(n, 1), ws=torch.ones(70, 1))
        assert float(y[0, 0]) == float(torch.tensor(K * 16384.0))
        check_linear(dev, torch.full((n, K), -128, dtype=torch.int8), torch.full((70, K), 127, dtype=torch.int8), torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize('n', [3, 40, 300])
def test_linear_strides(dev, n):
    i8 = _i8()
    for K in (64, 100, 512):
        x, w = _int_rows(1, n, K).to(dev), _int_rows(2, 200, K).to(dev)
        xs, ws = torch.rand(n, 1, device=dev), torch.rand(200, 1, device=dev)
        y = i8.linear(i8.Int8Rows(x, xs, 0), i8.Int8Rows(w, ws, 0))
        for off in (1, 4, 16):
            xv = torch.full((n, K + 48), 99, dtype=torch.int8, device=dev)[:, off:off + K].copy_(x)
            wv = torch.full((200, K + 33), 99, dtype=torch.int8, device=dev)[:, off:off + K].copy_(w)
            assert torch.equal(i8.linear(i8.Int8Rows(xv, xs, 0), i8.Int8Rows(wv, ws, 0)), y)
        z = i8.linear(i8.Int8Rows(x.t().contiguous().t(), xs, 0), i8.Int8Rows(w, ws.t().contiguous().t(), 0))
        assert torch.equal(z, y)
        z = i8.linear(i8.Int8Rows(x.view(1, n, K), xs.view(1, n, 1), 0), i8.Int8Rows(w, ws, 0))
        assert z.shape == (1, n, 200) and torch.equal(z[0], y)
        z = i8.linear(i8.Int8Rows(x[:1].expand(n, K), xs, 0), i8.Int8Rows(w, ws, 0))
        assert torch.equal(z, i8.linear(i8.Int8Rows(x[:1].expand(n, K).contiguous(), xs, 0), i8.Int8Rows(w, ws, 0)))


@pytest.mark.gpu
def test_rows_far_apart(dev):
    """Offsets past 32 bits: rows 2^31 + 64 bytes apart, the last of three beyond 4 GiB."""
    i8 = _i8()
    K, far = 256, (1 << 31) + 64
    buf = torch.zeros(2 * far + K, dtype=torch.int8, device=dev)
    rows = buf.as_strided((3, K), (far, 1))
    q = _int_rows(5, 3, K).to(dev)
    rows.copy_(q)
    s, other = torch.rand(3, 1, device=dev), i8.Int8Rows(_int_rows(6, 70, K).to(dev), torch.rand(70, 1, device=dev), 0)
    assert torch.equal(i8.linear(i8.Int8Rows(rows, s, 0), other), i8.linear(i8.Int8Rows(q, s, 0), other))
    assert torch.equal(i8.linear(other, i8.Int8Rows(rows, s, 0)), i8.linear(other, i8.Int8Rows(q, s, 0)))
    assert torch.equal(i8.dequantize(i8.Int8Rows(rows, s, 0)), i8.dequantize(i8.Int8Rows(q, s, 0)))
    dy = torch.randn(3, 40, device=dev)
    assert torch.equal(i8.weight_grad(dy, i8.Int8Rows(rows, s, 0)), i8.weight_grad(dy, i8.Int8Rows(q, s, 0)))


@pytest.mark.gpu
def test_linear_special_scales_and_empty(dev):
    i8 = _i8()
    x = i8.Int8Rows(_int_rows(1, 4, 64).to(dev), torch.tensor([[1.0], [float('nan')], [0.0], [2.0]], device=dev), 0)
    w = i8.Int8Rows(_int_rows(2, 40, 64).to(dev), torch.ones(40, 1, device=dev), 0)
    y = i8.linear(x, w, dtype=torch.float32)
    assert torch.isnan(y[1]).all() and not y[2].any() and torch.isfinite(y[[0, 3]]).all()
    assert i8.linear(i8.Int8Rows(x.q[:0], x.scale[:0], 0), w).shape == (0, 40)
    assert i8.linear(x, i8.Int8Rows(w.q[:0], w.scale[:0], 0)).shape == (4, 0)


# ---- the weight gradient

def check_wgrad(dev, dy, q, scale, group, transposed=False):
    i8 = _i8()
    n, N, K = dy.shape[0], dy.shape[1], q.shape[1]
    dw = i8.weight_grad(dy.to(dev), i8.Int8Rows(q.to(dev), scale.to(dev), group), transposed=transposed)
    assert dw.dtype == torch.float32 and dw.shape == ((K, N) if transposed else (N, K))
    x = values(q, scale, group).bfloat16().to(dev).double()
    d = dy.to(dev).double()
    ref, size = d.t() @ x, d.abs().t() @ x.abs()
    got = (dw.t() if transposed else dw).double()
    bound = 2 * (n + 64) * U * size + 1e-37
    assert bool(((got - ref).abs() <= bound).all()), float(((got - ref).abs() - bound).max())
    # and what a sum in random order gives, far below the bound of the worst case: the root mean square error
    if n >= 16:
        rms = float((got - ref).square().mean().sqrt() / ref.square().mean().sqrt())
        assert rms < 8 * U * n ** 0.5, rms
    return dw


WSHAPES = [(1, 1, 1), (1, 64, 64), (2, 3, 100), (7, 65, 33), (31, 64, 128), (32, 130, 64), (33, 127, 129), (64, 256, 256),
           (100, 500, 100), (129, 96, 1000), (300, 513, 257), (1000, 64, 64), (2048, 256, 512), (5001, 100, 200), (9000, 64, 40), (200, 3500, 3601), (77, 4096, 3841),
           (65, 12_300, 1030), (16_000, 16, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,N,K', WSHAPES)
def test_weight_grad(dev, n, N, K, dtype):
    dy = _randn(n + N, n, N, scale=1e-2).to(dtype)
    x = _randn(n + K, n, K)
    for group, transposed in ((0, False), (32, True), (128, False), (256, True)):
        q, s = ref_quantize(x, group, True)
        check_wgrad(dev, dy, q, s, group, transposed)
    q, s = ref_quantize(x, 64, False)                         # scales that are no powers of two
    check_wgrad(dev, dy, q, s, 64)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_weight_grad_places(dev, dtype):
    """One token: an outer product, each of its values exact."""
    i8 = _i8()
    for N, K, at, n in ((300, 260, 0, 1), (64, 70, 33, 40), (257, 129, 77, 300), (3600, 3590, 70, 130)):
        q = torch.zeros(n, K, dtype=torch.int8)
        q[at] = (torch.arange(K) % 127 + 1).to(torch.int8)
        dy = torch.zeros(n, N, dtype=dtype)
        dy[at] = ((torch.arange(N) % 200) * 0.25 + 1).to(dtype)
        s = torch.full((n, -(-K // 32)), 1.0) * torch.exp2(torch.arange(-(-K // 32)) % 5 - 2.0)
        for transposed in (False, True):
            dw = i8.weight_grad(dy.to(dev), i8.Int8Rows(q.to(dev), s.to(dev), 32), transposed=transposed).cpu()
            ref = dy[at].double()[:, None] * values(q, s, 32)[at].double()
            assert torch.equal(dw.double(), ref.t() if transposed else ref)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_weight_grad_wide_range_of_dy(dev, dtype):
    """fp16 and fp32 gradients over their whole range keep all their bits; infinities and NaN show in their column alone."""
    i8 = _i8()
    info = torch.finfo(dtype)
    dy = torch.zeros(40, 64, dtype=dtype)
    dy[0, 0], dy[1, 1], dy[2, 2], dy[3, 3] = info.max, info.tiny, 1 + info.eps, info.min
    dy[4, 4], dy[5, 5] = float('inf'), float('nan')
    dy[6, 6], dy[7, 6] = 1.0, info.eps
    q = torch.ones(40, 32, dtype=torch.int8)
    s = torch.ones(40, 1)
    dw = i8.weight_grad(dy.to(dev), i8.Int8Rows(q.to(dev), s.to(dev), 0)).cpu().double()
    ref = dy.double().sum(0)
    fin = [c for c in range(64) if c not in (4, 5)]
    assert torch.equal(dw[fin], ref[fin][:, None].expand(len(fin), 32))
    assert torch.isinf(dw[4]).all() or torch.isnan(dw[4]).all()
    assert torch.isnan(dw[5]).all()


@pytest.mark.gpu
def test_weight_grad_strides_nan_scales_and_empty(dev):
    i8 = _i8()
    q, s = ref_quantize(_randn(1, 70, 96), 32, True)
    q, s = q.to(dev), s.to(dev)
    dy = _randn(2, 70, 50).bfloat16().to(dev)
    dw = i8.weight_grad(dy, i8.Int8Rows(q, s, 32))
    dyv = torch.full((70, 57), 9.0, device=dev).bfloat16()[:, 3:53].copy_(dy)
    qv = torch.full((70, 111), 99, dtype=torch.int8, device=dev)[:, 5:101].copy_(q)
    assert torch.equal(i8.weight_grad(dyv, i8.Int8Rows(qv, s, 32)), dw)
    assert torch.equal(i8.weight_grad(dy.t().contiguous().t(), i8.Int8Rows(q, s, 32)), dw)
    assert torch.equal(i8.weight_grad(dy.view(7, 10, 50), i8.Int8Rows(q.view(7, 10, 96), s.view(7, 10, 3), 32)), dw)
    s2 = s.clone()
    s2[11, 1] = float('nan')                                  # a group that was not finite when it was kept
    bad = i8.weight_grad(dy, i8.Int8Rows(q, s2, 32))
    assert torch.isnan(bad[:, 32:64]).all() and torch.equal(bad[:, :32], dw[:, :32]) and torch.equal(bad[:, 64:], dw[:, 64:])
    none = i8.weight_grad(dy[:0], i8.Int8Rows(q[:0], s[:0], 32))
    assert none.shape == (50, 96) and not none.any()


@pytest.mark.gpu
def test_weight_grad_against_differences(dev):
    """The gradient of sum(dy * (x W^T)) along random directions of W, by differences in 64 bits."""
    i8 = _i8()
    q, s = ref_quantize(_randn(3, 200, 96), 32, True)
    x, dy = values(q, s, 32).double(), _randn(4, 200, 60)
    W = _randn(5, 60, 96).double()
    dw = i8.weight_grad(dy.to(dev), i8.Int8Rows(q.to(dev), s.to(dev), 32)).cpu().double()
    loss = lambda w: (dy.double() * (x @ w.t())).sum()  # noqa: E731
    for seed in range(4):
        d = _randn(seed + 9, 60, 96).double()
        slope = (loss(W + d) - loss(W - d)) / 2
        assert abs(float(slope - (dw * d).sum())) <= 2 * 264 * U * float(((dy.double().abs().t() @ x.abs()) * d.abs()).sum())


# ---- the norm's backward

def _adds(D):
    return (max(64, D / 256) + 16) * U


def _close(got, ref, bound):
    got = got.double()
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    d = (got - ref).abs()
    assert bool((d[fin] <= bound[fin]).all()), float((d - bound)[fin].max())


def check_norm_back(dev, dy, h, group, pow2, w, dh):
    from elara_amd import norms
    i8 = _i8()
    D, n = h.shape[-1], h.numel() // h.shape[-1]
    rstd = (1 / torch.sqrt((h.double() ** 2).mean(-1) + EPS)).float().to(dev)
    q, s = ref_quantize(h, group, pow2)
    H = values(q, s, group).double().to(dev)
    dy, w, dh = dy.to(dev), None if w is None else w.to(dev), None if dh is None else dh.to(dev)
    gx, gw = norms.rms_norm_backward_int8(dy, i8.Int8Rows(q.to(dev), s.to(dev), group), w, rstd, dh=dh)
    c, G = rstd.double()[..., None], dy.double()
    W = w.double() if w is not None else torch.ones(D, dtype=torch.float64, device=dev)
    xh, u = H * c, G * W
    dot = (u * xh).sum(-1, keepdim=True) / D
    dx = c * (u - xh * dot) + (dh.double() if dh is not None else 0)
    dw = (G * xh).reshape(n, D).sum(0)
    xt = dh.dtype if dh is not None else dy.dtype
    assert gx.dtype == xt and gx.shape == dy.shape and gw.dtype == torch.float32 and gw.shape == (D,)
    size = c.abs() * (u.abs() + xh.abs() * (u * xh).abs().sum(-1, keepdim=True) / D)
    err = size * (_adds(D) + 16 * U) + 2 * U * dx.abs()
    _close(gx, dx, err + HALF_ULP[xt] * (dx.abs() + err) + TINY[xt])
    _close(gw, dw, (n / 256 + 700) * U * (G * xh).abs().reshape(n, D).sum(0) + 1e-37)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', [1, 7, 31, 64, 100, 128, 200, 256, 500, 513, 1024, 2048, 2050, 4096, 8192, 8200, 20_001])
def test_norm_backward(dev, D, dtype):
    for n, group, pow2, wt, dt in ((1, 0, True, dtype, None), (5, 32, True, torch.float32, dtype), (67, 128, True, dtype, torch.float32),
                                   (700 if D <= 1024 else 90, 256, False, None, None), (33, 64, True, dtype, dtype)):
        h = _randn(D + n, n, D, scale=2.0)
        dy = _randn(n, n, D, scale=1e-2).to(dtype)
        w = (1 + 0.1 * _randn(5, D)).to(wt) if wt else None
        dh = _randn(7, n, D, scale=1e-2).to(dt) if dt else None
        check_norm_back(dev, dy, h, group, pow2, w, dh)


@pytest.mark.gpu
def test_norm_backward_strides_and_flags(dev):
    from elara_amd import norms
    i8 = _i8()
    h = _randn(1, 40, 300, scale=2.0).to(dev)
    kept = i8.quantize(h, group=64, pow2=True)
    rstd = (1 / torch.sqrt((h.double() ** 2).mean(-1) + EPS)).float()
    dy, w, dh = torch.randn(40, 300, device=dev).bfloat16(), torch.rand(300, device=dev), torch.randn(40, 300, device=dev)
    a, b = norms.rms_norm_backward_int8(dy, kept, w, rstd, dh=dh)
    qv = torch.full((40, 333), 99, dtype=torch.int8, device=dev)[:, 7:307].copy_(kept.q)
    dyv = torch.full((40, 311), 9.0, device=dev).bfloat16()[:, 5:305].copy_(dy)
    c, d = norms.rms_norm_backward_int8(dyv, i8.Int8Rows(qv, kept.scale, 64), w, rstd, dh=dh.t().contiguous().t())
    assert torch.equal(a, c) and torch.equal(b, d)
    c, d = norms.rms_norm_backward_int8(dy, kept, w, rstd, dh=dh, need_dweight=False)
    assert torch.equal(a, c) and d is None
    # the exact h in 8 bits: the same as the norm's own backward
    e, f = norms.rms_norm_backward(dy, i8.dequantize(kept, torch.float32), w, rstd, dh=dh)
    assert torch.equal(a, e) and torch.equal(b, f)
    z = torch.zeros(0, 300, device=dev)
    x, y = norms.rms_norm_backward_int8(z, i8.quantize(z), w, torch.zeros(0, device=dev))
    assert x.shape == (0, 300) and not y.any()


# ---- all of them as a model uses them

@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_kept_layer_against_autograd(dev, dtype):
    """A norm and a linear layer, their inputs kept in 8 bits: the gradients are those of autograd in 64 bits at the kept values (the
    weight's at the norm's kept output, the norm's at its kept input), to the bounds above and dy's own rounding."""
    from elara_amd import norms
    i8 = _i8()
    n, D, N = 300, 200, 130
    h = _randn(1, n, D).to(dtype).to(dev)
    g, W = (1 + 0.1 * _randn(2, D)).to(dtype).to(dev), _randn(3, N, D, scale=0.1).to(dtype).to(dev)
    dout = _randn(4, n, N, scale=1e-2).to(dtype).to(dev)
    y = norms.rms_norm(h, g, EPS)
    h8, y8 = i8.quantize(h, group=32, pow2=True), i8.quantize(y.y, group=32, pow2=True)
    dW = i8.weight_grad(dout, y8)
    dy = (dout.float() @ W.float()).to(dtype)
    dx, dg = norms.rms_norm_backward_int8(dy, h8, g, y.rstd)
    hk = i8.dequantize(h8, torch.float32).double()
    xh = hk * y.rstd.double()[:, None]
    u = dy.double() * g.double()
    ref_dx = y.rstd.double()[:, None] * (u - xh * (u * xh).mean(-1, keepdim=True))
    ref_dW = dout.double().t() @ i8.dequantize(y8, torch.float32).double()
    assert float((dW.double() - ref_dW).abs().max()) <= 2 * 364 * U * float((dout.double().abs().t() @ y.y.double().abs()).max())
    assert float((dx.double() - ref_dx).abs().max()) <= (HALF_ULP[dtype] + 100 * U) * float(ref_dx.abs().max()) * 1.01
    assert float((dg.double() - (dy.double() * xh).sum(0)).abs().max()) <= 702 * U * float((dy.double() * xh).abs().sum(0).max())
    # what keeping costs: half a step of the scale, at most max|h| / 127 of a group
    step = h8.scale.repeat_interleave(32, 1)[:, :D].double()
    assert bool(((hk - h.double()).abs() <= step / 2).all()) and bool((step * 63 < hk.abs().amax() + step).all())


# ---- streams, graphs, repeats

@pytest.mark.gpu
def test_streams_and_graphs(dev):
    """The calls on a side stream and in captured graphs, two of which replay in turn, give what they give eagerly."""
    from elara_amd import norms
    i8 = _i8()
    x = [torch.randn(300, 256, device=dev).bfloat16() for _ in range(2)]
    w = i8.quantize(torch.randn(130, 256, device=dev))
    dy = torch.randn(300, 130, device=dev).bfloat16()
    gain, rstd = torch.rand(256, device=dev), torch.rand(300, device=dev)

    def work(t):
        a = i8.quantize(t)
        k = i8.quantize(t, group=64, pow2=True)
        return [a.q, a.scale, i8.linear(a, w), i8.dequantize(k), i8.weight_grad(dy, k),
                *norms.rms_norm_backward_int8(t, k, gain, rstd)]
    eager = [work(t) for t in x]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work(x[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, eager[0]))
    ins, graphs, outs = [t.clone() for t in x], [], []
    for t in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(t))
        graphs.append(g)
    for turn in range(3):
        for i, g in enumerate(graphs):
            ins[i].copy_(x[(i + turn) % 2])
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i], eager[(i + turn) % 2])), (turn, i)
            work(x[0])


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """Calls in flight together share nothing, workspaces included."""
    i8 = _i8()
    dy = [torch.randn(6000, 96, device=dev) for _ in range(2)]
    k = [i8.quantize(torch.randn(6000, 200, device=dev), group=32, pow2=True) for _ in range(2)]
    w = i8.quantize(torch.randn(150, 200, device=dev))
    alone = [(i8.weight_grad(dy[i], k[i]), i8.linear(i8.quantize(dy[i].repeat(1, 3)[:, :200].contiguous()), w)) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((i8.weight_grad(dy[i], k[i]), i8.linear(i8.quantize(dy[i].repeat(1, 3)[:, :200].contiguous()), w)))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in got[i]:
            assert torch.equal(a, alone[i][0]) and torch.equal(b, alone[i][1])


@pytest.mark.gpu
def test_rows_of_one_dimension(dev):
    """One row without a leading dimension, through every call."""
    from elara_amd import norms
    i8 = _i8()
    x, dy = torch.randn(96, device=dev).bfloat16(), torch.randn(40, device=dev).bfloat16()
    r, w = i8.quantize(x, group=32, pow2=True), i8.quantize(torch.randn(40, 96, device=dev))
    y = i8.linear(i8.quantize(x), w)
    assert y.shape == (40,) and torch.equal(y, i8.linear(i8.quantize(x[None]), w)[0])
    dw = i8.weight_grad(dy, r)
    assert torch.equal(dw, i8.weight_grad(dy[None], i8.Int8Rows(r.q[None], r.scale[None], 32))) and dw.shape == (40, 96)
    g, rstd = torch.rand(96, device=dev), torch.tensor(0.7, device=dev)
    dx, dg = norms.rms_norm_backward_int8(x, r, g, rstd)
    two = norms.rms_norm_backward_int8(x[None], i8.Int8Rows(r.q[None], r.scale[None], 32), g, rstd[None])
    assert torch.equal(dx, two[0][0]) and torch.equal(dg, two[1])


@pytest.mark.gpu
def test_repeats_are_bitwise_equal(dev):
    i8 = _i8()
    q, s = ref_quantize(_randn(1, 6000, 128), 64, True)
    k = i8.Int8Rows(q.to(dev), s.to(dev), 64)
    dy = torch.randn(6000, 96, device=dev)
    first = i8.weight_grad(dy, k)
    for _ in range(5):
        assert torch.equal(i8.weight_grad(dy, k), first)


# ---- refusals

def test_refusals_of_the_c_entry_points():
    """Bad arguments come back as codes before any launch (no GPU needed)."""
    L = _lib.lib()
    p = ctypes.c_void_p(256)
    assert L.elr_quantize_int8(p, 0, -1, 8, 8, 0, 0, p, p, None) == -1
    assert L.elr_quantize_int8(p, 0, 1, 0, 8, 0, 0, p, p, None) == -1
    assert L.elr_quantize_int8(p, 9, 1, 8, 8, 0, 0, p, p, None) == -1
    assert L.elr_quantize_int8(p, 0, 1, 8, 8, 48, 0, p, p, None) == -2
    assert L.elr_quantize_int8(None, 0, 1, 8, 8, 0, 0, p, p, None) == -1
    assert L.elr_quantize_int8(ctypes.c_void_p(257), 0, 1, 8, 8, 0, 0, p, p, None) == -1
    assert L.elr_quantize_int8(None, 0, 0, 8, 8, 0, 0, None, None, None) == 0
    assert L.elr_dequantize_int8(p, 1, 8, 8, 7, p, p, 0, None) == -2
    assert L.elr_dequantize_int8(p, 1, 8, -1, 0, p, p, 0, None) == -1
    assert L.elr_dequantize_int8(p, 1, 8, 8, 0, None, p, 0, None) == -1
    assert L.elr_dequantize_int8(None, 0, 8, 8, 0, None, None, 0, None) == 0
    lin = lambda n, K, N, x=p, y=p, t=0: L.elr_int8_linear(x, n, K, K, p, p, N, K, p, y, t, None)  # noqa: E731
    assert lin(-1, 8, 8) == -1 and lin(1, -8, 8) == -1 and lin(1, 8, 8, t=3) == -1
    assert lin(1, 1 << 17, 8) == -2 and lin(1, 8, (1 << 30) + 1) == -2
    assert lin(1, 8, 8, x=None) == -1 and lin(1, 8, 8, y=None) == -1 and lin(1, 8, 8, y=ctypes.c_void_p(258)) == -1
    assert lin(0, 8, 8, x=None, y=None) == 0 and lin(1, 8, 0, y=None) == 0
    assert L.elr_int8_weight_grad_scratch_bytes(1, 1, 1, 7) == -1
    wg = lambda n, N, K, dw=p, group=0, t=2, sc=p, nb=1 << 40: L.elr_int8_weight_grad(  # noqa: E731
        p, t, n, N, N, p, K, K, group, p, dw, 0, sc, nb, None)
    assert wg(-1, 8, 8) == -1 and wg(1, 8, 8, t=5) == -1 and wg(1, 8, 8, group=16) == -2 and wg(1, 8, 8, dw=None) == -1
    assert wg(1, 0, 8, dw=None) == 0
    need = L.elr_int8_weight_grad_scratch_bytes(100_000, 64, 64, 2)
    assert need > 0 and wg(100_000, 64, 64, sc=None, nb=0) == -3 and wg(100_000, 64, 64, nb=need - 1) == -3
    nb = lambda n=1, D=8, group=0, xt=0, h=p, dw=None: L.elr_rms_norm_backward_int8(  # noqa: E731
        p, 0, n, D, D, h, D, group, p, None, xt, D, None, 0, p, p, dw, None, 0, None)
    assert nb(n=-1) == -1 and nb(group=3) == -2 and nb(xt=1) == -2 and nb(h=None) == -1 and nb(dw=p, n=5000) == -3
    assert nb(n=0) == 0


def test_refusals_of_cpu_tensors():
    from elara_amd import norms
    i8 = _i8()
    r = i8.Int8Rows(torch.zeros(2, 64, dtype=torch.int8), torch.ones(2, 1), 0)
    with pytest.raises(RuntimeError, match='cuda'):
        i8.quantize(torch.zeros(2, 64))
    with pytest.raises(RuntimeError, match='group must be'):
        i8.quantize(torch.zeros(2, 64), group=48)
    for call in (lambda: i8.dequantize(r), lambda: i8.linear(r, r), lambda: i8.weight_grad(torch.zeros(2, 4), r),
                 lambda: norms.rms_norm_backward_int8(torch.zeros(2, 64), r, None, torch.ones(2))):
        with pytest.raises(RuntimeError, match='cuda'):
            call()


@pytest.mark.gpu
def test_refusals(dev):
    from elara_amd import norms
    i8 = _i8()
    x = torch.randn(4, 64, device=dev)
    r = i8.quantize(x)
    g = i8.quantize(x, group=32)
    bad = [
        lambda: i8.quantize(x.double()), lambda: i8.quantize(x, group=16), lambda: i8.quantize(torch.tensor(1.0, device=dev)),
        lambda: i8.quantize(torch.zeros(3, 0, device=dev)),
        lambda: i8.dequantize(r, dtype=torch.float64), lambda: i8.dequantize(i8.Int8Rows(r.q, r.scale, 32)),
        lambda: i8.dequantize(i8.Int8Rows(r.q.int(), r.scale, 0)), lambda: i8.dequantize(i8.Int8Rows(r.q, r.scale.double(), 0)),
        lambda: i8.dequantize(i8.Int8Rows(r.q, r.scale.cpu(), 0)), lambda: i8.dequantize(i8.Int8Rows(r.q, r.scale, 5)),
        lambda: i8.linear(g, r), lambda: i8.linear(r, g), lambda: i8.linear(r, i8.quantize(x[:, :32].contiguous())),
        lambda: i8.linear(r, i8.quantize(x.view(2, 2, 64))), lambda: i8.linear(r, r, dtype=torch.int32),
        lambda: i8.linear(r, i8.Int8Rows(r.q, r.scale[:2], 0)),
        lambda: i8.weight_grad(x[:3], r), lambda: i8.weight_grad(x.double(), r), lambda: i8.weight_grad(x.view(2, 2, 64), r),
        lambda: i8.weight_grad(x, i8.Int8Rows(r.q, r.scale, 64).__class__(r.q.short(), r.scale, 0)),
        lambda: norms.rms_norm_backward_int8(x, i8.quantize(x[:, :32].contiguous()), None, torch.ones(4, device=dev)),
        lambda: norms.rms_norm_backward_int8(x, r, torch.ones(3, device=dev), torch.ones(4, device=dev)),
        lambda: norms.rms_norm_backward_int8(x, r, None, torch.ones(5, device=dev)),
        lambda: norms.rms_norm_backward_int8(x, r, None, torch.ones(4, device=dev), dh=x[:2]),
        lambda: norms.rms_norm_backward_int8(x, r, None, torch.ones(4, device=dev), dh=x.half()),
        lambda: norms.rms_norm_backward_int8(x.bfloat16(), r, None, torch.ones(4, device=dev), dh=x.half()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f'call {i} was taken')
    K = 1 << 17
    big = i8.Int8Rows(torch.zeros(1, K, dtype=torch.int8, device=dev), torch.ones(1, 1, device=dev), 0)
    with pytest.raises(RuntimeError, match='K must be at most'):
        i8.linear(big, big)
