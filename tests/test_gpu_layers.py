"""The dense layer and the layer norm (avatarcap_amd/network/layers.py) against plain float64 on the CPU: values and gradients, at the sizes, layouts and activations where a kernel can
go wrong.

Tolerances.  With u = half a step of the element type (finfo.eps / 2) an output v is off by at most u |v| from its own rounding.  What comes before it:
  * z is a sum of K products of exact inputs in float32: error <= (K + 2) 2^-24 sum|x||w|, and float32 inputs are carried as three bf16 whose dropped products are below
    2^-22 sum|x||w|; a bias adds one more rounding.  Zerr below.
  * activations are 1.1-Lipschitz (gelu and silu peak at 1.13, 1.10) and evaluated to 16 float32 steps of max(|z|, 1).
  * gradients: act' is taken at z rounded to the element type (error u |z| times |act''| <= 1, piecewise linear ones exact off their kink), dz is rounded once to the element type, and
    the products sum it over N (dx), M (dw, db): D = (2 u |dy| (|z| + 1)) per element, propagated by sum D |w| and sum D |x|, plus the float32 sums.
Every bound is evaluated elementwise from the actual magnitudes."""
import math

import pytest
import torch

from avatarcap_amd import _lib
from avatarcap_amd.network.layers import ACTS, layer_norm, linear

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
E32 = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def act64(z, act, slope):
    """(act(z), act'(z)) in float64."""
    if act is None:
        return z, torch.ones_like(z)
    if act == 'relu':
        return z.clamp(min=0), (z > 0).double()
    if act == 'leaky_relu':
        return torch.where(z > 0, z, slope * z), torch.where(z > 0, 1.0, slope).double()
    if act == 'soft_plus':
        return torch.where(z > 20, z, torch.log1p(torch.exp(z.clamp(max=20)))), torch.where(z > 20, torch.ones_like(z), torch.sigmoid(z))
    if act == 'sigmoid':
        s = torch.sigmoid(z)
        return s, s * torch.sigmoid(-z)
    if act == 'tanh':
        return torch.tanh(z), torch.cosh(z) ** -2
    if act == 'gelu':
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return z * s, s + z * s * (1 - s)


def make(m, k, n, dtype, layout='rows', bias=True, residual=False, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + m * 31 + k * 17 + n)
    rn = lambda *s: torch.randn(*s, generator=g)                                           # noqa: E731
    x = rn(m, k).to(dtype)
    if layout == 'channels':
        xd = x.t().contiguous().cuda().t()
    elif layout == 'padded':
        buf = torch.full((m, k + 5), float('nan'), dtype=dtype, device='cuda')
        buf[:, 2:2 + k] = x.cuda()
        xd = buf[:, 2:2 + k]
    elif layout == 'strided':
        buf = torch.full((m, 2 * k), float('nan'), dtype=dtype, device='cuda')
        buf[:, ::2] = x.cuda()
        xd = buf[:, ::2]
    else:
        xd = x.cuda()
    w = (rn(n, k) / math.sqrt(k)).to(dtype)
    b = (0.5 * rn(n)).to(dtype) if bias else None
    r = rn(m, n).to(dtype) if residual else None
    dy = rn(m, n).to(dtype)
    return xd, x, w, b, r, dy


def dev(t):
    return None if t is None else t.cuda()


def dbl(t):
    return None if t is None else t.detach().cpu().double()


def close(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), f'{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() - tol).max()):.3g} beyond its bound'


def check_linear(m, k, n, dtype, act=None, layout='rows', bias=True, residual=False, slope=0.02, grad=True, seed=0):
    xd, x, w, b, r, dy = make(m, k, n, dtype, layout, bias, residual, seed)
    u = unit(dtype)
    X, W, B, R, DY = dbl(x), dbl(w), dbl(b), dbl(r), dbl(dy)
    mag = X.abs() @ W.abs().t() + (0 if B is None else B.abs())
    z = X @ W.t() + (0 if B is None else B)
    zerr = ((k + 2) * E32 + 2.0 ** -22) * mag
    v, sl = act64(z, act, slope)
    y = v if R is None else v + R
    ytol = u * y.abs() + 1.2 * zerr + 16 * E32 * (z.abs().clamp(min=1) + (0 if R is None else R.abs())) * 1.01 + torch.finfo(dtype).tiny
    leaves = [xd, dev(w), dev(b), dev(r)]
    if not grad:
        got = linear(leaves[0], leaves[1], leaves[2], act=act, slope=slope, residual=leaves[3])
        close(got, y, ytol, 'y')
        return
    for t in leaves:
        if t is not None:
            t.requires_grad_()
    got = linear(leaves[0], leaves[1], leaves[2], act=act, slope=slope, residual=leaves[3])
    close(got, y, ytol, 'y')
    got.backward(dy.cuda())
    dz = DY * sl
    kink = (act in ('relu', 'leaky_relu')) * (z.abs() <= zerr + u * z.abs() + torch.finfo(dtype).tiny).double()    # the slope may be taken on the other side
    d = DY.abs() * ((2 * u * (z.abs() + 1) + zerr + 16 * E32) * (act is not None) + kink)
    gtol = lambda true, err, terms, mg: u * true.abs() + (1 + 2 * u) * err + ((terms + 2) * E32 + 2.0 ** -22) * mg + torch.finfo(dtype).tiny   # noqa: E731
    adz = dz.abs() + d
    dx = dz @ W
    close(leaves[0].grad, dx, gtol(dx, d @ W.abs(), n, adz @ W.abs()), 'dx')
    dw = dz.t() @ X
    close(leaves[1].grad, dw, gtol(dw, d.t() @ X.abs(), m, adz.t() @ X.abs()), 'dw')
    if b is not None:
        db = dz.sum(0)
        close(leaves[2].grad, db, gtol(db, d.sum(0), m, adz.sum(0)), 'db')
    if r is not None:
        assert torch.equal(leaves[3].grad.cpu(), dy)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('m,k,n', [(1, 1, 1), (1, 7, 3), (2, 64, 1), (1, 1024, 48), (17, 33, 65), (33, 545, 16), (33, 63, 17), (64, 64, 64), (65, 128, 129), (129, 100, 257), (300, 319, 256),
                                   (257, 512, 130), (1000, 8, 8)])
def test_sizes(m, k, n, dtype):
    check_linear(m, k, n, dtype, act='soft_plus')


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('act', [a for a in ACTS])
def test_activations_with_bias_and_residual(act, dtype):
    check_linear(70, 96, 136, dtype, act=act, residual=True)
    check_linear(70, 96, 136, dtype, act=act, bias=False)
    check_linear(5, 200, 24, dtype, act=act, residual=True)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('layout', ['padded', 'channels', 'strided'])
@pytest.mark.parametrize('m,k,n', [(1, 40, 9), (19, 40, 72), (130, 72, 3), (130, 72, 1), (257, 129, 4), (515, 256, 128), (258, 301, 31)])
def test_layouts(m, k, n, layout, dtype):
    check_linear(m, k, n, dtype, act='tanh', layout=layout, residual=True)


@pytest.mark.parametrize('dtype', DTYPES)
def test_large_tiles_and_splits(dtype):
    check_linear(2048, 768, 2048, dtype, act='gelu', grad=False)             # the largest tile, k past one step, several per XCD
    check_linear(2000, 776, 2072, dtype, act='relu', residual=True, grad=False, layout='channels')
    check_linear(40, 4096, 72, dtype, act='silu')                            # few tiles, a long sum: split
    check_linear(5000, 40, 24, dtype, act='leaky_relu')                      # the weight gradient splits over the rows
    check_linear(2050, 2050, 640, dtype, act='silu', grad=True)


def check_norm(m, c, dtype, affine=True, eps=1e-5, scale=1.5, shift=0.25, pad=0, grad=True):
    """Bounds: the row's sums are float32 over C values: mean to (C 2^-24) max|x| =: em, and with s = 1 / std, x^ = (x - mean) s to e = s em + 8 2^-24 (|x^| + 1) + (C + 8) 2^-24 |x^|
    (the variance's own relative error, halved by the root, is below (C + 4) 2^-24 plus (em s)^2).  Gradients are sums of products of x^, dy and g over the row or the columns."""
    gen = torch.Generator().manual_seed(m * 131 + c)
    x = (torch.randn(m, c, generator=gen) * scale + shift).to(dtype)
    g = (1 + 0.2 * torch.randn(c, generator=gen)).to(dtype) if affine else None
    b = (0.1 * torch.randn(c, generator=gen)).to(dtype) if affine else None
    dy = torch.randn(m, c, generator=gen).to(dtype)
    buf = torch.full((m, c + pad), float('nan'), dtype=dtype, device='cuda')
    buf[:, pad // 2:pad // 2 + c] = x.cuda()
    xd, gd, bd = buf[:, pad // 2:pad // 2 + c].detach(), dev(g), dev(b)
    if grad:
        for t in (xd, gd, bd):
            if t is not None:
                t.requires_grad_()
    X, DY, u = dbl(x), dbl(dy), unit(dtype)
    G = torch.ones(c, dtype=torch.float64) if g is None else dbl(g)
    B = torch.zeros(c, dtype=torch.float64) if b is None else dbl(b)
    mean = X.mean(1, keepdim=True)
    std = ((X - mean).pow(2).mean(1, keepdim=True) + eps).sqrt()
    xh = (X - mean) / std
    em = (c + 2) * E32 * X.abs().amax(1, keepdim=True)
    e = em / std + (c + 16) * E32 * (xh.abs() + 1) + (em / std) ** 2 * xh.abs()
    y = xh * G + B
    tiny = torch.finfo(dtype).tiny
    got = layer_norm(xd, gd, bd, eps=eps)
    close(got, y, u * y.abs() + (1 + u) * (e * G.abs() + 4 * E32 * (xh * G).abs() + 2 * E32 * B.abs()) + tiny, 'y')
    if not grad:
        return
    got.backward(dy.cuda())
    t = DY * G
    dx = (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True)) / std
    s1 = t.abs().mean(1, keepdim=True)
    s2 = (t.abs() * (xh.abs() + e)).mean(1, keepdim=True)
    err = ((c + 16) * E32 * (t.abs() + s1 + xh.abs() * s2) + e * s2 + xh.abs() * (t.abs() * e).mean(1, keepdim=True)) / std
    rel = (c + 8) * E32 + (em / std) ** 2
    close(xd.grad, dx, u * dx.abs() + (1 + u) * (err + rel * dx.abs()) + tiny, 'dx')
    if affine:
        dg, db = (DY * xh).sum(0), DY.sum(0)
        close(gd.grad, dg, u * dg.abs() + (1 + u) * ((DY.abs() * e).sum(0) + (m + 4) * E32 * (DY * xh).abs().sum(0)) + tiny, 'dg')
        close(bd.grad, db, u * db.abs() + (1 + u) * (m + 2) * E32 * DY.abs().sum(0) + tiny, 'db')


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('m,c', [(1, 1), (3, 2), (5, 3), (1, 7), (70, 8), (1, 9), (33, 31), (257, 64), (1, 256), (9000, 256), (9001, 70), (8193, 777), (66, 1023), (3, 1024), (40, 2049), (17, 4097),
                                 (5, 8191), (3, 8193), (2, 16384), (3, 16385), (21, 20000)])
def test_norm_sizes(m, c, dtype):
    check_norm(m, c, dtype)


@pytest.mark.parametrize('dtype', DTYPES)
def test_norm_layouts_and_values(dtype):
    check_norm(37, 100, dtype, affine=False)
    check_norm(37, 101, dtype, pad=6)
    check_norm(300, 16500, dtype, pad=3, grad=False)
    check_norm(1200, 260, dtype, scale=0.01, shift=4.0 if dtype == torch.float32 else 0.02)
    check_norm(7, 512, dtype, scale=100.0, shift=-50.0, eps=1.0)


# ---- values that a kernel must not lose ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('m,k,n', [(3, 40, 33), (70, 40, 33), (70, 100, 140), (300, 264, 300)])
def test_a_nan_or_infinity_reaches_its_own_row_only(m, k, n, dtype):
    xd, x, w, b, r, dy = make(m, k, n, dtype)
    for bad in (float('nan'), float('inf'), -float('inf')):
        x2 = x.clone()
        x2[m // 2, k - 1] = bad
        y = linear(x2.cuda(), dev(w), dev(b)).cpu()
        clean = linear(xd, dev(w), dev(b)).cpu()
        keep = torch.arange(m) != m // 2
        assert torch.equal(y[keep], clean[keep])
        assert not bool(torch.isfinite(y[m // 2]).any())
        if bad == bad:                                                       # w is nowhere zero: every output of the row is infinite, with the sign of the product
            want = torch.sign(w[:, k - 1].double()) * bad
            assert torch.equal(y[m // 2].double(), want)
        w2 = w.clone()
        w2[n - 1, 0] = bad
        y = linear(xd, dev(w2), dev(b)).cpu()
        assert torch.equal(y[:, :n - 1], clean[:, :n - 1]) and not bool(torch.isfinite(y[:, n - 1]).any())


def test_float32_keeps_its_range():
    """float32 goes through three bf16: the largest values, the smallest normal ones and sums that cancel.  In the last, w = 1 has a head alone, so the three non-zero x meet it as
    9 exact products; the order of a sum is not fixed, and each of at most 9 additions is off by half a step of a partial sum below 2.01 |a|: 9 2^-24 2.01 |a|."""
    g = torch.Generator().manual_seed(5)
    for m, k, n in ((70, 64, 70), (300, 64, 300)):
        x = torch.zeros(m, k)
        x[:, 0] = 3.4e38 * torch.sign(torch.randn(m, generator=g))
        x[:, 1] = 1.2e-38 * torch.rand(m, generator=g) * 3 + 1.2e-38
        w = torch.zeros(n, k)
        w[:, 0] = 0.5
        y = linear(x.cuda(), w.cuda()).cpu()
        assert torch.equal(y, (x[:, :1] * 0.5).expand(m, n))
        w[:, 0], w[:, 1] = 0.0, 1.0
        y = linear(x.cuda(), w.cuda()).cpu().double()
        assert bool(((y - x[:, 1:2].double()).abs() <= 2.0 ** -126).all())   # the planes' tails are below the smallest normal and may be flushed
        a = torch.randn(m, generator=g)
        x = torch.zeros(m, k)
        x[:, 0], x[:, 1], x[:, 2] = a, -a, 2.0 ** -20 * a
        y = linear(x.cuda(), torch.ones(n, k).cuda()).cpu()
        assert bool(((y.double() - x[:, 2:3].double()).abs() <= 9 * E32 * 2.01 * a.abs().double()[:, None]).all())


@pytest.mark.parametrize('act', [a for a in ACTS])
def test_activations_at_extreme_values(act):
    """z itself is exact here (one product by 1): the activation and its slope over the range, against float64; both are bounded to 16 steps of float32 of max(|value|, 1e-30) plus
    what half a step of z is worth, |z| <= 20 -> relative 2^-24 |z| of e^z.  An e^z below float32's smallest normal value 2^-126 may be zero, and silu and gelu multiply it by
    |z|: `least`."""
    z = torch.cat([torch.linspace(-30, 30, 4001), torch.tensor([0.0, -0.0, 1e-20, -1e-20, 1e-6, -1e-6, 20.0, 20.0001, 88.0, -88.0, 100.0, -100.0, 1e4, -1e4])])[:, None]
    one = torch.ones(1, 1)
    x, w = z.cuda().requires_grad_(), one.cuda()
    y = linear(x, w, act=act)
    y.backward(torch.ones_like(y))
    v, s = act64(z.double(), act, 0.02)
    rel = (16 + 3 * z.abs().double()) * E32
    least = 1e-37 + 2.0 ** -126 * z.abs().double()
    close(y, v, rel * v.abs() + least, act)
    if act == 'gelu':                                                        # Phi + z phi cancels near its zero: the terms' size counts
        cdf = 0.5 * torch.erfc(-z.double() / math.sqrt(2))
        size = cdf + (z.double().abs() * torch.exp(-z.double() ** 2 / 2) / math.sqrt(2 * math.pi))
    elif act == 'silu':
        size = torch.sigmoid(z.double()) * (1 + z.double().abs() * torch.sigmoid(-z.double()))
    else:
        size = s.abs()
    # float32's smallest normal: a slope below it may be zero.  gelu's e^(-z^2 / 2) carries z^2 / 2 steps
    size = size * (1 + (z.double() ** 2 / 8 if act == 'gelu' else 0))
    if act in ('relu', 'leaky_relu'):
        keep = z != 0
        assert torch.equal(x.grad.cpu()[keep], s.float()[keep])
    else:
        close(x.grad, s, rel * size + least, f"{act}'")
    inf = torch.tensor([[float('inf')], [float('nan')]]).cuda()
    got = linear(inf, w, act=act).cpu()
    assert float(got[0, 0]) == (1.0 if act in ('sigmoid', 'tanh') else float('inf')) and bool(torch.isnan(got[1, 0]))


def test_a_row_of_equal_values_has_a_finite_norm():
    for dtype in DTYPES:
        x = torch.full((5, 96), 3.0, dtype=dtype, device='cuda', requires_grad=True)
        y = layer_norm(x)
        assert bool((y == 0).all())
        y.backward(torch.randn(5, 96, device='cuda').to(dtype))
        assert bool(torch.isfinite(x.grad).all())
        bad = torch.randn(4, 96, device='cuda').to(dtype)
        good = layer_norm(bad.clone())
        bad[1, 7], bad[2, 95] = float('nan'), float('inf')
        y = layer_norm(bad)
        assert bool(torch.isnan(y[1:3]).all()) and torch.equal(y[0], good[0]) and torch.equal(y[3], good[3])


# ---- gradients against differences --------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('act', ['soft_plus', 'tanh', 'gelu', 'silu', 'sigmoid'])
def test_gradients_are_the_slope_of_the_forward_pass(act):
    """(f(v + h d) - f(v - h d)) / 2h along random directions, f the sum of y times fixed numbers in float64: truncation ~ h^2, rounding ~ 2^-24 |f terms| / h."""
    g = torch.Generator().manual_seed(3)
    x, w, b, r = (torch.randn(*s, generator=g).cuda().requires_grad_() for s in ((33, 20), (17, 20), (17,), (33, 17)))
    c = torch.randn(33, 17, generator=g).cuda()
    f = lambda *a: float((linear(a[0], a[1], a[2], act=act, residual=a[3]).double() * c.double()).sum())   # noqa: E731
    grads = torch.autograd.grad(linear(x, w, b, act=act, residual=r), (x, w, b, r), c)
    h = 2.0 ** -8
    with torch.no_grad():
        for i in range(4):
            d = torch.randn(grads[i].shape, generator=g).cuda()
            p, m = [x, w, b, r], [x, w, b, r]
            p[i], m[i] = p[i] + h * d, m[i] - h * d
            slope = (f(*p) - f(*m)) / (2 * h)
            want = float((grads[i].double() * d.double()).sum())
            scale = float((grads[i].double().abs() * d.double().abs()).sum())
            assert abs(slope - want) < 3e-3 * scale, (act, i, slope, want)
    x, gm, bt = (torch.randn(*s, generator=g).cuda().requires_grad_() for s in ((9, 40), (40,), (40,)))
    c = torch.randn(9, 40, generator=g).cuda()
    grads = torch.autograd.grad(layer_norm(x, gm, bt), (x, gm, bt), c)
    with torch.no_grad():
        for i in range(3):
            d = torch.randn(grads[i].shape, generator=g).cuda()
            p, m = [x, gm, bt], [x, gm, bt]
            p[i], m[i] = p[i] + h * d, m[i] - h * d
            slope = float(((layer_norm(*p).double() - layer_norm(*m).double()) * c.double()).sum()) / (2 * h)
            want = float((grads[i].double() * d.double()).sum())
            assert abs(slope - want) < 3e-3 * float((grads[i].double().abs() * d.double().abs()).sum()), (i, slope, want)


# ---- how a program uses them ------------------------------------------------------------------------------------------------------------------------------------
def test_shapes_views_and_partial_gradients():
    g = torch.Generator().manual_seed(11)
    x = torch.randn(2, 5, 7, 24, generator=g).cuda()
    w, b = torch.randn(9, 24, 1, generator=g).cuda(), torch.randn(9, generator=g).cuda()
    y = linear(x, w, b, act='relu')
    assert y.shape == (2, 5, 7, 9) and torch.equal(y.reshape(-1, 9), linear(x.reshape(-1, 24), w[:, :, 0], b, act='relu'))
    assert linear(x[0, 0, 0, :], w, b).shape == (9,)
    assert linear(x[:0], w, b).shape == (0, 5, 7, 9) and layer_norm(x[:0]).shape == (0, 5, 7, 24)
    for which in range(4):                                                  # one leaf at a time, the rest constants
        t = [x.reshape(-1, 24).clone(), w[:, :, 0].clone(), b.clone(), torch.randn(70, 9, generator=g).cuda()]
        full = [v.clone().requires_grad_() for v in t]
        one = [v.requires_grad_() if i == which else v for i, v in enumerate(t)]
        c = torch.randn(70, 9, generator=g).cuda()
        for a in (full, one):
            linear(a[0], a[1], a[2], act='silu', residual=a[3]).backward(c)
        assert torch.equal(full[which].grad, one[which].grad)
    # gradients that come as expanded or transposed tensors, and a zero-row batch
    xg = torch.randn(33, 24, generator=g).cuda().requires_grad_()
    wg = w[:, :, 0].clone().requires_grad_()
    linear(xg, wg).sum().backward()
    ref = torch.ones(33, 9, dtype=torch.float64)
    close(xg.grad, ref @ wg.detach().cpu().double(), 1e-5, 'dx of a sum')
    z = torch.zeros(0, 24, device='cuda', requires_grad=True)
    wg.grad = None
    bg = b.clone().requires_grad_()
    linear(z, wg, bg, act='gelu').sum().backward()
    assert z.grad.shape == (0, 24) and not bool(wg.grad.any()) and not bool(bg.grad.any())
    gm = torch.ones(24, device='cuda', requires_grad=True)
    layer_norm(z, gm).sum().backward()
    assert not bool(gm.grad.any())
    with pytest.raises(RuntimeError):                                       # no gradient of a gradient
        q = torch.randn(4, 24, device='cuda', requires_grad=True)
        (d,) = torch.autograd.grad(linear(q, wg, act='tanh').sum(), q, create_graph=True)
        d.sum().backward()


@pytest.mark.parametrize('act', ['soft_plus', 'sigmoid', 'tanh', 'gelu', 'silu'])
@pytest.mark.parametrize('m,k,n', [(300, 192, 256), (40, 72, 48), (2100, 264, 300), (5, 520, 200)])
def test_bf16_gradients_carry_two_roundings_and_no_third(m, k, n, act):
    """Root mean square errors: dx rounded once has e; dz rounded as well, sqrt(2) e = 1.41 e.  The kept z has 11 bits, 1/8 of a bf16 step: |act''| z / act' times that, squared, is below
    (2 / 8)^2 = 0.06 of one rounding's square where it counts, sqrt(2.06) = 1.44.  A z of 8 bits gives up to 1.55.  With 960 values the ratio of two such means spreads by 5 %."""
    g = torch.Generator().manual_seed(m + k)
    x, w, b, dy = (torch.randn(*s, generator=g).mul(f).bfloat16() for s, f in (((m, k), 1), ((n, k), k ** -0.5), ((n,), 0.1), ((m, n), 1)))
    leaf = dev(x).requires_grad_()
    (dx,) = torch.autograd.grad(linear(leaf, dev(w), dev(b), act=act), leaf, dev(dy))
    exact = (dy.double() * act64(x.double() @ w.double().t() + b.double(), act, 0.02)[1]) @ w.double()
    err, once = ((t.double().cpu() - exact).square().mean().sqrt().item() for t in (dx, exact.bfloat16()))
    assert err < 1.44 * (1.05 if m * k < 10000 else 1.01) * once, (err, once)


@pytest.mark.parametrize('what', ['linear', 'bias only', 'layer_norm'])
@pytest.mark.parametrize('graph_in_dy', [False, True])
def test_a_derivative_of_the_gradients_raises_and_leaves_nothing_out(what, graph_in_dy):
    q = torch.randn(4, 24, device='cuda', requires_grad=what != 'bias only')
    b = torch.randn(24, device='cuda', requires_grad=True)
    w = torch.randn(24, 24, device='cuda')
    y = layer_norm(q, b) if what == 'layer_norm' else linear(q, w, b, act='tanh', residual=q)
    dy = torch.ones(4, 24, device='cuda', requires_grad=graph_in_dy)
    leaf = b if what == 'bias only' else q
    (plain,) = torch.autograd.grad(y, leaf, dy.detach(), retain_graph=True)
    (d,) = torch.autograd.grad(y, leaf, dy, create_graph=True)
    assert torch.equal(d.detach(), plain)
    with pytest.raises(RuntimeError, match='no derivative'):
        (d.sum() + y.sum()).backward()                                      # y's own part would go through: the sum must not


@pytest.mark.parametrize('dtype', DTYPES)
def test_the_same_bits_every_time_and_on_another_stream(dtype):
    xd, x, w, b, r, dy = make(3000, 264, 200, dtype, residual=True)

    def run():
        leaves = [t.detach().clone().requires_grad_() for t in (xd, dev(w), dev(b))]
        y = linear(leaves[0], leaves[1], leaves[2], act='gelu', residual=dev(r))
        h = layer_norm(y, torch.ones(200, dtype=dtype, device='cuda', requires_grad=True))
        return (y, h) + torch.autograd.grad(h, leaves, dy.cuda())
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    third = run()
    torch.cuda.synchronize()
    for a, c, d in zip(first, second, third):
        assert torch.equal(a, c) and torch.equal(a, d)


def test_captured_graphs_replay_with_new_inputs():
    """Two graphs of a training step, captured one after the other, replayed in turn with eager work between: each keeps its own workspace."""
    def step(x, w, b, dy):
        y = linear(x, w, b, act='silu')
        h = layer_norm(y)
        return (h,) + torch.autograd.grad(h, (x, w, b), dy)
    graphs = []
    for m, k, n in ((1500, 136, 72), (40, 33, 65)):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            static = [torch.randn(m, k, device='cuda').requires_grad_(), torch.randn(n, k, device='cuda').requires_grad_(), torch.randn(n, device='cuda').requires_grad_(),
                      torch.randn(m, n, device='cuda')]
            for _ in range(2):
                step(*static)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs = step(*static)
        graphs.append((g, static, outs, (m, k, n)))
    for turn in range(3):
        for g, static, outs, (m, k, n) in graphs:
            with torch.no_grad():
                for t in static:
                    t.copy_(torch.randn(t.shape, device='cuda'))
            g.replay()
            torch.cuda.synchronize()
            fresh = [t.detach().clone().requires_grad_() for t in static[:3]]
            for a, c in zip(outs, step(*fresh, static[3])):
                assert torch.equal(a, c)
            torch.cuda.synchronize()


def test_a_residual_block_as_it_is_used():
    """x + W2 gelu(W1 norm(x) + b1) + b2 and its gradients, float32, against float64; relative to the largest value of each output 2e-5 (sums of 200 .. 900 float32 products)."""
    g = torch.Generator().manual_seed(17)
    t = [torch.randn(*s, generator=g) * f for s, f in (((900, 200), 1.0), ((200,), 0.3), ((200,), 0.1), ((560, 200), 200 ** -0.5), ((560,), 0.1), ((200, 560), 560 ** -0.5), ((200,), 0.1))]
    dy = torch.randn(900, 200, generator=g)

    def block(x, gm, bt, w1, b1, w2, b2, norm, lin):
        return lin(lin(norm(x, gm, bt), w1, b1, 'gelu', None), w2, b2, None, x)
    a = [v.cuda().requires_grad_() for v in t]
    y = block(*a, norm=lambda x, gm, bt: layer_norm(x, gm, bt), lin=lambda x, w, b, act, r: linear(x, w, b, act=act, residual=r))
    y.backward(dy.cuda())
    d = [v.double().requires_grad_() for v in t]

    def lin64(x, w, b, act, r):
        z = x @ w.t() + b
        z = z * 0.5 * torch.erfc(-z / math.sqrt(2)) if act else z
        return z if r is None else z + r
    ref = block(*d, norm=lambda x, gm, bt: torch.nn.functional.layer_norm(x, (200,), gm, bt), lin=lin64)
    ref.backward(dy.double())
    for got, want in [(y, ref)] + [(p.grad, q.grad) for p, q in zip(a, d)]:
        close(got, want.detach(), 2e-5 * float(want.detach().abs().max()), 'block')


@pytest.mark.parametrize('name', ['shared', 'geo', 'clr', 'recon'])
def test_mlp_forward_is_the_network_s_own_stack(name):
    """MLP.forward (any widths, layer by layer on linear) for the four stacks of the networks, with gradients, against the same stack of torch layers in float64 on the CPU."""
    import golden_inputs as gi
    from common import mlp_sd
    from avatarcap_amd.network.mlp import MLP
    kw = gi.MLP_CONFIGS[name]['kwargs']
    net = MLP(**kw)
    net.load_state_dict({k: torch.from_numpy(v) for k, v in mlp_sd(name).items()})
    ref = MLP(**kw).double()
    ref.load_state_dict({k: torch.from_numpy(v).double() for k, v in mlp_sd(name).items()})
    net = net.cuda()
    for B, N in ((1, 300), (2, 77), (1, 1)):
        x = torch.randn(B, kw['in_channels'], N, generator=torch.Generator().manual_seed(B * 10 + N))
        xd, xr = x.cuda().requires_grad_(), x.double().requires_grad_()
        y = net(xd)
        h = xr
        last = len(ref.fc_list) - 1
        for l, fc in enumerate(ref.fc_list):
            conv = fc if l == last else fc[0]
            if l in ref.res_layers:
                h = torch.cat([h, xr], 1)
            w = ref._weight(conv)
            h = torch.einsum('oc,bcn->bon', w, h) + conv.bias[None, :, None]
            act = ref.last_op if l == last else ref.nlactv
            h = act64(h, act, 0.02)[0] if act not in ('relu', 'leaky_relu') else torch.where(h > 0, h, (0.02 if act == 'leaky_relu' else 0.0) * h)
        assert y.shape == h.shape == (B, kw['out_channels'], N)
        scale = float(h.detach().abs().max())
        close(y, h.detach(), 2e-5 * max(scale, 1e-3), name)
        c = torch.randn(h.shape, generator=torch.Generator().manual_seed(1))
        net.zero_grad()
        ref.zero_grad()
        y.backward(c.cuda())
        h.backward(c.double())
        pairs = [(xd.grad, xr.grad)] + [(p.grad, dict(ref.named_parameters())[k].grad) for k, p in net.named_parameters()]
        for got, want in pairs:
            close(got, want, 1e-4 * float(want.abs().max()) + 1e-12, name)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('m,k,n', [(1, 3, 2), (17, 33, 65), (70, 9, 5), (130, 70, 131), (300, 520, 7)])
def test_nothing_outside_of_the_outputs_is_written(m, k, n, dtype):
    """The C entries on buffers between margins: inputs framed by NaNs, outputs by a pattern; row strides larger than the rows."""
    L, ctx = _lib.lib(), _lib.ctx(0)
    e = torch.finfo(dtype).bits // 8

    class Box:
        def __init__(self, rows, cols, fill=None, pad=3):
            self.rows, self.cols, self.ld = rows, cols, cols + pad
            self.raw = torch.full((1024 + rows * self.ld + 1024,), float('nan'), dtype=dtype, device='cuda')
            self.v = self.raw[1024:1024 + rows * self.ld].view(rows, self.ld)[:, :cols]
            if fill is not None:
                self.v.copy_(fill)
            self.ptr = self.raw.data_ptr() + 1024 * e

        def outside_untouched(self):
            mask = torch.ones_like(self.raw, dtype=torch.bool)
            mask[1024:1024 + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols] = False
            return bool(torch.isnan(self.raw[mask]).all()) and bool(torch.isfinite(self.v).all())
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    import ctypes as C
    gen = torch.Generator().manual_seed(m + k + n)
    x, w, b, r, dy = (Box(*s, fill=torch.randn(*s, generator=gen).to(dtype).cuda()) for s in ((m, k), (n, k), (1, n), (m, n), (m, n)))
    y, z = Box(m, n), Box(m, n)
    nb = C.c_int64()
    _lib.check(L.avc_linear_workspace(m, n, k, code, x.ld, 1, C.byref(nb)))
    ws = torch.empty(max(1, nb.value), dtype=torch.uint8, device='cuda')
    _lib.check(L.avc_linear(ctx, x.ptr, x.ld, 1, w.ptr, w.ld, b.ptr, r.ptr, r.ld, 6, 0.0, m, n, k, code, y.ptr, y.ld, z.ptr, z.ld, ws.data_ptr(), nb.value, None))
    torch.cuda.synchronize()
    assert all(t.outside_untouched() for t in (x, w, b, r, y, z))
    dx, dw, db = Box(m, k, pad=0), Box(n, k, pad=0), Box(1, n, pad=0)
    _lib.check(L.avc_linear_backward_workspace(m, n, k, code, C.byref(nb)))
    ws = torch.empty(max(1, nb.value), dtype=torch.uint8, device='cuda')
    _lib.check(L.avc_linear_backward(ctx, dy.ptr, dy.ld, x.ptr, x.ld, 1, w.ptr, w.ld, z.ptr, z.ld, 6, 0.0, m, n, k, code, dx.ptr, dw.ptr, db.ptr, ws.data_ptr(), nb.value, None))
    torch.cuda.synchronize()
    assert all(t.outside_untouched() for t in (dx, dw, db))
    y2, dx2, dg, dbt = Box(m, k), Box(m, k), Box(1, k), Box(1, k)
    gm, dyk = Box(1, k, fill=torch.randn(1, k, generator=gen).to(dtype).cuda()), Box(m, k, fill=torch.randn(m, k, generator=gen).to(dtype).cuda())
    st = torch.empty(2, m, device='cuda')
    _lib.check(L.avc_layer_norm(ctx, x.ptr, x.ld, gm.ptr, None, 1e-5, m, k, code, y2.ptr, y2.ld, st[0].data_ptr(), st[1].data_ptr(), None))
    _lib.check(L.avc_layer_norm_backward_workspace(m, k, code, C.byref(nb)))
    ws = torch.empty(max(1, nb.value), dtype=torch.uint8, device='cuda')
    _lib.check(L.avc_layer_norm_backward(ctx, dyk.ptr, dyk.ld, x.ptr, x.ld, gm.ptr, st[0].data_ptr(), st[1].data_ptr(), m, k, code, dx2.ptr, dx2.ld, dg.ptr, dbt.ptr, ws.data_ptr(), nb.value, None))
    torch.cuda.synchronize()
    assert all(t.outside_untouched() for t in (y2, dx2, dg, dbt))


def test_in_place_outputs():
    """y may be res itself (linear) or x itself (layer_norm) at the C entries."""
    L, ctx = _lib.lib(), _lib.ctx(0)
    g = torch.Generator().manual_seed(2)
    for m, k, n in ((5, 40, 24), (300, 72, 136), (40, 4096, 64)):
        x, w, r = (torch.randn(*s, generator=g).cuda() for s in ((m, k), (n, k), (m, n)))
        want = linear(x, w, act='tanh', residual=r)
        import ctypes as C
        nb = C.c_int64()
        _lib.check(L.avc_linear_workspace(m, n, k, 0, k, 1, C.byref(nb)))
        ws = torch.empty(max(1, nb.value), dtype=torch.uint8, device='cuda')
        _lib.check(L.avc_linear(ctx, x.data_ptr(), k, 1, w.data_ptr(), k, None, r.data_ptr(), n, 5, 0.0, m, n, k, 0, r.data_ptr(), n, None, 0, ws.data_ptr(), nb.value, None))
        torch.cuda.synchronize()
        assert torch.equal(r, want)
    for m, c in ((7, 5), (33, 100), (9, 1023), (5, 9001), (3, 20001)):
        x = torch.randn(m, c, generator=g).cuda()
        want = layer_norm(x)
        _lib.check(L.avc_layer_norm(ctx, x.data_ptr(), c, None, None, 1e-5, m, c, 0, x.data_ptr(), c, None, None, None))
        torch.cuda.synchronize()
        assert torch.equal(x, want)


def test_the_current_device_stays_and_refusals_on_the_device():
    x, w = torch.randn(4, 8, device='cuda'), torch.randn(3, 8, device='cuda')
    before = torch.cuda.current_device()
    linear(x, w)
    assert torch.cuda.current_device() == before
    with pytest.raises(TypeError):
        linear(x, w.half())
    with pytest.raises(TypeError):
        linear(x.double(), w.double())
    with pytest.raises(ValueError):
        linear(x, w[:, :5])
    with pytest.raises(ValueError):
        linear(x, w, torch.randn(4, device='cuda'))
    with pytest.raises(ValueError):
        linear(x, w, residual=torch.randn(4, 4, device='cuda'))
    with pytest.raises(ValueError):
        linear(x, w, act='swish')
    with pytest.raises(ValueError):
        linear(x, w, act='leaky_relu', slope=-0.1)
    with pytest.raises(RuntimeError):
        linear(x, w.cpu())
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(7, device='cuda'))
    with pytest.raises(ValueError):
        layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError):
        layer_norm(x[:, :0])


def test_offsets_past_32_bits():
    """Matrices of more than 2^32 bytes and 2^31 elements: the last rows of the large call against a small call on them, to half a step of the type (their sums may be ordered otherwise)."""
    m, k, n = 9_000_001, 256, 240
    x = torch.empty(m, k, dtype=torch.bfloat16, device='cuda')
    x[:] = torch.randn(1, k, device='cuda')
    tail = torch.randn(700, k, device='cuda').to(x.dtype)
    x[-700:] = tail
    w, b = (torch.randn(n, k, device='cuda') / 16).to(x.dtype).requires_grad_(), torch.randn(n, device='cuda').to(x.dtype).requires_grad_()
    y = linear(x, w, b, act='relu')
    assert y.numel() > 2 ** 31
    close(y[-700:].detach(), dbl(linear(tail, w, b, act='relu')), 2 * unit(x.dtype) * dbl(y[-700:]).abs() + 1e-6, 'last rows')
    # a gradient in which the last rows alone count
    dy = torch.zeros(m, n, dtype=x.dtype, device='cuda')
    dy[-700:] = torch.randn(700, n, device='cuda').to(x.dtype)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    t = tail.clone().requires_grad_()
    w2, b2 = w.detach().clone().requires_grad_(), b.detach().clone().requires_grad_()
    dt2, dw2, db2 = torch.autograd.grad(linear(t, w2, b2, act='relu'), (t, w2, b2), dy[-700:].contiguous())
    for got, want in ((dw, dw2), (db, db2)):
        close(got, dbl(want), 2 * unit(x.dtype) * dbl(want).abs() + 1e-4 * float(want.abs().max()), 'gradients')
    del dy, y
    h = layer_norm(x)
    close(h[-700:], dbl(layer_norm(tail)), 2 * unit(x.dtype) * dbl(h[-700:]).abs() + 1e-6, 'norm of the last rows')
    del h
    xt = torch.empty(k, m, dtype=torch.bfloat16, device='cuda')              # channel-first points, their rows 18 MB apart
    xt[:] = x.t()
    y1 = linear(xt.t(), w.detach()[:1])
    close(y1[-700:], dbl(linear(tail, w.detach()[:1])), 2 * unit(x.dtype) * dbl(y1[-700:]).abs() + 1e-2 * 2.0 ** -8, 'one output')
    y2 = linear(xt.t(), w.detach()[:40])
    close(y2[-700:], dbl(linear(tail, w.detach()[:40])), 2 * unit(x.dtype) * dbl(y2[-700:]).abs() + 1e-2 * 2.0 ** -8, 'forty outputs')
    wl = w.detach()[:5].clone().requires_grad_()
    out = linear(xt.t(), wl)
    (dw5,) = torch.autograd.grad(out, wl, torch.cat([torch.zeros(m - 700, 5, device='cuda', dtype=x.dtype), torch.ones(700, 5, device='cuda', dtype=x.dtype)]))
    want = dbl(tail).sum(0).expand(5, k)
    close(dw5, want, 2 * unit(x.dtype) * want.abs() + 700 * E32 * dbl(tail).abs().sum(0), 'weight gradient of channel-first points')


def test_slopes_where_float16_overflows():
    """z = +-80000 is infinite in float16 while gelu and silu, and their slopes, are 0 or z and 1: the gradient stays finite."""
    for act in ('gelu', 'silu', 'tanh', 'sigmoid', 'soft_plus'):
        x = torch.tensor([[-400.0], [400.0]], dtype=torch.float16, device='cuda')
        w = torch.tensor([[200.0]], dtype=torch.float16, device='cuda').requires_grad_()
        y = linear(x, w, act=act)
        (g,) = torch.autograd.grad(y, w, torch.tensor([[1.0], [0.0]], dtype=torch.float16, device='cuda'))
        assert float(y[0, 0].abs()) <= 1 and float(g) == 0.0, (act, y, g)


def test_more_rows_than_a_launch_takes():
    m, k, n = (1 << 26) + 77, 8, 24
    x = torch.randn(1, k, device='cuda').to(torch.bfloat16).expand(m, k).contiguous()
    x[-400:] = torch.randn(400, k, device='cuda').to(x.dtype)
    w = torch.randn(n, k, device='cuda').to(x.dtype).requires_grad_()
    y = linear(x, w, act='relu')
    assert torch.equal(y[-400:], linear(x[-400:].contiguous(), w, act='relu')) and torch.equal(y[:1].expand(5, n), y[12345:12350])
    dy = torch.zeros_like(y)
    dy[-400:] = 1
    (dw,) = torch.autograd.grad(y, w, dy)
    want = ((dbl(x[-400:]) @ dbl(w).t() > 0).double().t() @ dbl(x[-400:]))
    kink = (dbl(x[-400:]) @ dbl(w).t()).abs() < 1e-5
    assert not bool(kink.any())
    close(dw, want, 2 * unit(x.dtype) * want.abs() + 400 * E32 * dbl(x[-400:]).abs().sum(0), 'dw')


def test_empty_batches_of_the_mlp():
    from avatarcap_amd.network.mlp import MLP
    net = MLP(6, 2, [16, 8], res_layers=[1]).cuda()
    for shape in ((1, 6, 0), (0, 6, 5), (2, 6, 0)):
        assert net(torch.zeros(shape, device='cuda')).shape == (shape[0], 2, shape[2])
    with pytest.raises(ValueError):
        net(torch.zeros(1, 5, 4, device='cuda'))
    with pytest.raises(TypeError):
        net(torch.zeros(1, 6, 4, device='cuda').half())
    half = net.half()
    assert half(torch.ones(1, 6, 4, device='cuda').half()).dtype == torch.float16


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('layout', ['rows', 'channels'])
def test_padded_copies_and_cuts(layout, dtype):
    """Odd sizes large enough that operands are copied to padded rows and the product is cut into a main part and strips (the workspace says so)."""
    import ctypes as C
    m, k, n = 4099, 1027, 2055
    nb = C.c_int64()
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    xr, xc = (k, 1) if layout == 'rows' else (1, m)
    _lib.check(_lib.lib().avc_linear_workspace(m, n, k, code, xr, xc, C.byref(nb)))
    copied = (k + 5) * m * (4 if code == 0 else 2)
    assert nb.value >= (0 if code == 0 and layout == 'rows' else copied * 0.99)
    check_linear(m, k, n, dtype, act='silu', layout=layout, residual=True)
    check_linear(m, k, n, dtype, layout=layout, bias=False)
