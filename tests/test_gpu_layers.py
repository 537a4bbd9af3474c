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
        return torch.tanh(z), 1 - torch.tanh(z) ** 2
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
