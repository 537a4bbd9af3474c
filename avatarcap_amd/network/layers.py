"""The layers an MLP is made of as differentiable calls on the HIP library: the dense layer with bias, activation and residual in its epilogue, and the layer norm.

    y = linear(x, weight, bias, act='relu', residual=r)        y = act(x W^T + b) + r
    y = layer_norm(x, weight, bias)                            y = (x - mean) / sqrt(var + eps) * g + b over the last axis

`linear` is what one step of the reference's `MLP.forward` does (network/mlp.py:56-72: a Conv1d(k=1) and its activation), for any widths; network/mlp.py calls it.  Tensors are
float32, bfloat16 or float16, all of one call alike, on the HIP device; there is no CPU path.  Both run on the current stream of the tensors' device, whichever device is current,
take their workspace from torch's allocator (so a captured graph keeps its own) and have a backward pass of the same kernels (csrc/linear.hip, linear_tile.hip, layer_norm.hip).
No gradient of a gradient: taking one raises.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from .. import _lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}                 # avc_dtype
ACTS = {None: 0, 'relu': 1, 'leaky_relu': 2, 'soft_plus': 3, 'sigmoid': 4, 'tanh': 5, 'gelu': 6, 'silu': 7}   # avc_act


def _check_first(who, x):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f'{who}: x: expected a torch.Tensor, got {type(x).__name__}')
    if not x.is_cuda:
        raise RuntimeError(f'{who} runs on the HIP device only; there is no CPU path (x lives on {x.device})')
    if x.dtype not in DTYPES:
        raise TypeError(f'{who}: float32, bfloat16 or float16, got {x.dtype}')


def _check_like(who, name, t, x):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f'{who}: {name}: expected a torch.Tensor, got {type(t).__name__}')
    if t.dtype is not x.dtype:
        raise TypeError(f'{who}: {name} is {t.dtype}, x is {x.dtype}')
    if t.get_device() != x.get_device():
        raise RuntimeError(f'{who}: {name} lives on {t.device}, x on {x.device}')


_ROW_TOP, _COLUMN_TOP = 1 << 22, 1 << 25                                          # include/avcap.h: the strides that the kernels address


def _rows(t):
    """`t` (rows, columns) with adjacent columns, copied if they are not or the rows lie further apart than the kernels reach."""
    if (t.stride(1) == 1 or t.shape[1] == 1) and (t.stride(0) < _ROW_TOP or t.shape[0] <= 1):
        return t
    return t.contiguous()


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _matrix(x, column_top=_COLUMN_TOP):
    """`x` (rows, columns) and its strides, one of which is 1: rows of adjacent values, or channel-first (a transposed view).  Copied otherwise."""
    m, k = x.shape
    if (k == 1 or x.stride(1) == 1) and (m <= 1 or x.stride(0) < _ROW_TOP):
        return x, _row_stride(x), 1
    if x.stride(0) == 1 and m > 1 and x.stride(1) < column_top:
        return x, 1, x.stride(1)
    x = x.contiguous()
    return x, k, 1


def _ptr(t):
    return None if t is None else t.data_ptr()


# Bytes of workspace, a function of sizes and type alone.
@functools.lru_cache(maxsize=4096)
def _forward_bytes(m, n, k, dt, xr, xc):
    nbytes = C.c_int64()
    _lib.check(_lib.lib().avc_linear_workspace(m, n, k, dt, xr, xc, C.byref(nbytes)))
    return nbytes.value


@functools.lru_cache(maxsize=4096)
def _backward_bytes(m, n, k, dt):
    nbytes = C.c_int64()
    _lib.check(_lib.lib().avc_linear_backward_workspace(m, n, k, dt, C.byref(nbytes)))
    return nbytes.value


@functools.lru_cache(maxsize=4096)
def _norm_backward_bytes(m, c, dt):
    nbytes = C.c_int64()
    _lib.check(_lib.lib().avc_layer_norm_backward_workspace(m, c, dt, C.byref(nbytes)))
    return nbytes.value


def _space(nbytes, like):
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def _stream(t):
    return torch._C._cuda_getCurrentRawStream(t.get_device())         # what torch.cuda.current_stream(t.device).cuda_stream is, without the objects around it


class _NoSecond(torch.autograd.Function):
    @staticmethod
    def forward(ctx, live, *grads):
        return tuple(g.detach() for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError('linear, layer_norm: the gradients have no derivative of their own')


def _once(backward, ctx, dy):
    """The backward pass under create_graph, which is when the engine leaves gradients enabled: a derivative taken of its results raises, whether dy itself carries a graph or not,
    instead of leaving out what runs through x and the weights."""
    with torch.no_grad():
        out = list(backward(ctx, dy))
    at = [i for i, g in enumerate(out) if g is not None and g is not dy]
    for i, g in zip(at, _NoSecond.apply(torch.zeros((), requires_grad=True), *[out[i] for i in at]) if at else ()):
        out[i] = g
    return tuple(out)


def _linear_forward(x, w, bias, res, act, slope, want_z):
    m, k = x.shape
    n = w.shape[0]
    dt = DTYPES[x.dtype]
    x, xr, xc = _matrix(x)
    w = _rows(w)
    y = x.new_empty((m, n))
    z = x.new_empty((m, n)) if want_z else None            # bf16 of soft_plus ... silu: float16 bits (csrc/linear.h KeptZ)
    nbytes = _forward_bytes(m, n, k, dt, xr, xc)
    ws = _space(nbytes, x)
    _lib.check(_lib.lib().avc_linear(_lib.ctx(x.get_device()), x.data_ptr(), xr, xc, w.data_ptr(), _row_stride(w), _ptr(bias), _ptr(res), 0 if res is None else _row_stride(res), act, slope, m, n, k,
                                     dt, y.data_ptr(), n, _ptr(z), n, _ptr(ws), nbytes, _stream(x)))
    return y, z


def _linear_backward(ctx, dy):
    x, w, saved = ctx.saved_tensors
    need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
    dx = dw = db = None
    if need_x or need_w or need_b:
        (m, k), n, dt = x.shape, w.shape[0], DTYPES[dy.dtype]
        g = _rows(dy)
        x, xr, xc = _matrix(x, _ROW_TOP)
        w = _rows(w)
        dx = g.new_empty((m, k)) if need_x else None
        dw = g.new_empty((n, k)) if need_w else None
        db = g.new_empty((n,)) if need_b else None
        nbytes = _backward_bytes(m, n, k, dt)
        ws = _space(nbytes, g)
        _lib.check(_lib.lib().avc_linear_backward(_lib.ctx(g.get_device()), g.data_ptr(), _row_stride(g), x.data_ptr(), xr, xc, w.data_ptr(), _row_stride(w), _ptr(saved), n, ctx.act, ctx.slope,
                                                  m, n, k, dt, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nbytes, _stream(g)))
    return dx, dw, db, dy if need_r else None, None, None


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, res, act, slope):
        # relu and leaky_relu leave the sign of z in y: z is kept only where y does not have it
        from_y = act in (1, 2) and res is None
        y, z = _linear_forward(x, w, bias, res, act, slope, want_z=act != 0 and not from_y)
        ctx.save_for_backward(x, w, y if from_y else z)
        ctx.act, ctx.slope = act, slope
        return y

    @staticmethod
    def backward(ctx, dy):
        return _once(_linear_backward, ctx, dy) if torch.is_grad_enabled() else _linear_backward(ctx, dy)


def linear(x, weight, bias=None, act=None, slope=0.02, residual=None):
    """act(x W^T + b) + residual in one pass.

    x (..., K); weight (N, K), or (N, K, 1) as Conv1d(k=1) keeps it; bias (N); residual (..., N) -> (..., N).  act: None, 'relu', 'leaky_relu' (z > 0 ? z : slope z, slope >= 0),
    'soft_plus' (torch's threshold of 20), 'sigmoid', 'tanh', 'gelu' (z Phi(z), not the tanh form), 'silu'.  x may be a transposed view (channel-first points) or any slice with one
    unit stride; other layouts are copied.  Sums are float32 and each output is rounded once; float32 products keep 24 bits."""
    if act not in ACTS:
        raise ValueError(f'linear: unknown activation {act!r}, known are {[a for a in ACTS if a]}')
    _check_first('linear', x)
    _check_like('linear', 'weight', weight, x)
    if bias is not None:
        _check_like('linear', 'bias', bias, x)
    if residual is not None:
        _check_like('linear', 'residual', residual, x)
    if weight.dim() == 3 and weight.shape[2] == 1:
        weight = weight[:, :, 0]
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f'linear: x {tuple(x.shape)} does not fit weight {tuple(weight.shape)}')
    n, k = weight.shape
    if n < 1 or k < 1:
        raise ValueError(f'linear: a weight of shape {tuple(weight.shape)} has no values')
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != n):
        raise ValueError(f'linear: bias {tuple(bias.shape)} for {n} outputs')
    if residual is not None and residual.shape != x.shape[:-1] + (n,):
        raise ValueError(f'linear: residual {tuple(residual.shape)}, the output is {tuple(x.shape[:-1]) + (n,)}')
    if act == 'leaky_relu' and not 0.0 <= slope < float('inf'):
        raise ValueError(f'linear: leaky_relu takes a finite slope >= 0, got {slope}')
    m = x.numel() // k
    x2 = x if x.dim() == 2 else x.reshape(m, k)
    r2 = None if residual is None else _rows(residual if residual.dim() == 2 else residual.reshape(m, n))
    if bias is not None and n > 1 and bias.stride(0) != 1:
        bias = bias.contiguous()
    code = ACTS[act]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or (residual is not None and residual.requires_grad)):
        y = _Linear.apply(x2, weight, bias, r2, code, slope)
    else:
        y, _ = _linear_forward(x2, weight, bias, r2, code, slope, want_z=False)
    return y if x.dim() == 2 else y.reshape(x.shape[:-1] + (n,))


def _norm_forward(x, g, b, eps, want_stats):
    m, c = x.shape
    x = _rows(x)
    y = x.new_empty((m, c))
    stats = x.new_empty((2, m), dtype=torch.float32) if want_stats else None
    p = _ptr(stats)
    _lib.check(_lib.lib().avc_layer_norm(_lib.ctx(x.get_device()), x.data_ptr(), _row_stride(x), _ptr(g), _ptr(b), eps, m, c, DTYPES[x.dtype], y.data_ptr(), c, p, p + 4 * m if p else p, _stream(x)))
    return y, stats


def _norm_backward(ctx, dy):
    x, g, stats = ctx.saved_tensors
    need_x, need_g, need_b = ctx.needs_input_grad[:3]
    (m, c), dt = x.shape, DTYPES[dy.dtype]
    x, dy = _rows(x), _rows(dy)
    dx = dy.new_empty((m, c)) if need_x else None
    dg = dy.new_empty((c,)) if need_g else None
    db = dy.new_empty((c,)) if need_b else None
    nbytes = _norm_backward_bytes(m, c, dt) if need_g or need_b else 0
    ws = _space(nbytes, dy)
    p = stats.data_ptr()
    _lib.check(_lib.lib().avc_layer_norm_backward(_lib.ctx(dy.get_device()), dy.data_ptr(), _row_stride(dy), x.data_ptr(), _row_stride(x), _ptr(g), p, p + 4 * m, m, c, dt, _ptr(dx), c, _ptr(dg),
                                                  _ptr(db), _ptr(ws), nbytes, _stream(dy)))
    return dx, dg, db, None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, g, b, eps):
        y, stats = _norm_forward(x, g, b, eps, want_stats=True)
        ctx.save_for_backward(x, g, stats)
        return y

    @staticmethod
    def backward(ctx, dy):
        return _once(_norm_backward, ctx, dy) if torch.is_grad_enabled() else _norm_backward(ctx, dy)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """The layer norm over the last axis: x (..., C), weight and bias (C) or None -> (..., C).  Mean and biased variance in float32, the variance from centred values."""
    _check_first('layer_norm', x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f'layer_norm: x {tuple(x.shape)} has no values along its last axis')
    c = x.shape[-1]
    for name, t in (('weight', weight), ('bias', bias)):
        if t is not None:
            _check_like('layer_norm', name, t, x)
            if t.dim() != 1 or t.shape[0] != c:
                raise ValueError(f'layer_norm: {name} {tuple(t.shape)} for rows of {c}')
    eps = float(eps)
    if not 0.0 <= eps < float('inf'):
        raise ValueError(f'layer_norm: eps must be finite and >= 0, got {eps}')
    x2 = x if x.dim() == 2 else x.reshape(x.numel() // c, c)
    if weight is not None and weight.stride(0) != 1:
        weight = weight.contiguous()
    if bias is not None and bias.stride(0) != 1:
        bias = bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        y = _LayerNorm.apply(x2, weight, bias, eps)
    else:
        y, _ = _norm_forward(x2, weight, bias, eps, want_stats=False)
    return y if x.dim() == 2 else y.reshape(x.shape)
