"""The dense layer's and the layer norm's surface without a GPU: what the Python calls and the C entries refuse, and the workspace arithmetic."""
import ctypes as C

import pytest
import torch

from avatarcap_amd import _lib
from avatarcap_amd.network.layers import _matrix, _rows, layer_norm, linear
from avatarcap_amd.network.mlp import MLP

ARG, CAPACITY = -1, _lib.AVC_ERR_CAPACITY
ANY = 4096                                                                   # a non-NULL pointer: a refused call reads nothing through it


@pytest.mark.skipif(torch.cuda.is_available(), reason='checks the no-GPU failure mode')
def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match='HIP device only'):
        linear(torch.zeros(2, 3), torch.zeros(4, 3))
    with pytest.raises(RuntimeError, match='HIP device only'):
        layer_norm(torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match='HIP device only'):
        MLP(3, 1, [4])(torch.zeros(1, 3, 2))
    with pytest.raises(ValueError):
        MLP(3, 1, [4])(torch.zeros(1, 4, 2))
    with pytest.raises(TypeError):
        linear([1.0], torch.zeros(4, 1))
    with pytest.raises(ValueError, match='unknown activation'):
        linear(torch.zeros(2, 3), torch.zeros(4, 3), act='step')


def test_layouts_that_need_no_copy():
    x = torch.zeros(6, 8)
    for t, strides in ((x, (8, 1)), (x[:, 2:7], (8, 1)), (x.t(), (1, 8)), (x[::2], (16, 1)), (x[:1].expand(5, 8), (0, 1)), (x[:, :1], (8, 1)), (x[0:1], (8, 1))):
        y, r, c = _matrix(t)
        assert y.data_ptr() == t.data_ptr() and (r, c) == strides, t.stride()
    y, r, c = _matrix(x[:, ::2])
    assert (r, c) == (4, 1) and y.is_contiguous()
    assert _rows(x[:, 1:5]).data_ptr() == x[:, 1:5].data_ptr() and _rows(x.t()).is_contiguous()


def _linear(lib, m=4, n=3, k=5, dt=0, ctx=ANY, x=ANY, xr=None, xc=1, w=ANY, ldw=None, res=None, ldr=0, act=0, y=ANY, ldy=None, z=None, ldz=0, ws=None, nbytes=0):
    return lib.avc_linear(ctx, x, k if xr is None else xr, xc, w, k if ldw is None else ldw, None, res, ldr, act, 0.0, m, n, k, dt, y, n if ldy is None else ldy, z, ldz, ws, nbytes, None)


def test_the_c_entries_refuse_what_they_document():
    lib = _lib.lib()
    for bad in (dict(ctx=None), dict(x=None), dict(w=None), dict(y=None), dict(m=-1), dict(n=0), dict(k=0), dict(m=1 << 31), dict(dt=3), dict(dt=-1), dict(act=8), dict(act=-1),
                dict(xr=8, xc=2), dict(xr=-5), dict(xr=1 << 22), dict(xr=1, xc=1 << 25), dict(ldw=-1), dict(ldw=1 << 22), dict(ldy=2), dict(res=ANY, ldr=-1), dict(z=ANY, ldz=2)):
        assert _linear(lib, **bad) == ARG, bad
        assert lib.avc_last_error()
    need = C.c_int64()
    assert lib.avc_linear_workspace(40, 72, 4096, 0, 4096, 1, C.byref(need)) == 0 and need.value > 0 and need.value % 4 == 0      # a long sum over few tiles is split
    for ws, nbytes in ((None, 0), (ANY, need.value - 1), (ANY + 4, need.value), (None, need.value)):
        assert _linear(lib, m=40, n=72, k=4096, ws=ws, nbytes=nbytes) == CAPACITY
    assert lib.avc_linear_workspace(0, 72, 4096, 0, 4096, 1, C.byref(need)) == 0 and need.value == 0
    assert lib.avc_linear_workspace(1, 4096, 1024, 1, 1024, 1, C.byref(need)) == 0 and need.value == 0                              # one row: no splits
    assert lib.avc_linear_workspace(4, 3, 5, 0, 5, 1, None) == ARG and lib.avc_linear_workspace(4, 3, 5, 9, 5, 1, C.byref(need)) == ARG

    def backward(m=600, n=3, k=5, dt=0, ctx=ANY, dy=ANY, lddy=3, x=ANY, xr=5, xc=1, w=ANY, ldw=5, saved=ANY, lds=3, act=1, dx=ANY, dw=ANY, db=ANY, ws=ANY, nbytes=1 << 40):
        return lib.avc_linear_backward(ctx, dy, lddy, x, xr, xc, w, ldw, saved, lds, act, 0.0, m, n, k, dt, dx, dw, db, ws, nbytes, None)
    for bad in (dict(ctx=None), dict(dy=None), dict(x=None), dict(w=None), dict(saved=None), dict(act=9), dict(lddy=-1), dict(lddy=1 << 22), dict(ldw=1 << 22), dict(lds=1 << 22), dict(xr=7, xc=7),
                dict(xr=1, xc=1 << 22), dict(n=0), dict(dt=4)):
        assert backward(**bad) == ARG, bad
    assert backward(nbytes=8) == CAPACITY and backward(ws=None) == CAPACITY and backward(ws=ANY + 8) == CAPACITY
    assert lib.avc_linear_backward_workspace(8, 8, 8, 0, C.byref(need)) == 0 and need.value == 0                                     # one launch
    assert lib.avc_linear_backward_workspace(0, 8, 8, 0, C.byref(need)) == 0

    def norm(m=4, c=5, dt=0, ctx=ANY, x=ANY, ldx=5, eps=1e-5, y=ANY, ldy=5, mean=None, rstd=None):
        return lib.avc_layer_norm(ctx, x, ldx, None, None, eps, m, c, dt, y, ldy, mean, rstd, None)
    for bad in (dict(ctx=None), dict(x=None), dict(y=None), dict(c=0), dict(m=-1), dict(c=1 << 26), dict(dt=5), dict(ldx=-1), dict(ldy=4), dict(eps=-1.0), dict(eps=float('nan')),
                dict(mean=ANY), dict(rstd=ANY)):
        assert norm(**bad) == ARG, bad

    def norm_backward(m=600, c=5, dt=0, ctx=ANY, dy=ANY, lddy=5, x=ANY, ldx=5, mean=ANY, rstd=ANY, dx=ANY, lddx=5, dg=ANY, ws=ANY, nbytes=1 << 40):
        return lib.avc_layer_norm_backward(ctx, dy, lddy, x, ldx, None, mean, rstd, m, c, dt, dx, lddx, dg, None, ws, nbytes, None)
    for bad in (dict(ctx=None), dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(lddy=-1), dict(ldx=-1), dict(lddx=4), dict(c=0), dict(dt=3)):
        assert norm_backward(**bad) == ARG, bad
    assert norm_backward(nbytes=8) == CAPACITY and norm_backward(ws=None) == CAPACITY


def test_workspace_is_a_function_of_sizes_and_grows_with_the_splits_only():
    lib, need = _lib.lib(), C.c_int64()
    for dt in (0, 1, 2):
        for m, n, k in ((65537, 256, 545), (16384, 8192, 4096), (8192, 2048, 2048), (300, 17, 9)):
            got = []
            for _ in range(2):
                assert lib.avc_linear_workspace(m, n, k, dt, k, 1, C.byref(need)) == 0
                got.append(need.value)
            assert got[0] == got[1] and got[0] <= 4 * 100_000_000                # float32 sums of all splits: at most 1e8 of them
            assert lib.avc_linear_backward_workspace(m, n, k, dt, C.byref(need)) == 0
            assert need.value <= 4 * 100_000_000 + 4 * m * n + 4 * 2048 * n + 1024
