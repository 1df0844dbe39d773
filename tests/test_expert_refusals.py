"""What the C entry points of the expert rows and the 4-bit products refuse, before anything reaches a GPU (the addresses are never read)."""
import ctypes as C

import pytest

OK, INVALID, WORKSPACE, UNSUPPORTED = 0, -1, -3, -4
P = C.c_void_p(1 << 20)          # an aligned address that is never read
ODD = C.c_void_p((1 << 20) + 2)
BIG = 2 ** 31 - 1


@pytest.fixture(scope='module')
def lib():
    import gunet_amd
    return gunet_amd._lib.lib


def test_sort(lib):
    def sort(index=P, t=4, k=2, e=3, offsets=P, order=P, slot=P, ws=None, nbytes=0):
        return lib.gunet_expert_sort(index, t, k, e, offsets, order, slot, ws, nbytes, None)
    for kw in (dict(t=-1), dict(k=0), dict(k=-3), dict(e=0), dict(t=2 ** 30, k=2), dict(t=2 ** 40), dict(index=None), dict(offsets=None), dict(order=None), dict(slot=None)):
        assert sort(**kw) == INVALID, kw
    assert sort(e=1025) == UNSUPPORTED and b'1024' in lib.gunet_last_error()
    assert lib.gunet_expert_sort_workspace_bytes(64, 2, 64) == 0
    need = lib.gunet_expert_sort_workspace_bytes(4097, 2, 64)
    assert need >= 2 * 64 * 4
    assert sort(t=4097, e=64) == WORKSPACE and sort(t=4097, e=64, ws=P, nbytes=need - 1) == WORKSPACE
    assert sort(t=4097, e=64, ws=C.c_void_p((1 << 20) + 1), nbytes=need) == INVALID
    assert lib.gunet_expert_sort_workspace_bytes(BIG, 1, 1024) <= 256 * 1024 * 4
    assert lib.gunet_expert_sort_workspace_bytes(-1, 2, 64) == 0


def test_rows(lib):
    def dispatch(x=P, dtype=0, offsets=P, slot=P, t=4, k=2, e=3, width=8, rows=P):
        return lib.gunet_expert_dispatch(x, dtype, offsets, slot, t, k, e, width, rows, None)

    def dispatch_grad(g=P, dtype=0, slot=P, t=4, k=2, width=8, out=P):
        return lib.gunet_expert_dispatch_grad(g, dtype, slot, t, k, width, out, None)

    def combine(rows=P, dtype=0, w=P, slot=P, t=4, k=2, width=8, out=P):
        return lib.gunet_expert_combine(rows, dtype, w, slot, t, k, width, out, None)

    def grad(g=P, rows=P, dtype=0, w=P, offsets=P, slot=P, t=4, k=2, e=3, width=8, gr=P, gw=P):
        return lib.gunet_expert_combine_grad(g, rows, dtype, w, offsets, slot, t, k, e, width, gr, gw, None)

    for fn in (dispatch, dispatch_grad, combine, grad):
        for kw in (dict(dtype=3), dict(dtype=-1), dict(t=-1), dict(k=0), dict(t=2 ** 31), dict(width=-1), dict(width=2 ** 30 + 1), dict(slot=None)):
            assert fn(**kw) == INVALID, (fn.__name__, kw)
        assert fn(t=0) == OK
    for fn in (dispatch, dispatch_grad, combine):
        assert fn(width=0) == OK
    for fn, names in ((dispatch, ('x', 'offsets', 'rows')), (dispatch_grad, ('g', 'out')), (combine, ('rows', 'w', 'out')),
                      (grad, ('g', 'rows', 'w', 'offsets', 'gr', 'gw'))):
        for name in names:
            assert fn(**{name: None}) == INVALID, (fn.__name__, name)
    # a tensor that does not lie on its element's size cannot be read at all
    assert dispatch(x=C.c_void_p((1 << 20) + 1), dtype=1) == INVALID and combine(out=ODD) == INVALID
    assert grad(gr=C.c_void_p((1 << 20) + 1), dtype=2) == INVALID and dispatch_grad(g=ODD) == INVALID


def test_mxfp4(lib):
    assert lib.gunet_mxfp4_code_bytes(1, 5, 33) == 5 * 2 * 16 and lib.gunet_mxfp4_scale_bytes(1, 5, 33) == 5 * 8
    assert lib.gunet_mxfp4_code_bytes(3, 5, 257) == 3 * 5 * 9 * 16 and lib.gunet_mxfp4_scale_bytes(3, 5, 257) == 3 * 2 * 5 * 8
    assert lib.gunet_mxfp4_code_bytes(1, 5, 0) == 0 and lib.gunet_mxfp4_code_bytes(1, 5, 2 ** 22 + 1) == 0

    def quantize(x=P, dtype=0, g=1, rows=4, k=64, codes=P, scales=P):
        return lib.gunet_mxfp4_quantize(x, dtype, g, rows, k, codes, scales, None)

    def dequantize(codes=P, scales=P, g=1, rows=4, k=64, x=P, dtype=0):
        return lib.gunet_mxfp4_dequantize(codes, scales, g, rows, k, x, dtype, None)

    for fn in (quantize, dequantize):
        for kw in (dict(dtype=3), dict(g=-1), dict(g=65536), dict(rows=-1), dict(rows=2 ** 31), dict(k=0), dict(k=2 ** 22 + 1), dict(x=None), dict(x=ODD),
                   dict(codes=None), dict(scales=None), dict(codes=C.c_void_p((1 << 20) + 8)), dict(scales=C.c_void_p((1 << 20) + 4))):
            assert fn(**kw) == INVALID, (fn.__name__, kw)
        assert fn(rows=0) == OK and fn(g=0) == OK


def test_products(lib):
    assert lib.gunet_mxfp4_dense_workspace_bytes(40, 64) == 40 * 32 + 40 * 8 and lib.gunet_mxfp4_dense_workspace_bytes(4, 64) == 0
    need = lib.gunet_mxfp4_dense_workspace_bytes(40, 64)
    assert lib.gunet_mxfp4_expert_dense_workspace_bytes(4, 64) == 256 + 4 * 8

    def dense(x=P, dtype=0, rows=40, k=64, wc=P, ws=P, bias=None, n=8, act=0, out=P, out_dtype=0, scratch=P, nbytes=1 << 30):
        return lib.gunet_mxfp4_dense_forward(x, dtype, rows, k, wc, ws, bias, n, act, out, out_dtype, scratch, nbytes, None)

    def expert(x=P, dtype=0, offsets=P, slot=P, rows=20, top_k=2, e=3, k=64, wc=P, ws=P, bias=None, n=8, act=0, out=P, out_dtype=0, scratch=P, nbytes=1 << 30):
        return lib.gunet_mxfp4_expert_dense_forward(x, dtype, offsets, slot, rows, top_k, e, k, wc, ws, bias, n, act, out, out_dtype, scratch, nbytes, None)

    for fn in (dense, expert):
        for kw in (dict(dtype=3), dict(out_dtype=7), dict(rows=-1), dict(k=0), dict(k=2 ** 22 + 1), dict(n=0), dict(n=-4), dict(act=12), dict(act=-1), dict(x=None), dict(wc=None), dict(ws=None), dict(out=None),
                   dict(wc=C.c_void_p((1 << 20) + 8)), dict(ws=C.c_void_p((1 << 20) + 4)), dict(x=ODD), dict(out=ODD), dict(scratch=C.c_void_p((1 << 20) + 8))):
            assert fn(**kw) == INVALID, (fn.__name__, kw)
        assert fn(scratch=None) == WORKSPACE and fn(nbytes=need - 1) == WORKSPACE
        assert fn(rows=0) == OK
    for kw in (dict(offsets=None), dict(top_k=0), dict(e=0), dict(rows=2 ** 30, top_k=2), dict(e=65536)):
        assert expert(**kw) == INVALID, kw
    assert expert(nbytes=lib.gunet_mxfp4_expert_dense_workspace_bytes(40, 64) - 1) == WORKSPACE
    assert expert(rows=2, nbytes=lib.gunet_mxfp4_expert_dense_workspace_bytes(4, 64) - 1) == WORKSPACE


def test_constants_match_the_header():
    import os
    import re
    from conftest import ROOT
    from gunet_amd import _lib
    with open(os.path.join(ROOT, 'include', 'gunet_hip.h')) as f:
        defines = dict(re.findall(r'#define\s+(GUNET_[A-Z0-9_]+)\s+\(?(-?\d+)\)?', f.read()))
    assert [int(defines['GUNET_DTYPE_' + t]) for t in ('F32', 'BF16', 'F16')] == [_lib.DTYPE_F32, _lib.DTYPE_BF16, _lib.DTYPE_F16]
    assert int(defines['GUNET_MAX_EXPERTS']) == _lib.MAX_EXPERTS


def test_python_checks_need_no_gpu():
    import torch
    import gunet_amd as amd
    with pytest.raises(TypeError, match='CUDA'):
        amd.expert_plan(torch.zeros((4, 2), dtype=torch.int32), 3)
    with pytest.raises(TypeError, match='CUDA'):
        amd.mxfp4_quantize(torch.zeros((4, 64)))
    with pytest.raises(TypeError, match='Mxfp4Tensor'):
        amd.mxfp4_dense(torch.zeros((4, 64)), torch.zeros((8, 64)))
