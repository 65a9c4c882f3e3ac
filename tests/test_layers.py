"""CPU-side checks of the layer operators (optex_group_norm, optex_gemm_bias_act and their backward passes): every call that the
kernels could not serve is refused on the host, before anything is launched."""
import ctypes

import pytest
import torch

from optimaltextures_amd import _lib, layers, ops

F32, BF16, F16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.fixture(scope="module")
def mem():
    """host memory that stands for device memory in calls that are refused"""
    buf = (ctypes.c_char * (1 << 16))()
    base = (ctypes.addressof(buf) + 255) // 256 * 256
    return buf, base


def norm_args(base, **over):
    a = dict(x=base, ldx=8, xss=64, y=base + 8192, ldy=8, yss=64, dtype=F32, n=8, C=8, S=2, G=2, w=None, b=None, astride=0, adtype=F32,
             eps=1e-5, act=0, mean=None, rstd=None, ws=base + 16384, wsb=1 << 15, st=None)
    a.update(over)
    return list(a.values())


def test_group_norm_refuses_on_the_host(lib, mem):
    base = mem[1]
    need = lib.optex_group_norm_ws_bytes(1 << 20, 8, 2, 2, F32)
    assert need > 0 and lib.optex_group_norm_ws_bytes(0, 8, 2, 2, F32) == 0
    bad = [dict(dtype=3), dict(adtype=BF16), dict(n=-1), dict(S=-1), dict(C=0), dict(G=0), dict(G=3), dict(act=4), dict(act=-1),
           dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(astride=4), dict(mean=base), dict(x=None), dict(y=None),
           dict(x=base + 1), dict(ldx=7), dict(ldy=4), dict(xss=63), dict(yss=10), dict(y=base + 32), dict(y=base, ldy=9, yss=72),
           dict(w=base + 2), dict(ws=base + 16384 + 4), dict(w=base + 8192 + 32), dict(b=base + 8192), dict(mean=base + 64, rstd=base + 20000),
           dict(mean=base + 20000, rstd=base + 20004), dict(mean=base + 20002, rstd=base + 20100)]
    for over in bad:
        assert lib.optex_group_norm(*norm_args(base, **over)) == -1, over
        assert b"optex_group_norm" in lib.optex_last_error(), over
    # a map that does not fit on chip needs its scratch
    for over in (dict(ws=None), dict(wsb=need - 1)):
        assert lib.optex_group_norm(*norm_args(base, n=1 << 20, xss=8 << 20, yss=8 << 20, y=base + (1 << 40), **over)) == -1, over
        assert b"scratch buffer too small" in lib.optex_last_error()
    assert lib.optex_group_norm(*norm_args(base, C=1 << 21, ldx=1 << 21, ldy=1 << 21)) == -3
    assert lib.optex_group_norm(*norm_args(base, n=1 << 20, S=1 << 30, C=512, ldx=512, G=1)) == -3
    # nothing to do: nothing is read, nothing is launched
    assert lib.optex_group_norm(*norm_args(base, n=0, x=None, y=None, ws=None, wsb=0)) == 0
    assert lib.optex_group_norm(*norm_args(base, S=0, x=None, y=None, ws=None, wsb=0)) == 0


def norm_grad_args(base, **over):
    a = dict(dy=base, lddy=8, dyss=64, x=base + 4096, ldx=8, xss=64, dx=base + 8192, lddx=8, dxss=64, dtype=F32, n=8, C=8, S=2, G=2,
             mean=base + 12288, rstd=base + 12300, w=None, b=None, astride=0, adtype=F32, act=0, dw=None, db=None, ws=base + 16384,
             wsb=1 << 15, st=None)
    a.update(over)
    return list(a.values())


def test_group_norm_backward_refuses_on_the_host(lib, mem):
    base = mem[1]
    need = lib.optex_group_norm_backward_ws_bytes(8, 8, 2, 2, F32)
    bad = [dict(dtype=-1), dict(adtype=F16), dict(G=5), dict(act=9), dict(astride=7), dict(mean=None), dict(rstd=None), dict(dy=None),
           dict(x=None), dict(dx=None), dict(lddy=7), dict(dxss=1), dict(dx=base + 16), dict(dx=base + 4096 + 16), dict(dw=base + 3),
           dict(db=base + 1), dict(wsb=need - 1), dict(ws=None), dict(ws=base + 16384 + 8), dict(w=base + 20000, dw=base + 20000),
           dict(dw=base + 20000, db=base + 20016), dict(dw=base + 12288), dict(dw=base + 4096), dict(db=base + 8192)]
    for over in bad:
        assert lib.optex_group_norm_backward(*norm_grad_args(base, **over)) == -1, over
        assert b"optex_group_norm_backward" in lib.optex_last_error(), over
    assert lib.optex_group_norm_backward(*norm_grad_args(base, n=0)) == 0


def product_args(base, **over):
    a = dict(X=base, ldx=8, W=base + 2048, ldw=8, bias=None, res=None, ldr=16, Y=base + 8192, ldy=16, pre=None, ldp=16, dtype=F32, bdtype=F32,
             n=4, M=16, K=8, act=0, ws=None, wsb=0, st=None)
    a.update(over)
    return list(a.values())


def test_gemm_bias_act_refuses_on_the_host(lib, mem):
    base = mem[1]
    bad = [dict(dtype=5), dict(bdtype=BF16), dict(n=-1), dict(M=-2), dict(K=-1), dict(act=4), dict(X=None), dict(W=None), dict(Y=None),
           dict(X=base + 2), dict(ldx=7), dict(ldw=0), dict(ldy=15), dict(res=base + 9000, ldr=3), dict(pre=base + 9000, ldp=3),
           dict(bias=base + 1), dict(Y=base), dict(Y=base + 2048), dict(pre=base), dict(pre=base + 2048), dict(pre=base + 8192),
           dict(res=base + 8192 + 4), dict(res=base + 8192, ldr=17), dict(res=base + 4096, pre=base + 4096)]
    for over in bad:
        assert lib.optex_gemm_bias_act(*product_args(base, **over)) == -1, over
        assert b"optex_gemm_bias_act" in lib.optex_last_error(), over
    # a split sum needs its scratch
    need = lib.optex_gemm_bias_act_ws_bytes(4, 16, 512, F32)
    if need:
        assert lib.optex_gemm_bias_act(*product_args(base, K=512, ldx=512, ldw=512, W=base + 20000, ws=base, wsb=need - 1)) == -1
    assert lib.optex_gemm_bias_act(*product_args(base, n=0, X=None, Y=None)) == 0
    assert lib.optex_gemm_bias_act(*product_args(base, M=0, W=None, Y=None)) == 0


def product_grad_args(base, **over):
    a = dict(dY=base, lddy=16, X=base + 2048, ldx=8, W=base + 4096, ldw=8, pre=base + 6144, ldp=16, dX=base + 8192, lddx=8, dW=base + 10240,
             lddw=8, db=base + 12288, dtype=F32, bdtype=F32, n=4, M=16, K=8, act=2, ws=base + 16384, wsb=1 << 15, st=None)
    a.update(over)
    return list(a.values())


def test_gemm_bias_act_backward_refuses_on_the_host(lib, mem):
    base = mem[1]
    need = lib.optex_gemm_bias_act_backward_ws_bytes(4, 16, 8, F32, 2)
    assert need > 0
    bad = [dict(dtype=7), dict(bdtype=F16), dict(act=-1), dict(dY=None), dict(pre=None), dict(lddy=9), dict(ldp=1), dict(W=None), dict(X=None),
           dict(lddx=7), dict(lddw=2), dict(db=base + 12289), dict(dX=base), dict(dW=base + 2048), dict(db=base + 4096), dict(dW=base + 8192),
           dict(db=base + 8192), dict(ws=None), dict(wsb=need - 1), dict(ws=base + 16384 + 2)]
    for over in bad:
        assert lib.optex_gemm_bias_act_backward(*product_grad_args(base, **over)) == -1, over
        assert b"optex_gemm_bias_act_backward" in lib.optex_last_error(), over


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU failure mode")
def test_layer_operators_fail_loudly_without_gpu():
    x, w = torch.rand(2, 4, 4, 8), torch.rand(8, 8, requires_grad=True)
    for f in (lambda: ops.group_norm(x, 2), lambda: ops.gemm_bias_act(x, w.detach()), lambda: layers.group_norm_act(x, 2),
              lambda: layers.linear_act(x, w), lambda: ops.group_norm_backward(x, x, x, x, 2),
              lambda: ops.gemm_bias_act_backward(x, x, w.detach())):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()


def test_rows_and_maps_describe_strided_views():
    """ops._rows / ops._maps: which views are passed through, which are copied"""
    x = torch.arange(2 * 5 * 6 * 16, dtype=torch.float32).reshape(2, 5, 6, 16)
    v, ld = ops._rows(x[..., 4:12])
    assert ld == 16 and v.data_ptr() == x[..., 4:12].data_ptr()
    v, ld, ss, n = ops._maps(x[:, 1:3, :, :8])      # a crop of whole rows, half of the channels
    assert (ld, ss, n) == (16, 5 * 6 * 16, 12) and v.data_ptr() == x[:, 1:3].data_ptr()
    for view in (x[:, :, 1:4], x[..., ::2], x.permute(0, 3, 1, 2), x[:, :1].expand(2, 5, 6, 16), x[0, 0, 0].expand(2, 5, 6, 16)):
        v, ld, ss, n = ops._maps(view)
        assert v.is_contiguous() and torch.equal(v, view)
        v, ld = ops._rows(view)
        assert v.is_contiguous() and torch.equal(v, view) and ld == view.shape[-1]
    v, ld, ss, n = ops._maps(x[0, 0, :, :5])
    assert (ld, ss, n) == (5, 16, 1)
    assert ops._rows(x[:, 0, 0, 3:9])[1] == 5 * 6 * 16
