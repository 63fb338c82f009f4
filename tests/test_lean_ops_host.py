"""Argument checks of the lean training-step operators that need no GPU: the C entry
points refuse bad shapes, types, layouts and workspaces before any device work, and the
Python calls refuse CPU tensors."""
import pytest
import torch

import paper_01_anti_decoy_pnfirtau_b200 as P
from paper_01_anti_decoy_pnfirtau_b200 import _lib

BF16, FP32 = _lib.DTYPE_BF16, _lib.DTYPE_F32
A = 1 << 20  # an address that is never read: every call below is refused first


def refused(rc, code, word):
    assert rc == code and word in _lib.last_error(), (rc, _lib.last_error())


def gated(M=4, D=64, F=128, act=0, dtype=BF16, ldx=64, ldh=128, x=A, h=A, pre=None, ldp=128, b_dtype=FP32):
    return _lib.lib().pnft_gated_fwd(x, ldx, A, 64, A, 64, None, None, b_dtype, h, ldh, pre, ldp, M, D, F, act, dtype, None,
                                     None)


def test_gated_fwd_refuses():
    refused(gated(M=-1), _lib.EINVAL, "shape")
    refused(gated(D=0), _lib.EINVAL, "shape")
    refused(gated(F=0), _lib.EINVAL, "shape")
    refused(gated(act=2), _lib.EINVAL, "activation")
    refused(gated(dtype=FP32), _lib.EUNSUPPORTED, "float16")
    refused(gated(h=None), _lib.EINVAL, "null")
    refused(gated(pre=A, ldp=100), _lib.EINVAL, "stride")
    refused(gated(pre=A + 8), _lib.EINVAL, "aligned")
    refused(gated(ldh=127), _lib.EINVAL, "stride")
    refused(gated(M=65, ldx=65), _lib.EUNSUPPORTED, "aligned")
    refused(gated(M=65, x=A + 2), _lib.EUNSUPPORTED, "aligned")
    refused(gated(ldx=56), _lib.EUNSUPPORTED, "aligned")
    refused(gated(b_dtype=5), _lib.EINVAL, "bias type")
    assert gated(M=0, x=None) == _lib.OK


def test_gated_backward_refuses():
    L = _lib.lib()
    n = L.pnft_gated_bwd_workspace_size(4, 64, 128)
    assert n > 0 and L.pnft_gated_bwd_workspace_size(0, 64, 128) == 0

    def bwd(dh=A, lddh=128, pre=None, ldp=128, lddx=64, lddw=64, b=FP32, t=BF16, ws=A, nb=n, ldx=64, F=128):
        return L.pnft_gated_bwd(A, ldx, A, 64, A, 64, None, None, b, pre, ldp, dh, lddh, A, lddx, t, A, A, lddw, t, A, A, ws,
                                nb, 4, 64, F, 0, BF16, None, None)

    refused(bwd(dh=None), _lib.EINVAL, "null")
    refused(bwd(lddh=127), _lib.EINVAL, "stride")
    refused(bwd(lddx=63), _lib.EINVAL, "stride")
    refused(bwd(lddw=63), _lib.EINVAL, "stride")
    refused(bwd(pre=A + 2), _lib.EINVAL, "aligned")
    refused(bwd(lddh=129), _lib.EUNSUPPORTED, "aligned")
    refused(bwd(dh=A + 2), _lib.EUNSUPPORTED, "aligned")
    refused(bwd(b=7), _lib.EINVAL, "type")
    refused(bwd(t=-1), _lib.EINVAL, "type")
    refused(bwd(ws=None), _lib.EINVAL, "workspace")
    refused(bwd(nb=n - 1), _lib.EINVAL, "workspace")
    refused(bwd(ldx=65), _lib.EUNSUPPORTED, "aligned")


def wgrad(K=64, M=16, N=32, c1=None, row_split=16, rows=16, ldc=32, dtype=BF16, c_dtype=FP32, lddy=16):
    return _lib.lib().pnft_weight_grad(A, lddy, A, 32, A, c1, ldc, row_split, rows, c_dtype, None, 0, K, M, N, dtype, None, None)


def test_weight_grad_refuses():
    refused(wgrad(K=-1), _lib.EINVAL, "shape")
    refused(wgrad(dtype=FP32), _lib.EUNSUPPORTED, "float16")
    refused(wgrad(c_dtype=9), _lib.EINVAL, "type")
    refused(wgrad(row_split=8, rows=8), _lib.EINVAL, "null")
    refused(wgrad(row_split=8, rows=8, c1=A), _lib.EINVAL, "multiple of 128")
    two = dict(M=256, lddy=256, row_split=128, c1=A)
    refused(wgrad(rows=129, **two), _lib.EINVAL, "layout")  # more rows than the split leaves
    refused(wgrad(rows=120, **{**two, "M": 240}), _lib.EINVAL, "layout")  # past the product's end
    refused(wgrad(ldc=31), _lib.EINVAL, "layout")
    refused(wgrad(lddy=17), _lib.EUNSUPPORTED, "aligned")


def test_stream_xent_refuses():
    L = _lib.lib()
    n = L.pnft_stream_xent_fwd_workspace_size(100, 1000, 64, 1)
    assert L.pnft_stream_xent_fwd_workspace_size(100, 1000, 64, 0) > n  # the state goes there when it is not kept

    def fwd(M=100, V=1000, dtype=BF16, ws=A, nb=n, ldh=64, ldw=64, saved=A, loss=A, h=A):
        return L.pnft_stream_xent_fwd(h, ldh, A, ldw, A, -100, saved, None, loss, 1, ws, nb, M, V, 64, dtype, None, None)

    refused(fwd(M=0), _lib.EINVAL, "rows")
    refused(fwd(V=0), _lib.EINVAL, "shape")
    refused(fwd(dtype=FP32), _lib.EUNSUPPORTED, "float16")
    refused(fwd(loss=None), _lib.EINVAL, "null")
    refused(fwd(h=None), _lib.EINVAL, "null")
    refused(fwd(ldh=63), _lib.EINVAL, "stride")
    refused(fwd(saved=A + 8), _lib.EINVAL, "aligned")
    refused(fwd(ws=None), _lib.EINVAL, "workspace")
    refused(fwd(nb=n - 1), _lib.EINVAL, "workspace")
    refused(fwd(saved=None), _lib.EINVAL, "workspace")
    refused(fwd(ldw=65), _lib.EUNSUPPORTED, "aligned")
    m = L.pnft_stream_xent_bwd_workspace_size(10, 1000, 64)
    bwd = lambda dh=A, dw=A, nb=m, lddh=64, t=BF16, ldw=64: L.pnft_stream_xent_bwd(  # noqa: E731
        A, ldw, A, A, 1, 0, 1, dh, lddh, t, dw, 64, t, A, nb, 10, 1000, 64, BF16, None, None)
    refused(bwd(dh=None, dw=None), _lib.EINVAL, "null")
    refused(bwd(nb=m - 1), _lib.EINVAL, "workspace")
    refused(bwd(lddh=63), _lib.EINVAL, "stride")
    refused(bwd(t=5), _lib.EINVAL, "type")
    refused(bwd(ldw=65), _lib.EUNSUPPORTED, "aligned")


def test_stream_xent_memory_stays_small():
    """The backward's buffers for the repository's language model (32 x 511 rows, vocabulary
    33278, width 256) and a long batch: a fraction of the logits' 2 bytes per row and word."""
    L = _lib.lib()
    for M, V, D in ((16352, 33278, 256), (131072, 33278, 256), (4096, 128000, 2048)):
        kept = L.pnft_stream_xent_saved_size(M, D)
        work = max(L.pnft_stream_xent_fwd_workspace_size(M, V, D, 1), L.pnft_stream_xent_bwd_workspace_size(M, V, D))
        assert kept < 0.06 * 2 * M * V and work < 0.6 * 2 * M * V, (M, V, D, kept, work)


def test_act8_and_copies_refuse():
    L = _lib.lib()
    pack = lambda M=4, D=100, ldx=100, ldq=104, lde=1, dtype=BF16, x=A: L.pnft_act8_pack(x, ldx, A, ldq, A, lde, M, D, dtype, None)  # noqa: E731
    refused(pack(D=0), _lib.EINVAL, "shape")
    refused(pack(dtype=3), _lib.EINVAL, "dtype")
    refused(pack(x=None), _lib.EINVAL, "null")
    refused(pack(ldx=99), _lib.EINVAL, "stride")
    refused(pack(ldq=100), _lib.EINVAL, "stride")
    refused(pack(lde=0), _lib.EINVAL, "stride")
    assert pack(M=0, x=None) == _lib.OK
    refused(L.pnft_copy_rows16(A, 8, A, 4, 2, 8, None), _lib.EINVAL, "layout")
    refused(L.pnft_copy_rows16(A, 8, A, 9, 2, 8, None), _lib.EUNSUPPORTED, "aligned")
    refused(L.pnft_copy_rows16(A, 8, A + 2, 8, 2, 8, None), _lib.EUNSUPPORTED, "aligned")
    n = L.pnft_act8_weight_grad_workspace_size(4, 16, 100)
    grad = lambda dtype=BF16, lddy=16, dy=A, ws=A, nb=n, lddw=100, N=16: L.pnft_act8_weight_grad(  # noqa: E731
        dy, lddy, A, 112, A, 112, A, lddw, FP32, ws, nb, 4, N, 100, dtype, None, None)
    refused(grad(dtype=FP32), _lib.EUNSUPPORTED, "float16")
    refused(grad(lddw=99), _lib.EINVAL, "shape")
    refused(grad(lddy=15), _lib.EINVAL, "shape")
    refused(grad(dy=None), _lib.EINVAL, "null")
    refused(grad(nb=n - 1), _lib.EINVAL, "workspace")
    refused(grad(lddy=17), _lib.EUNSUPPORTED, "aligned")


def test_python_calls_refuse_cpu_tensors_and_bad_arguments():
    x, w = torch.randn(4, 64).bfloat16(), torch.randn(128, 64).bfloat16()
    with pytest.raises(RuntimeError, match="CUDA"):
        P.gated_linear(x, w, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.streamed_cross_entropy(x, w, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        P.act8_pack(x)
