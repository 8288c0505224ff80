"""Refusals and workspace sizes of the grouped products: everything the host decides without a GPU."""
import pytest
import torch

from infinite_dreams import _capi, infinite_dreams_ext as ext

LIB = _capi.lib
P = 1 << 20   # an aligned address that is never read


def _launch(A=P, B=P, C=P, off=P, bits=32, T=8, N=8, K=8, E=2, lda=8, ldb=8, sb=64, ldc=8, tb=0, bias=None, act=0,
            dtype=0):
    return LIB.gemm_grouped_launch(A, B, C, off, bits, T, N, K, E, lda, ldb, sb, ldc, tb, bias, act, 1, dtype, None, 0,
                                   None)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(K=-1), dict(E=0), dict(bits=16), dict(dtype=2), dict(tb=2),
                                 dict(act=3), dict(A=None), dict(off=None), dict(C=None), dict(lda=7), dict(ldb=7),
                                 dict(ldc=7), dict(sb=63), dict(A=P + 1), dict(bias=P + 1), dict(off=P + 2),
                                 dict(off=P + 4, bits=64)], ids=str)
def test_invalid_arguments(bad):
    assert _launch(**bad) == _capi.GEMM_ERR_INVALID_ARG
    assert LIB.gemm_last_error()


def test_unsupported_and_missing_workspace():
    assert _launch(E=1025) == _capi.GEMM_ERR_UNSUPPORTED
    assert _launch(T=1 << 31) == _capi.GEMM_ERR_UNSUPPORTED
    assert _launch(T=8, K=7, lda=7) == _capi.GEMM_ERR_WORKSPACE
    assert _launch(T=0) == _capi.GEMM_OK and _launch(N=0, sb=0) == _capi.GEMM_OK   # nothing to do


def test_workspace_sizes():
    ws = LIB.gemm_grouped_workspace_bytes
    head = LIB.gemm_workspace_counter_bytes()
    assert ws(P, P, 8, 64, 64, 2, 64, 64, 64 * 64, 0) == 0
    # rows of 77 elements are copied to 128: A, then both matrices of B
    assert ws(P, P, 100, 64, 77, 2, 77, 64, 77 * 64, 0) == head + 100 * 128 * 2
    assert ws(P, P, 100, 77, 64, 2, 64, 77, 64 * 77, 0) == head + 2 * 64 * 128 * 2
    assert ws(P + 2, P, 100, 64, 64, 2, 64, 64, 64 * 64, 0) == head + 100 * 64 * 2
    # a matrix stride that TMA cannot address
    assert ws(P, P, 100, 64, 64, 2, 64, 64, 64 * 64 + 1, 0) == head + 2 * 64 * 64 * 2


def test_torch_surface_refuses_cpu_tensors():
    A, B = torch.zeros(4, 8, dtype=torch.float16), torch.zeros(2, 8, 8, dtype=torch.float16)
    off = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="A must be CUDA tensor"):
        ext.grouped_gemm(A, B, off)
    with pytest.raises(RuntimeError, match="activation must be one of"):
        ext.grouped_gemm(A, B, off, activation="tanh")
    keep, ext._fast = ext._fast, None
    try:
        with pytest.raises(RuntimeError, match="A must be CUDA tensor"):
            ext.grouped_gemm(A, B, off)
    finally:
        ext._fast = keep




def _wgrad(A=P, G=P, D=P, off=P, bits=32, T=8, M=8, N=8, E=2, lda=8, ldg=8, ldd=8, sd=64, dtype=0):
    return LIB.gemm_grouped_wgrad_launch(A, G, D, off, bits, T, M, N, E, lda, ldg, ldd, sd, dtype, None, 0, None)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(E=0), dict(bits=8), dict(dtype=-1), dict(A=None), dict(G=None),
                                 dict(D=None), dict(off=None), dict(lda=7), dict(ldg=7), dict(ldd=7), dict(sd=63),
                                 dict(G=P + 1), dict(off=P + 1)], ids=str)
def test_wgrad_invalid_arguments(bad):
    assert _wgrad(**bad) == _capi.GEMM_ERR_INVALID_ARG


def test_wgrad_limits_and_workspace():
    head = LIB.gemm_workspace_counter_bytes()
    assert _wgrad(E=1025) == _capi.GEMM_ERR_UNSUPPORTED
    assert _wgrad(M=7, lda=7) == _capi.GEMM_ERR_WORKSPACE
    assert _wgrad(M=0) == _capi.GEMM_OK
    assert LIB.gemm_grouped_wgrad_workspace_bytes(P, P, 100, 64, 64, 64, 64) == 0
    assert LIB.gemm_grouped_wgrad_workspace_bytes(P, P, 100, 77, 64, 77, 64) == head + 100 * 128 * 2


def _lora(X=P, W=P, down=P, up=P, C=P, ids=P, bits=32, T=8, N=8, K=8, L=2, R=8, ldx=8, ldw=8, tw=0, ldd=8, sd=64, td=0,
          ldu=8, su=64, tu=0, ldc=8, scale=None, bias=None, act=0, dtype=0):
    return LIB.gemm_lora_launch(X, W, down, up, C, ids, bits, T, N, K, L, R, ldx, ldw, tw, ldd, sd, td, ldu, su, tu, ldc,
                                scale, bias, act, dtype, None, 0, None)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(K=0), dict(L=0), dict(R=0), dict(bits=1), dict(dtype=5), dict(tw=2),
                                 dict(td=-1), dict(tu=2), dict(act=-1), dict(X=None), dict(W=None), dict(down=None),
                                 dict(up=None), dict(ids=None), dict(ldx=7), dict(ldw=7), dict(ldc=7), dict(ldd=7),
                                 dict(sd=63), dict(ldu=7), dict(su=63), dict(up=P + 1), dict(ids=P + 2),
                                 dict(scale=P + 2)], ids=str)
def test_lora_invalid_arguments(bad):
    assert _lora(**bad) == _capi.GEMM_ERR_INVALID_ARG


def test_lora_limits_and_workspace():
    head = LIB.gemm_workspace_counter_bytes()
    assert _lora(R=1025, ldd=1025, sd=1 << 20, su=1 << 20) == _capi.GEMM_ERR_UNSUPPORTED
    assert _lora() == _capi.GEMM_ERR_WORKSPACE
    assert _lora(T=0) == _capi.GEMM_OK
    ws = LIB.gemm_lora_workspace_bytes
    # h of 100 rows x 16 ranks in fp32
    assert ws(P, P, P, 100, 64, 64, 2, 8, 64, 64, 0, 64, 512, 0) == head + 100 * 16 * 4
    # up with rows of 6 elements is copied to 64
    assert (ws(P, P, P, 100, 64, 64, 2, 6, 64, 64, 0, 6, 384, 1) - ws(P, P, P, 100, 64, 64, 2, 6, 64, 64, 0, 64, 384, 0)
            == 2 * 64 * 128)


def test_lora_refuses_cpu_tensors():
    z = lambda *s: torch.zeros(s, dtype=torch.float16)   # noqa: E731
    with pytest.raises(RuntimeError, match="x must be CUDA tensor"):
        ext.lora_gemm(z(4, 8), z(8, 8), z(2, 8, 4), z(2, 4, 8), torch.zeros(4, dtype=torch.int32))
