"""The ends of the ranges that the grouped and adapted products take."""
import pytest

from infinite_dreams import _capi
from test_grouped_cpu import LIB, _launch, _lora, _wgrad


@pytest.mark.parametrize("n", [(1 << 31) - 1, (1 << 31) - 1023])
def test_extents_that_do_not_round_up_in_32_bits(n):
    """Rows and columns are rounded up to whole tiles in 32 bits: what would overflow is refused."""
    for call in (lambda: _launch(T=n), lambda: _launch(N=n, ldb=n, ldc=n, sb=8 * n), lambda: _launch(K=n, lda=n, sb=8 * n),
                 lambda: _wgrad(T=n), lambda: _wgrad(M=n, lda=n, sd=8 * n), lambda: _wgrad(N=n, ldg=n, ldd=n, sd=8 * n),
                 lambda: _lora(T=n), lambda: _lora(N=n, ldw=n, ldu=n, ldc=n, su=8 * n),
                 lambda: _lora(K=n, ldx=n, sd=8 * n)):
        assert call() == _capi.GEMM_ERR_UNSUPPORTED
        assert b"2^31 - 1024" in LIB.gemm_last_error()
    # the largest that is taken goes on to the next check (the workspace, then the device)
    assert _launch(T=n - 1024, K=7, lda=7) == _capi.GEMM_ERR_WORKSPACE
