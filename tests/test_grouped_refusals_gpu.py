"""Calls of the grouped and adapted products that are refused because their result would be wrong."""
import pytest
import torch
from torch.autograd import forward_ad

from grouped_helpers import counts_to_offsets, randn, stacked

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["compiled", "ctypes"])
def ext(request, cuda_device):
    from infinite_dreams import infinite_dreams_ext
    keep = infinite_dreams_ext._fast
    if request.param == "ctypes":
        infinite_dreams_ext._fast = None
    yield infinite_dreams_ext
    infinite_dreams_ext._fast = keep
    torch.cuda.synchronize()
    infinite_dreams_ext.check_device_errors()


def test_forward_mode_is_refused(ext):
    """No tangent is dropped in silence, under no_grad either; plain tensors inside a level are fine."""
    from infinite_dreams.grouped import grouped_linear
    off = counts_to_offsets([10, 20])
    A, B = randn((30, 64), torch.float16, 1), stacked(2, 64, 64, torch.float16, 2)
    W, down, up = B[0], stacked(2, 64, 8, torch.float16, 3), stacked(2, 8, 64, torch.float16, 4)
    ids, bias = torch.zeros(30, dtype=torch.int32, device="cuda"), randn((64,), torch.float16, 5)
    want = ext.grouped_gemm(A, B, off)
    with forward_ad.dual_level(), torch.no_grad():
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (A, B, bias)]
        for call in (lambda: ext.grouped_gemm(dual[0], B, off), lambda: ext.grouped_gemm(A, dual[1], off),
                     lambda: ext.grouped_gemm_wgrad(dual[0], A, off), lambda: ext.grouped_gemm_wgrad(A, dual[0], off),
                     lambda: ext.lora_gemm(dual[0], W, down, up, ids),
                     lambda: ext.lora_gemm(A, W, down, up, ids, bias=dual[2])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises((RuntimeError, NotImplementedError)):
            grouped_linear(dual[0], B, off)
        assert torch.equal(ext.grouped_gemm(A, B, off), want)
