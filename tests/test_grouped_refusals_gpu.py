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


def test_out_that_shares_memory_through_another_pitch(ext):
    """Refused by the elements that meet, whatever the layouts; rows that lie between each other's are fine."""
    off, T = counts_to_offsets([10, 20, 30]), 60
    buf = randn((66 * 512,), torch.float16, 1)
    rows = lambda at, pitch, n=64: buf.as_strided((T, n), (pitch, 1), at)   # noqa: E731
    B, ids = stacked(3, 64, 64, torch.float16, 2), torch.zeros(T, dtype=torch.int32, device="cuda")
    W, down, up = B[0], stacked(2, 64, 8, torch.float16, 3), stacked(2, 8, 64, torch.float16, 4)
    G = randn((T, 16), torch.float16, 5)
    numbers = torch.zeros(2048, dtype=torch.int32, device="cuda")
    numbers[:4] = off
    as_out = numbers.view(torch.float16)[:4096 - 4096 % 64].view(-1, 64)
    for call in (lambda: ext.grouped_gemm(rows(0, 96), B, off, out=rows(10, 128)),
                 lambda: ext.grouped_gemm(rows(0, 512), B, off, out=rows(32, 256)),
                 lambda: ext.grouped_gemm(rows(0, 512), buf.as_strided((3, 64, 64), (64 * 128, 128, 1), 40), off,
                                          out=rows(64, 256)),
                 lambda: ext.grouped_gemm(rows(0, 512), B, off, bias=buf.as_strided((3, 64), (512, 2), 65),
                                          out=rows(64, 512)),
                 lambda: ext.grouped_gemm(rows(0, 64).t().t(), B, off, out=rows(30, 65)),
                 lambda: ext.lora_gemm(rows(0, 512), W, down, up, ids, bias=buf[600:664], out=rows(64, 256)),
                 lambda: ext.lora_gemm(rows(0, 512), W, buf.as_strided((2, 64, 8), (8, 512, 1), 65), up, ids,
                                       out=rows(64, 512)),
                 lambda: ext.grouped_gemm_wgrad(G, buf.as_strided((T, 16), (500, 1), 3), off,
                                                out=buf.as_strided((3, 16, 16), (6000, 300, 1), 0)),
                 lambda: ext.grouped_gemm(rows(0, 512)[:64], B, numbers[:4], out=as_out[:T])):
        with pytest.raises(RuntimeError, match="share memory"):
            call()
    for x, out in ((rows(0, 512), rows(64, 256)), (rows(64, 256), rows(0, 512)), (rows(0, 512), rows(448, 512))):
        want = ext.grouped_gemm(x.clone(), B, off)
        assert torch.equal(ext.grouped_gemm(x, B, off, out=out), want)
    # out's rows are the elements 576..639 and 832..895: 700..763 lie between them
    want = ext.lora_gemm(rows(0, 512).clone(), W, down, up, ids, bias=buf[700:764].clone())
    assert torch.equal(ext.lora_gemm(rows(0, 512), W, down, up, ids, bias=buf[700:764], out=rows(64, 256)), want)
    weights = buf.as_strided((3, 64, 64), (64 * 128, 128, 1), 0)
    weights.copy_(B)
    out = buf.as_strided((T, 64), (256, 1), 64)   # beside the weights' columns
    want = ext.grouped_gemm(G.repeat(1, 4), B, off)
    assert torch.equal(ext.grouped_gemm(G.repeat(1, 4), weights, off, out=out), want)
    between = buf.as_strided((3, 64, 16), (6400, 100, 1), 64)   # a gradient between the rows of an operand
    x = buf.as_strided((T, 64), (100, 1), 0)
    want = ext.grouped_gemm_wgrad(x.clone(), G, off)
    assert torch.equal(ext.grouped_gemm_wgrad(x, G, off, out=between), want)
