"""The calls around the products whose weight is picked by the row: operands that share memory, several threads, a
first call inside a capture, element counts past 32 bits."""
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from grouped_helpers import check, counts_to_offsets, randn, ref_grouped, ref_lora, stacked

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    from infinite_dreams import infinite_dreams_ext as ext
    yield
    torch.cuda.synchronize()
    ext.check_device_errors()


@pytest.fixture(params=["compiled", "ctypes"])
def ext(request, cuda_device):
    from infinite_dreams import infinite_dreams_ext
    keep = infinite_dreams_ext._fast
    if request.param == "ctypes":
        infinite_dreams_ext._fast = None
    yield infinite_dreams_ext
    infinite_dreams_ext._fast = keep


def test_out_that_shares_memory(ext):
    off = counts_to_offsets([10, 20, 30])
    buf = randn((60, 128), torch.float16, 1)
    B = stacked(3, 64, 64, torch.float16, 2)
    left, right = buf[:, :64], buf[:, 64:]
    want = ext.grouped_gemm(left, B, off)
    ext.grouped_gemm(left, B, off, out=right)   # columns of one buffer that do not meet
    assert torch.equal(right, want)
    x = left.contiguous()
    ids = torch.zeros(60, dtype=torch.int32, device="cuda")
    W, down, up = B[0], stacked(2, 64, 8, torch.float16, 3), stacked(2, 8, 64, torch.float16, 4)
    G = randn((60, 16), torch.float16, 5)
    for call in (lambda: ext.grouped_gemm(left, B, off, out=buf[:, 32:96]),
                 lambda: ext.grouped_gemm(x, B, off, out=x),
                 lambda: ext.grouped_gemm(x, B, off, out=B.view(-1)[:60 * 64].view(60, 64)),
                 lambda: ext.grouped_gemm_wgrad(G, G.clone(), off, out=G.view(-1)[:768].view(3, 16, 16)),
                 lambda: ext.lora_gemm(x, W, down, up, ids, out=x),
                 lambda: ext.lora_gemm(left, W, down, up, ids, out=buf[:, 63:127])):
        with pytest.raises(RuntimeError, match="share memory"):
            call()


def test_out_that_takes_part_in_autograd(ext):
    """A given out may not ask for gradients, and a graph that saved it notices the write."""
    off = counts_to_offsets([10, 20])
    A, B = randn((30, 64), torch.float16, 1), stacked(2, 64, 64, torch.float16, 2)
    out = torch.zeros(30, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(RuntimeError, match="no gradients"):
        ext.grouped_gemm(A, B, off, out=out.clone().requires_grad_())
    w = torch.ones(30, 64, dtype=torch.float16, device="cuda", requires_grad=True)
    y = (w * out).sum()
    ext.grouped_gemm(A, B, off, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_inference_mode(ext):
    """Weights that ask for gradients and a preallocated out, as a server holds them."""
    off = counts_to_offsets([10, 20])
    A, B = randn((30, 64), torch.float16, 1), stacked(2, 64, 64, torch.float16, 2).requires_grad_()
    W, down, up = (torch.nn.Parameter(w) for w in (randn((64, 64), torch.float16, 3, 0.1),
                                                   stacked(2, 64, 8, torch.float16, 4),
                                                   stacked(2, 8, 64, torch.float16, 5)))
    ids = (torch.arange(30, device="cuda") % 3 - 1).int()
    plain = torch.empty(30, 64, dtype=torch.float16, device="cuda")
    with torch.inference_mode():
        made = torch.empty_like(plain)
        want = ext.grouped_gemm(A, B, off)
        for out in (plain, made):
            assert torch.equal(ext.grouped_gemm(A, B, off, out=out), want)
            assert torch.equal(ext.lora_gemm(A, W, down, up, ids, out=out), ext.lora_gemm(A, W, down, up, ids))
        ext.grouped_gemm_wgrad(A, A, off, out=torch.empty(2, 64, 64, dtype=torch.float16, device="cuda"))


def test_several_threads(ext):
    """Four threads train and serve on one stream, with operands that are repacked: every pass gives the same bits."""
    from infinite_dreams.grouped import grouped_linear
    off = counts_to_offsets([10, 190, 50, 50])
    wrong = []

    def work(i):
        x = randn((300, 257), torch.bfloat16, i).requires_grad_()
        weight = stacked(4, 257, 511, torch.bfloat16, 10 + i).requires_grad_()
        W, down, up = randn((257, 511), torch.bfloat16, 20 + i, 0.1), *(
            stacked(3, *s, torch.bfloat16, 30 + i) for s in ((257, 8), (8, 511)))
        ids = (torch.arange(300, device="cuda") % 4 - 1).int()
        dy, first = randn((300, 511), torch.bfloat16, 40 + i), None
        for _ in range(40):
            y = grouped_linear(x, weight, off)
            dx, dw = torch.autograd.grad(y, (x, weight), dy)
            with torch.no_grad():
                z = ext.lora_gemm(x, W, down, up, ids)
            got = (y.detach(), dx, dw, z)
            first = first or got
            if not all(torch.equal(a, b) for a, b in zip(first, got)):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []


FIRST_CALL = """
import torch
from grouped_helpers import check, counts_to_offsets, randn, ref_grouped, ref_lora, stacked
from infinite_dreams import infinite_dreams_ext as ext
dt = torch.float16
off, ids = counts_to_offsets([10, 0, 190, 50]), (torch.arange(250, device="cuda") % 4 - 1).int()
A, B, C, D = randn((250, 256), dt, 1), stacked(4, 256, 512, dt, 2), randn((250, 257), dt, 3), stacked(4, 257, 511, dt, 4)
W, down, up = randn((256, 512), dt, 5, 0.1), stacked(3, 256, 8, dt, 6), stacked(3, 8, 512, dt, 7)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y, z = ext.grouped_gemm(A, B, off), ext.grouped_gemm(C, D, off)
    w, v = ext.grouped_gemm_wgrad(A, y, off), ext.lora_gemm(A, W, down, up, ids)
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
check(y, *ref_grouped(A, B, off))
check(z, *ref_grouped(C, D, off))
check(v, *ref_lora(A, W, down, up, ids))
assert torch.equal(w, ext.grouped_gemm_wgrad(A, y, off))
ext.check_device_errors()
"""


def test_first_call_of_a_process_inside_a_capture(cuda_device):
    here = Path(__file__).resolve().parent
    path = [str(here), str(here.parent / "infinite-dreams_b200")]
    code = f"import sys; sys.path[:0] = {path!r}\n" + FIRST_CALL
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_more_than_2_to_the_31_elements_of_rows(cuda_device):
    from infinite_dreams import infinite_dreams_ext as ext
    T, K, N = 70001, 64, 32768
    A, B = randn((T, K), torch.bfloat16, 1), stacked(3, K, N, torch.bfloat16, 2)
    first = [0, 5, 40000, T - 3]
    off = torch.tensor(first, device="cuda")
    out = ext.grouped_gemm(A, B, off)
    for r, e in ((0, 0), (39990, 1), (T - 200, 2)):   # 5 rows of each
        check(out[r:r + 5], *ref_grouped(A[r:r + 5], B[e:e + 1], counts_to_offsets([5])), f"rows from {r}")
    assert not out[T - 3:].any()
    w = ext.grouped_gemm_wgrad(A, out, off)
    few = torch.tensor([0, T - 3 - first[2]], device="cuda")
    assert torch.equal(w[2:, :, -64:], ext.grouped_gemm_wgrad(A[40000:], out[40000:, -64:], few))


def test_stacks_of_more_than_2_to_the_32_elements(cuda_device):
    from infinite_dreams import infinite_dreams_ext as ext
    E, K, N = 70, 4096, 16384
    B = torch.zeros(E, K, N, dtype=torch.bfloat16, device="cuda")
    B[69] = randn((K, N), torch.bfloat16, 1, K ** -0.5)
    A, G, off = randn((E, K), torch.bfloat16, 2), randn((E, N), torch.bfloat16, 3), torch.arange(E + 1, device="cuda")
    out = ext.grouped_gemm(A, B, off)
    check(out[69:], *ref_grouped(A[69:], B[69:], counts_to_offsets([1])))
    assert not out[:69].any()
    ext.grouped_gemm_wgrad(A, G, off, out=B)
    for e in (0, 69):   # a product of two 16-bit numbers, rounded once
        assert torch.equal(B[e], (A[e].double()[:, None] * G[e].double()).to(torch.bfloat16))


@pytest.mark.parametrize("T", [7, 600])
def test_adapters_past_2_to_the_31_elements(cuda_device, T):
    from infinite_dreams import infinite_dreams_ext as ext
    L, R, K, N = 40000, 16, 4096, 4096
    used = (0, 39999, 33333)
    down = torch.zeros(L, K, R, dtype=torch.bfloat16, device="cuda")
    up = torch.zeros(L, R, N, dtype=torch.bfloat16, device="cuda")
    for i, a in enumerate(used):
        down[a], up[a] = randn((K, R), torch.bfloat16, i, K ** -0.5), randn((R, N), torch.bfloat16, 5 + i)
    x, W = randn((T, K), torch.bfloat16, 9), randn((K, N), torch.bfloat16, 10, K ** -0.5)
    pick = torch.arange(T, device="cuda") % 4 - 1
    ids = torch.tensor([-1, *used], device="cuda")[pick + 1]
    out = ext.lora_gemm(x, W, down, up, ids)
    check(out, *ref_lora(x, W, down[list(used)], up[list(used)], pick))
