"""grouped_gemm_wgrad and grouped_linear: gradients against 64 bits, against differences, in graphs and together."""
import pytest
import torch

from grouped_helpers import DTYPES, check, counts_to_offsets, randn, ref_grouped, ref_wgrad, stacked

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    from infinite_dreams import infinite_dreams_ext as ext
    yield
    torch.cuda.synchronize()
    ext.check_device_errors()


# lengths around the 16-row steps and the 64-row stages, empty groups, long ones
COUNTS = [[1], [0, 0, 1], [15, 16, 17], [63, 64, 65, 0], [127, 1, 128], [49, 33, 400, 0, 1], [2000, 700], [64] * 9,
          [1] * 40]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c[:6])))
def test_wgrad_counts(counts, dtype):
    from infinite_dreams import infinite_dreams_ext as ext
    T = sum(counts)
    A, G, off = randn((T, 320), dtype, 1), randn((T, 264), dtype, 2), counts_to_offsets(counts, torch.int64)
    ref, tol = ref_wgrad(A, G, off)
    got = ext.grouped_gemm_wgrad(A, G, off)
    check(got, ref, tol)
    stored = torch.full((len(counts), 264, 320), float("nan"), dtype=dtype, device="cuda")
    out = ext.grouped_gemm_wgrad(A, G, off, out=stored.transpose(1, 2))
    assert out.data_ptr() == stored.data_ptr()
    check(stored.transpose(1, 2), ref, tol, "stored N x K")


@pytest.mark.parametrize("K,N", [(1, 1), (8, 520), (256, 256), (257, 255), (777, 1023), (72, 64), (1000, 24), (33, 2000)])
def test_wgrad_sizes(K, N):
    from infinite_dreams import infinite_dreams_ext as ext
    counts = [70, 0, 33, 200]
    A, G, off = randn((303, K), torch.float16, 1), randn((303, N), torch.float16, 2), counts_to_offsets(counts)
    ref, tol = ref_wgrad(A, G, off)
    check(ext.grouped_gemm_wgrad(A, G, off), ref, tol)


def test_wgrad_of_no_rows():
    from infinite_dreams import infinite_dreams_ext as ext
    A, G = randn((0, 100), torch.float16, 1), randn((0, 60), torch.float16, 2)
    assert torch.equal(ext.grouped_gemm_wgrad(A, G, torch.zeros(4, dtype=torch.int32, device="cuda")),
                       torch.zeros((3, 100, 60), dtype=torch.float16, device="cuda"))


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_other_rows_do_not_enter(bad):
    """inf and NaN in a neighbour's rows and behind the last group, whichever operand holds them."""
    from infinite_dreams import infinite_dreams_ext as ext
    for counts in ([17, 5, 30, 3], [64, 70, 1, 130]):
        T = sum(counts) + 9
        A, G, off = randn((T, 192), torch.bfloat16, 1), randn((T, 136), torch.bfloat16, 2), counts_to_offsets(counts)
        clean = ext.grouped_gemm_wgrad(A, G, off)
        A[counts[0]:counts[0] + counts[1]] = bad
        G[sum(counts[:3]):sum(counts)] = bad
        A[-9:], G[-9:] = bad, bad
        got = ext.grouped_gemm_wgrad(A, G, off)
        assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
        assert not bool(got[1].isfinite().any()) and not bool(got[3].isfinite().any())


def test_wgrad_strides():
    from infinite_dreams import infinite_dreams_ext as ext
    counts, dt = [40, 90], torch.bfloat16
    off = counts_to_offsets(counts)
    big_a, big_g = randn((130, 300), dt, 1), randn((130, 301), dt, 2)
    given = torch.full((2, 150, 400), 5.0, dtype=dt, device="cuda")
    for A, G, out in [(big_a[:, 16:144], big_g[:, :200], None), (big_a[:, 3:131], big_g[:, 1:201], None),
                      (randn((128, 130), dt, 3).t(), big_a[:1, :200].expand(130, 200), None),
                      (big_a[:, :128], big_a[:, 8:208], given[:, 8:136, 16:216]),
                      (big_a[:, :128], big_a[:, 8:208], given[:, 8:136, 3:203])]:
        ref, tol = ref_wgrad(A, G, off)
        check(ext.grouped_gemm_wgrad(A, G, off, out=out), ref, tol)
    assert bool((given[:, :8] == 5).all()) and bool((given[:, 136:] == 5).all())
    assert bool((given[:, :, :3] == 5).all()) and bool((given[:, :, 216:] == 5).all())
    with pytest.raises(RuntimeError, match="row-major or a transposed view"):
        ext.grouped_gemm_wgrad(A, G, off, out=torch.empty((128, 200, 2), dtype=dt, device="cuda").permute(2, 0, 1))


def test_wgrad_is_the_same_from_call_to_call():
    from infinite_dreams import infinite_dreams_ext as ext
    A, G, off = randn((1000, 512), torch.float16, 1), randn((1000, 768), torch.float16, 2), counts_to_offsets([900, 100])
    first = ext.grouped_gemm_wgrad(A, G, off)
    assert all(torch.equal(first, ext.grouped_gemm_wgrad(A, G, off)) for _ in range(5))


def test_wgrad_both_bindings_give_the_same_bits():
    from infinite_dreams import infinite_dreams_ext as ext
    A, G, off = randn((100, 77), torch.float16, 1), randn((100, 80), torch.float16, 2), counts_to_offsets([60, 40])
    out = torch.empty((2, 80, 77), dtype=torch.float16, device="cuda").transpose(1, 2)
    fast = ext.grouped_gemm_wgrad(A, G, off), ext.grouped_gemm_wgrad(A, G, off, out=out).clone()
    keep, ext._fast = ext._fast, None
    try:
        slow = ext.grouped_gemm_wgrad(A, G, off), ext.grouped_gemm_wgrad(A, G, off, out=out)
    finally:
        ext._fast = keep
    assert all(torch.equal(f, s) for f, s in zip(fast, slow))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("stored", ["kn", "nk"])
def test_linear_gradients(stored, dtype):
    """y, dx and dweight of a step with empty groups and rows of no group; the gradient has its weight's strides."""
    from infinite_dreams.grouped import grouped_linear
    counts, K, N = [100, 0, 37, 260], 200, 328
    T = sum(counts) + 20
    off = counts_to_offsets(counts)
    x, W = randn((T, K), dtype, 1).requires_grad_(), stacked(4, K, N, dtype, 2, stored).requires_grad_()
    dy = randn((T, N), dtype, 3)
    y = grouped_linear(x, W, off)
    dx, dW = torch.autograd.grad(y, (x, W), dy)
    with torch.no_grad():
        check(y, *ref_grouped(x, W, off), "y")
        check(dx, *ref_grouped(dy, W.transpose(1, 2), off), "dx")
        check(dW, *ref_wgrad(x, dy, off), "dW")
    assert dW.stride() == W.stride()


def test_linear_against_differences():
    """The function is linear in each input, so a central difference of any width is the derivative, up to the
    rounding of the two outputs."""
    from infinite_dreams import infinite_dreams_ext as ext
    from infinite_dreams.grouped import grouped_linear
    counts, K, N, dt = [40, 0, 25], 96, 120, torch.float16
    off = counts_to_offsets(counts)
    x, W = randn((65, K), dt, 1).requires_grad_(), stacked(3, K, N, dt, 2).requires_grad_()
    dy = randn((65, N), dt, 3)
    dx, dW = torch.autograd.grad(grouped_linear(x, W, off), (x, W), dy)
    with torch.no_grad():
        for leaf, grad, other in ((x, dx, lambda v: (v, W)), (W, dW, lambda v: (x, v))):
            step = randn(tuple(leaf.shape), dt, 4, 0.25)
            plus, minus = (leaf + step).detach(), (leaf - step).detach()     # fp16 values: the step is their difference
            width = plus.double() - minus.double()
            ends = [ext.grouped_gemm(*other(v), off).double() for v in (plus, minus)]
            difference = float(((ends[0] - ends[1]) * dy.double()).sum())
            along = float((grad.double() * width).sum())
            # each output and each gradient value is within its bound of the exact one
            bounds = sum(float((ref_grouped(*other(v), off)[1] * dy.double().abs()).sum()) for v in (plus, minus))
            g_tol = (ref_grouped(dy, W.transpose(1, 2), off) if leaf is x else ref_wgrad(x, dy, off))[1]
            assert abs(difference - along) <= bounds + float((g_tol * width.abs()).sum())


def test_linear_asks_only_for_what_is_needed():
    from infinite_dreams.grouped import grouped_linear
    off = counts_to_offsets([5, 6])
    x, W = randn((11, 64), torch.float16, 1), stacked(2, 64, 72, torch.float16, 2)
    (dW,) = torch.autograd.grad(grouped_linear(x, W.requires_grad_(), off).sum(), W)     # dy is expanded
    check(dW, *ref_wgrad(x, torch.ones(11, 72, dtype=torch.float16, device="cuda"), off))
    W = W.detach()
    (dx,) = torch.autograd.grad(grouped_linear(x.requires_grad_(), W, off).sum(), x)
    check(dx, *ref_grouped(torch.ones(11, 72, dtype=torch.float16, device="cuda"), W.transpose(1, 2), off))


def test_raw_operators_refuse_gradients():
    from infinite_dreams import infinite_dreams_ext as ext
    off = counts_to_offsets([5, 6])
    x, W = randn((11, 64), torch.float16, 1).requires_grad_(), stacked(2, 64, 72, torch.float16, 2)
    with pytest.raises(RuntimeError, match="grouped_linear"):
        ext.grouped_gemm(x, W, off)
    with torch.no_grad():
        ext.grouped_gemm(x, W, off)


def _expert_block(x, W1, W2, off):
    from infinite_dreams.grouped import grouped_linear
    return grouped_linear(torch.relu(grouped_linear(x, W1, off)), W2, off)


def test_an_expert_block_trains_like_its_formula():
    """Two products with a ReLU between them, forward and backward, as one uses them."""
    counts, K, H, dt = [70, 0, 130, 9], 128, 320, torch.bfloat16
    off = counts_to_offsets(counts)
    x = randn((209, K), dt, 1).requires_grad_()
    W1, W2 = (stacked(4, *s, dt, i).requires_grad_() for i, s in ((2, (K, H)), (3, (H, K))))
    dy = randn((209, K), dt, 4)
    y = _expert_block(x, W1, W2, off)
    dx, dW1, dW2 = torch.autograd.grad(y, (x, W1, W2), dy)
    with torch.no_grad():
        # the formula, with h and dh rounded where the block rounds them.  What is left: the roundings of the results
        # (2^-8 of each value), and values of h and dh that the block rounds to the neighbour or to the other side of 0
        # because its sums err in the last bits of fp32, which moves few of them by one step (2^-7 of a value)
        h_ref, _ = ref_grouped(x, W1, off)
        h = torch.relu(h_ref).to(dt)
        dh_ref, _ = ref_grouped(dy, W2.transpose(1, 2), off)
        mask = h_ref > 0
        dh = (dh_ref * mask).to(dt)
        for got, ref in ((y, ref_grouped(h, W2, off)[0]), (dW2, ref_wgrad(h, dy, off)[0]),
                         (dx, ref_grouped(dh, W1.transpose(1, 2), off)[0]), (dW1, ref_wgrad(x, dh, off)[0])):
            assert float((got.double() - ref).norm() / ref.norm()) <= 2.0 ** -8 + 2.0 ** -7


def test_a_step_captured_and_replayed():
    """Forward and backward of the block in one graph, replayed with new values and new counts."""
    K, H, dt = 128, 192, torch.float16
    off = counts_to_offsets([100, 28, 72])
    x = randn((200, K), dt, 1).requires_grad_()
    W1, W2 = (stacked(3, *s, dt, i).requires_grad_() for i, s in ((2, (K, H)), (3, (H, K))))
    dy = randn((200, K), dt, 4)

    def step():
        return torch.autograd.grad(_expert_block(x, W1, W2, off), (x, W1, W2), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for counts, seed in (([100, 28, 72], 1), ([0, 190, 3], 5)):
        off.copy_(counts_to_offsets(counts))
        x.data.copy_(randn((200, K), dt, seed))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), counts


def test_linear_in_both_bindings():
    """The compiled function and the one in Python: the same bits, the same refusal of a second derivative."""
    from infinite_dreams import infinite_dreams_ext as ext
    from infinite_dreams.grouped import grouped_linear
    off = counts_to_offsets([30, 0, 50])
    x, W = randn((80, 72), torch.bfloat16, 1).requires_grad_(), stacked(3, 72, 88, torch.bfloat16, 2).requires_grad_()
    dy = randn((80, 88), torch.bfloat16, 3)

    def step():
        y = grouped_linear(x, W, off)
        return (y.detach(), *torch.autograd.grad(y, (x, W), dy))

    def twice():
        dx, = torch.autograd.grad(grouped_linear(x, W, off), x, dy.requires_grad_(), create_graph=True)
        torch.autograd.grad(dx.sum(), W)

    fast = step()
    with pytest.raises(RuntimeError):
        twice()
    keep, ext._fast = ext._fast, None
    try:
        slow = step()
        with pytest.raises(RuntimeError):
            twice()
    finally:
        ext._fast = keep
    assert all(torch.equal(f, s) for f, s in zip(fast, slow))
    with torch.no_grad():
        assert not grouped_linear(x, W, off).requires_grad


def test_weights_as_parameters_of_a_module():
    """Gradients accumulate into .grad over two backward passes, as an optimizer reads them."""
    from infinite_dreams.grouped import grouped_linear
    off = counts_to_offsets([20, 44])
    W = torch.nn.Parameter(stacked(2, 64, 96, torch.float16, 1))
    x, dy = randn((64, 64), torch.float16, 2), randn((64, 96), torch.float16, 3)
    grouped_linear(x, W, off).backward(dy)
    once = W.grad.clone()
    grouped_linear(x, W, off).backward(dy)
    assert torch.equal(W.grad, once + once)
