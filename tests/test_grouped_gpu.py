"""grouped_gemm against a 64-bit reference, at the sizes, strides and groups where it can go wrong."""
import pytest
import torch

from grouped_helpers import DTYPES, check, counts_to_offsets, randn, ref_grouped, stacked

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    from infinite_dreams import infinite_dreams_ext as ext
    yield
    torch.cuda.synchronize()
    ext.check_device_errors()


def _run(counts, K, N, dtype, stored="kn", bias=False, act="none", spare=0, first=0, index=torch.int32, seed=1):
    from infinite_dreams import infinite_dreams_ext as ext
    T, E = first + sum(counts) + spare, len(counts)
    A, B = randn((T, K), dtype, seed), stacked(E, K, N, dtype, seed + 1, stored)
    b = randn((E, N), dtype, seed + 2, 0.5) if bias else None
    off = counts_to_offsets(counts, index, first)
    out = ext.grouped_gemm(A, B, off, bias=b, activation=act)
    ref, tol = ref_grouped(A, B, off, b, act)
    check(out, ref, tol, f"{counts} {K}x{N}")
    return A, B, b, off, out


# one row, empty groups, groups around the 16/32-row steps, the 64- and 256-row tiles and the 32-row chunks
COUNTS = [[1], [0, 1, 0], [0, 0], [16, 17, 15, 1], [63, 64, 65], [31, 33, 0, 32], [256, 257, 255],
          [600, 1, 0, 97, 513], [1000, 3]]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c)))
def test_counts(counts, stored, dtype):
    _run(counts, 192, 384, dtype, stored, index=torch.int64 if len(counts) % 2 else torch.int32)


@pytest.mark.parametrize("K,N", [(1, 1), (8, 8), (64, 128), (72, 136), (777, 1023), (96, 129), (1000, 127), (2048, 256),
                                 (33, 520)])
@pytest.mark.parametrize("counts", [[3, 0, 40], [300, 90]], ids=["few", "many"])
@pytest.mark.parametrize("stored", ["kn", "nk"])
def test_sizes(K, N, counts, stored):
    _run(counts, K, N, torch.float16, stored, bias=True, act="relu")


@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
@pytest.mark.parametrize("counts", [[5, 9], [200, 400]], ids=["few", "many"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_epilogue(act, counts, dtype):
    _run(counts, 320, 264, dtype, "nk", bias=True, act=act)


@pytest.mark.parametrize("counts,N", [
    ([8192], 4096), ([3001, 0, 257, 4100], 4096), ([5000, 3400], 4096), ([2000, 0, 5600, 500, 1093], 4096),
    ([1100, 5700, 1400], 4120), ([9000, 257, 30], 4000), ([2560, 5120, 1], 5001)], ids=str)
@pytest.mark.parametrize("stored,dtype", [("kn", torch.float16), ("nk", torch.bfloat16)])
def test_tall_tiles(counts, N, stored, dtype):
    """Large groups: two row parts to a tile, one, and last waves done part by part (or not)."""
    _run(counts, 136, N, dtype, stored, bias=True, act="gelu", first=3, spare=5)
    _run(counts, 1000, N, dtype, stored)


def test_tall_tiles_without_reduction():
    from infinite_dreams import infinite_dreams_ext as ext
    b = randn((2, 4096), torch.float16, 1)
    out = ext.grouped_gemm(torch.empty(8192, 0, dtype=torch.float16, device="cuda"),
                           torch.empty(2, 0, 4096, dtype=torch.float16, device="cuda"),
                           counts_to_offsets([3000, 5192]), bias=b)
    assert torch.equal(out[:3000], b[:1].expand(3000, -1)) and torch.equal(out[3000:], b[1:].expand(5192, -1))


def test_no_reduction():
    """K = 0: act(bias) in the rows of the groups."""
    _run([3, 0, 70], 0, 200, torch.bfloat16, bias=True, act="gelu")
    _run([300, 90], 0, 264, torch.float16)


@pytest.mark.parametrize("counts", [[2] * 128, [0] * 500 + [7] * 12 + [0] * 512, [1] * 1024, [40] * 100],
                         ids=["128", "mostly empty", "1024", "100 of 40"])
def test_many_groups(counts):
    _run(counts, 128, 192, torch.bfloat16)


@pytest.mark.parametrize("counts", [[3, 5], [300, 200]], ids=["few", "many"])
@pytest.mark.parametrize("N", [256, 260, 261])
def test_rows_outside_the_groups(counts, N):
    """Rows before the first and behind the last group: zero in a new output, untouched in a given one."""
    from infinite_dreams import infinite_dreams_ext as ext
    A, B, _, off, out = _run(counts, 128, N, torch.float16, spare=37, first=11)
    given = torch.full((A.shape[0], N + 11), 7.0, dtype=A.dtype, device="cuda")
    ext.grouped_gemm(A, B, off, out=given[:, :N])
    assert torch.equal(given[11:-37, :N], out[11:-37])
    assert bool((given[:11] == 7).all()) and bool((given[-37:] == 7).all()) and bool((given[:, N:] == 7).all())


@pytest.mark.parametrize("counts", [[3, 5, 2], [300, 70, 200]], ids=["few", "many"])
def test_other_groups_values_do_not_spread(counts):
    """inf and NaN in one group's rows or weights, and behind the last row, stay there."""
    from infinite_dreams import infinite_dreams_ext as ext
    K, N = 100, 200
    T = sum(counts) + 5
    A, B, off = randn((T, K), torch.float16, 1), stacked(3, K, N, torch.float16, 2), counts_to_offsets(counts)
    clean = ext.grouped_gemm(A, B, off)
    rows = slice(counts[0], counts[0] + counts[1])
    A[rows] = float("nan")
    A[-5:] = float("inf")
    B[1] = float("inf")
    got = ext.grouped_gemm(A, B, off)
    assert bool(got[rows].isnan().all())
    got[rows] = clean[rows] = 0
    assert torch.equal(got, clean)


@pytest.mark.parametrize("counts", [[9, 20], [300, 100]], ids=["few", "many"])
def test_strides(counts):
    """Rows with a pitch, stacked weights cut out of larger ones, unaligned bases, expanded and permuted weights."""
    from infinite_dreams import infinite_dreams_ext as ext
    K, N, T, dt = 136, 144, sum(counts), torch.bfloat16
    off = counts_to_offsets(counts)
    big_a, big_b = randn((T, K + 24), dt, 3), randn((4, K + 8, N + 40), dt, 4, 0.1)
    odd_a, odd_b = randn((T * (K + 1) + 1,), dt, 5), randn((2 * K * N + 1,), dt, 6, 0.1)
    for A, B in [(big_a[:, 8:8 + K], big_b[1:3, :K, 32:32 + N]),
                 (big_a[:, 3:3 + K], big_b[::2, 1:1 + K, 7:7 + N]),
                 (odd_a[1:].view(T, K + 1)[:, :K], odd_b[1:].view(2, K, N)),
                 (randn((K, T), dt, 7).t(), odd_b[1:].view(2, N, K).transpose(1, 2)),
                 (big_a[:1, :K].expand(T, K), big_b[:1, :K, :N].expand(2, K, N)),
                 (big_a[:, :K], randn((K, 2, N), dt, 8, 0.1).transpose(0, 1)),
                 (big_a[:, :K], randn((K, N, 2), dt, 9, 0.1).permute(2, 0, 1))]:
        ref, tol = ref_grouped(A, B, off)
        check(ext.grouped_gemm(A, B, off), ref, tol, f"{A.stride()} {B.stride()}")


def test_input_gradient_is_the_transposed_product():
    from infinite_dreams import infinite_dreams_ext as ext
    counts = [130, 0, 70]
    dy, B, off = randn((200, 264), torch.float16, 1), stacked(3, 520, 264, torch.float16, 2), counts_to_offsets(counts)
    ref, tol = ref_grouped(dy, B.transpose(1, 2), off)
    check(ext.grouped_gemm(dy, B.transpose(1, 2), off), ref, tol)


def test_bad_offsets_are_clamped_and_reported():
    """Decreasing or outside offsets: no access leaves the operands, other groups are right, the host learns of it."""
    from infinite_dreams import infinite_dreams_ext as ext
    K, N, T = 128, 256, 100
    A, B = randn((T, K), torch.float16, 1), stacked(3, K, N, torch.float16, 2)
    for bad, read_as in [([0, 40, 20, 100], [0, 40, 40, 100]), ([-5, 40, 50, 1000], [0, 40, 50, 100])]:
        out = ext.grouped_gemm(A, B, torch.tensor(bad, device="cuda"))
        ref, tol = ref_grouped(A, B, torch.tensor(read_as))
        check(out, ref, tol, str(bad))
        with pytest.raises(RuntimeError, match="group offsets"):
            ext.check_device_errors()


def test_both_bindings_give_the_same_bits():
    from infinite_dreams import infinite_dreams_ext as ext
    A, B = randn((90, 100), torch.bfloat16, 1), stacked(3, 100, 201, torch.bfloat16, 2, "nk")
    off, b = counts_to_offsets([30, 0, 55]), randn((3, 201), torch.bfloat16, 3)
    fast = ext.grouped_gemm(A, B, off, bias=b, activation="gelu")
    keep, ext._fast = ext._fast, None
    try:
        slow = ext.grouped_gemm(A, B, off, bias=b, activation="gelu")
    finally:
        ext._fast = keep
    assert torch.equal(fast.view(torch.int16), slow.view(torch.int16))


def test_other_stream_and_chained_calls():
    """Launches on a side stream and back to back, each reading the one before."""
    from infinite_dreams import infinite_dreams_ext as ext
    off = counts_to_offsets([50, 200, 6])
    B = stacked(3, 256, 256, torch.float16, 1)
    x0 = randn((256, 256), torch.float16, 2)

    def chain(sync):
        x = x0
        for _ in range(6):
            x = ext.grouped_gemm(x, B, off)
            if sync:
                torch.cuda.synchronize()
        return x

    want = chain(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain(False)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_two_graphs_replayed_at_once():
    """Two graphs captured on one stream (their operands are repacked into scratch), replayed on two, then with new
    offsets and values: every replay gives the eager bits."""
    from infinite_dreams import infinite_dreams_ext as ext
    K, N, T = 333, 777, 600
    A = [randn((T, K), torch.float16, i) for i in range(2)]
    B = [stacked(4, K, N, torch.float16, 10 + i) for i in range(2)]
    off = counts_to_offsets([100, 0, 300, 150])
    ext.grouped_gemm(A[0], B[0], off)
    torch.cuda.synchronize()
    graphs, outs, side = [], [], [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side[0]):
            outs.append(ext.grouped_gemm(A[i], B[i], off))
        graphs.append(g)
    for counts in ([100, 0, 300, 150], [7, 500, 3, 0]):
        off.copy_(counts_to_offsets(counts))
        want = [ext.grouped_gemm(A[i], B[i], off) for i in range(2)]
        for _ in range(5):
            torch.cuda.synchronize()
            for i in range(2):
                with torch.cuda.stream(side[i]):
                    graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(outs[i], want[i]) for i in range(2)), counts
        A[0].mul_(0.5)
