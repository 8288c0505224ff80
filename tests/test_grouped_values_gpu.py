"""grouped_gemm at the ends of the types' ranges and where padding lies beside the operands."""
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


@pytest.mark.parametrize("counts", [[5, 9], [200, 400], [2000, 6200]], ids=["few", "many", "tall"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_gelu_of_values_up_to_the_largest(counts, dtype):
    """gelu(x) = x for large finite x, 0 for their negatives, inf for inf, and NaN where 0 * inf or NaN stands."""
    from infinite_dreams import infinite_dreams_ext as ext
    T, N = sum(counts), 4096 if sum(counts) > 8000 else 264
    top = torch.finfo(dtype).max
    values = torch.tensor([top, -top, top * 0.75, -top * 0.51, top * 0.51, 1e4, -1e4, float("inf"), float("-inf"),
                           float("nan"), 2.0, -2.0], device="cuda").to(dtype)
    x = values.repeat(T // len(values) + 1)[:T]
    A, B = torch.zeros(T, 8, dtype=dtype, device="cuda"), torch.zeros(2, 8, N, dtype=dtype, device="cuda")
    A[:, 0] = 1.0
    b = torch.zeros(2, N, dtype=dtype, device="cuda")
    off = counts_to_offsets(counts)
    for v in values:
        b[:] = v
        got = ext.grouped_gemm(A, B, off, bias=b, activation="gelu")      # the value as the bias
        want = torch.nn.functional.gelu(v.double()).to(dtype)
        step = torch.finfo(dtype).eps * want.abs().float()                # small values: one rounding and the fit
        off_by = (got.float() - want.float()).abs()
        same = (got == want) | (got.isnan() & want.isnan()) | (off_by <= step)
        assert bool(same.all()), (float(v), got[0, 0].item(), want.item())
    A[:, 0], B[:, 0, :] = x, 1.0                                          # and as the products (0 * inf is in none)
    B[:, 1:, :], A[:, 1:] = 0.0, 0.0
    got = ext.grouped_gemm(A, B, off, activation="gelu")
    want = torch.nn.functional.gelu(x.double()).to(dtype)[:, None].expand(T, N)
    same = (got == want) | (got.isnan() & want.isnan()) | ((got.float() - want.float()).abs()
                                                           <= torch.finfo(dtype).eps * want.abs().float())
    assert bool(same.all())


def _padded(shape, rows, cols, dtype, seed, scale=1.0):
    """A tensor of this shape cut out of one with `rows` more rows and `cols` more columns, all of them NaN."""
    full = torch.full((*shape[:-2], shape[-2] + rows, shape[-1] + cols), float("nan"), dtype=dtype, device="cuda")
    part = full[..., :shape[-2], :shape[-1]]
    part.copy_(randn(shape, dtype, seed, scale))
    return part


@pytest.mark.parametrize("K,N", [(133, 141), (65, 129), (7, 263), (1029, 8), (1, 1)])
@pytest.mark.parametrize("counts", [[1], [9, 0, 20], [300, 0, 100], [1500, 6700]], ids=["one", "few", "many", "tall"])
@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_padding_does_not_enter(K, N, counts, stored, dtype):
    """NaN beside and below every operand whose pitch is aligned while its width is not."""
    from infinite_dreams import infinite_dreams_ext as ext
    T, E = sum(counts), len(counts)
    if T > 8000:
        N += 4000
    off = counts_to_offsets(counts)
    A = _padded((T, K), 3, -K % 8 + 8, dtype, 1)
    if stored == "kn":
        B = _padded((E, K, N), 2, -N % 8 + 8, dtype, 2, K ** -0.5)
    else:
        B = _padded((E, N, K), 2, -K % 8 + 8, dtype, 2, K ** -0.5).transpose(1, 2)
    check(ext.grouped_gemm(A, B, off), *ref_grouped(A, B, off))
    if T < 8000:
        G = _padded((T, N), 3, -N % 8 + 8, dtype, 3)
        check(ext.grouped_gemm_wgrad(A, G, off), *ref_wgrad(A, G, off))


# few rows: the bound on the tiles selects clusters of 2, 4 and 8 for the last (here the only) wave
@pytest.mark.parametrize("K", [1024, 2048, 4096, 8200])
@pytest.mark.parametrize("N", [129, 520, 1500])
@pytest.mark.parametrize("counts", [[1], [5, 0, 2], [33, 64]], ids=str)
@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_few_rows_with_the_sum_split_over_a_cluster(K, N, counts, act, dtype):
    from infinite_dreams import infinite_dreams_ext as ext
    A, B, b = randn((sum(counts), K), dtype, 1), stacked(len(counts), K, N, dtype, 2), randn((len(counts), N), dtype, 3)
    off = counts_to_offsets(counts)
    check(ext.grouped_gemm(A, B, off, bias=b, activation=act), *ref_grouped(A, B, off, b, act))
