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
