"""lora_gemm over the whole range of values: inf and NaN in the weights of an adapter that owns its tile, and products
with `down` far from 1."""
import pytest
import torch

from grouped_helpers import DTYPES, check, randn, ref_lora, stacked

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    from infinite_dreams import infinite_dreams_ext as ext
    yield
    torch.cuda.synchronize()
    ext.check_device_errors()


@pytest.mark.parametrize("T", [1, 40, 300])
@pytest.mark.parametrize("ids", ["one", "one and none", "two"])
@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_infinite_weights_give_the_definition_whatever_the_neighbours(T, ids, stored, dtype, bad):
    """h * inf is +-inf by the sign of h and h * NaN is NaN, in the columns that hold one; the rest as without."""
    from infinite_dreams import infinite_dreams_ext as ext
    K, N, L, R = 64, 264, 3, 24
    # whole numbers: h is exact in 16 bits for every other rank (its second part is 0) and needs both for the others
    x = torch.randint(1, 3, (T, K), generator=torch.Generator().manual_seed(T)).to(dtype).cuda()
    down = torch.zeros(L, K, R, dtype=dtype, device="cuda")
    down[:, 0, :] = 1.0
    down[:, 1, 1::2] = 1.0 + torch.finfo(dtype).eps * 3
    down[:, :2, ::3] *= -1.0
    W, up = stacked(1, K, N, dtype, 1, stored)[0], stacked(L, R, N, dtype, 3, stored)
    if stored == "nk":
        down = down.transpose(1, 2).contiguous().transpose(1, 2)
    pick = torch.arange(T, device="cuda")
    pick = {"one": pick * 0 + 1, "one and none": torch.where(pick % 3 == 1, -1, 1), "two": 1 + pick % 2}[ids]
    clean = ext.lora_gemm(x, W, down, up, pick)
    for rank, cols in ((0, slice(3, 9)), (7, slice(130, 200)), (21, slice(250, 264))):
        up[1, rank, cols] = bad
    got = ext.lora_gemm(x, W, down, up, pick)
    mine, h = pick == 1, x.double() @ down[1].double()
    want = clean.clone()
    for rank, cols in ((0, slice(3, 9)), (7, slice(130, 200)), (21, slice(250, 264))):
        want[:, cols] = torch.where(mine[:, None], (h[:, rank] * bad)[:, None].to(dtype), want[:, cols])
    assert torch.equal(got.nan_to_num(7.5, 1e4, -1e4), want.nan_to_num(7.5, 1e4, -1e4))
