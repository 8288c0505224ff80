"""lora_gemm over the whole range of values: inf and NaN in the weights of an adapter that owns its tile, and products
with `down` far from 1."""
import pytest
import torch

from grouped_helpers import DTYPES, check, half_step, randn, ref_lora, rounded, stacked, sum_error

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


def _bound(x, W, down, up, adapter, scale):
    """(reference, bound) with the same accuracy of h whatever its size: an fp32 sum, scaled, in two bf16 parts.

    The first part is off by at most 2^-8 of h (half a step), the rest is exact in fp32, and its own rounding is off by
    2^-8 of that: 2^-16 of h.  (Rounding to an infinite first part instead takes the largest finite one, 2^-8 off too.)
    The sums are bounded as in grouped_helpers.sum_error: 16 products an instruction, each addition off by 2^-23 of the
    magnitudes, four products of parts to a rank.
    """
    K, R = x.shape[1], down.shape[2]
    xd = x.double()
    v, mag = xd @ W.double(), xd.abs() @ W.double().abs()
    err = torch.zeros_like(v)
    for a in range(down.shape[0]):
        at = (adapter == a).nonzero().flatten()
        s, d, u = float(scale[a]), down[a].double(), up[a].double()
        h, h_mag = s * (xd[at] @ d), abs(s) * (xd[at].abs() @ d.abs())
        v[at] += h @ u
        mag[at] += h.abs() @ u.abs()
        err[at] += (sum_error(K, h_mag) + 2.0 ** -24 * h_mag + 2.0 ** -16 * h.abs()) @ u.abs()
    # the parts' products reach 1 + 2^-7 of h * u, and cover a rank up to four times
    return v, rounded(v, err + sum_error(K + 4 * R, 1.01 * mag), x.dtype)


def _infinite_alike(got, ref, tol, dtype):
    """check(), where a reference past the type's range has to be infinite (give or take the bound)."""
    top = torch.finfo(dtype).max
    out = ref.abs() - tol > top * (1 + half_step(dtype))
    assert torch.equal(got[out], (ref.sign() * float("inf"))[out].to(dtype))
    # close to the end of the range either of the two is right
    sure = ref.abs() + tol <= top
    check(torch.where(sure, got, torch.zeros_like(got)), torch.where(sure, ref, torch.zeros_like(ref)), tol)


@pytest.mark.parametrize("T", [1, 50, 300, 2100])
@pytest.mark.parametrize("R", [1, 16, 40])
@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_products_with_down_of_any_size(T, R, stored, dtype):
    """Scales from 1e-8 to 1e10 against `up` the other way round (its smallest are subnormal in fp16)."""
    from infinite_dreams import infinite_dreams_ext as ext
    K, N = 200, 136
    scales = [1e-8, 1e-6, 3e-5, 1e-3, 1.0, 2e4, 7e6, 1e10]
    L = len(scales)
    x, W = randn((T, K), dtype, 1), stacked(1, K, N, dtype, 2, stored)[0] * 1e-3
    down, up = stacked(L, K, R, dtype, 3, stored), stacked(L, R, N, torch.float32, 4, stored)
    up = (up * (0.5 / torch.tensor(scales, device="cuda")).clamp(2.0 ** -22, 2e4)[:, None, None]).to(dtype)
    scale = torch.tensor(scales, device="cuda")
    for ids in (torch.arange(T, device="cuda") % L, torch.arange(T, device="cuda") * 0 + 7, torch.full((T,), 0, device="cuda")):
        got = ext.lora_gemm(x, W, down, up, ids, scale=scale)
        _infinite_alike(got, *_bound(x, W, down, up, ids, scale), dtype)


@pytest.mark.parametrize("T", [3, 80])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_products_with_down_at_the_ends_of_the_ranges(T, dtype):
    """h exactly at the end of fp16's and of bf16's range, and beyond either, with `up` that brings it back."""
    from infinite_dreams import infinite_dreams_ext as ext
    K, N, R = 64, 64, 8
    x = torch.zeros(T, K, dtype=dtype, device="cuda")
    x[:, 0] = 1.0
    W, down, up = torch.zeros(K, N, dtype=dtype, device="cuda"), torch.zeros(1, K, R, dtype=dtype, device="cuda"), None
    down[:, 0, :] = torch.tensor([1, -1, 1.5, 0.5, -0.25, 0, 1, -1], dtype=dtype)
    ids = torch.zeros(T, dtype=torch.int32, device="cuda")
    top = torch.finfo(torch.bfloat16).max
    for h, u in ((65504.0, 1e-4), (65519.0, 1e-4), (65520.0, -1e-4), (65536.0, 1e-4), (2.0 ** 20 + 3, 2.0 ** -24),
                 (2.0 ** -24, 30000.0), (2.0 ** -30 * 3, -2e4), (1e-12, 6e4), (top * 0.6, 1e-30),
                 (top * 0.66667, 1e-36), (torch.finfo(torch.float32).max * 0.66666, 2.0 ** -120)):
        up = torch.full((1, R, N), u, dtype=dtype, device="cuda")
        up[0, 1::2] *= -0.5
        scale = torch.tensor([h], device="cuda")
        got = ext.lora_gemm(x, W, down, up, ids, scale=scale)
        _infinite_alike(got, *_bound(x, W, down, up, ids, scale), dtype)


def _padded(shape, dtype, seed, scale=1.0):
    """A tensor of this shape cut out of one with more rows and columns, all of them NaN, whose pitch is aligned."""
    full = torch.full((*shape[:-2], shape[-2] + 2, -(-shape[-1] // 8) * 8 + 8), float("nan"), dtype=dtype, device="cuda")
    part = full[..., :shape[-2], :shape[-1]]
    part.copy_(randn(shape, dtype, seed, scale))
    return part


@pytest.mark.parametrize("R", [3, 16, 21, 40, 65])
@pytest.mark.parametrize("T", [1, 40, 300, 2101])
@pytest.mark.parametrize("K,N", [(133, 141), (1029, 265)])
@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_padding_does_not_enter(R, T, K, N, stored, dtype):
    """NaN beside and below every operand whose pitch is aligned while its width is not."""
    from infinite_dreams import infinite_dreams_ext as ext
    L = 4
    x = _padded((T, K), dtype, 1)
    W, down, up = (_padded(s, dtype, i, f) if stored == "kn" else
                   _padded((*s[:-2], s[-1], s[-2]), dtype, i, f).transpose(-1, -2)
                   for s, i, f in (((K, N), 2, K ** -0.5), ((L, K, R), 3, K ** -0.5), ((L, R, N), 4, R ** -0.5)))
    ids = torch.arange(T, device="cuda") % (L + 1) - 1
    check(ext.lora_gemm(x, W, down, up, ids), *ref_lora(x, W, down, up, ids))


@pytest.mark.parametrize("K", [1024, 2048, 4096, 8200])
@pytest.mark.parametrize("N", [129, 1500])
@pytest.mark.parametrize("T", [1, 7, 64])
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_few_rows_with_the_sum_split_over_a_cluster(K, N, T, act, dtype):
    from infinite_dreams import infinite_dreams_ext as ext
    W, down, up = stacked(1, K, N, dtype, 1)[0], stacked(3, K, 24, dtype, 2), stacked(3, 24, N, dtype, 3)
    x, b, ids = randn((T, K), dtype, 4), randn((N,), dtype, 5), torch.arange(T, device="cuda") % 4 - 1
    check(ext.lora_gemm(x, W, down, up, ids, bias=b, activation=act), *ref_lora(x, W, down, up, ids, None, b, act))
