"""gemm_ex into columns of a wider matrix: the values of a contiguous output, and nothing beside them is written."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 16, 64, 300, 1000])
@pytest.mark.parametrize("N", [1, 9, 260, 261, 1023, 1024])
@pytest.mark.parametrize("K", [64, 4096])
def test_columns_beside_the_output_stay(cuda_device, M, N, K):
    from infinite_dreams import infinite_dreams_ext as ext
    g = torch.Generator(device="cuda").manual_seed(M + N)
    A = torch.randn(M, K, generator=g, device="cuda").half()
    B = (torch.randn(K, N, generator=g, device="cuda") * K ** -0.5).half()
    bias = torch.randn(N, generator=g, device="cuda").half()
    cfgs = [None] + list(range(0, ext.NUM_CFG, max(1, ext.NUM_CFG // 24)))
    for cfg in cfgs:
        want = ext.gemm_ex(A, B, bias=bias, activation="relu", cfg_id=cfg)
        wide = torch.full((M + 2, (N + 7) // 8 * 8 + 16), 7.0, dtype=torch.float16, device="cuda")
        got = wide[1:-1, 8:8 + N]
        ext.gemm_ex(A, B, bias=bias, activation="relu", cfg_id=cfg, out=got)
        assert torch.equal(got, want), cfg
        got.fill_(7.0)
        assert bool((wide == 7).all()), cfg
    torch.cuda.synchronize()
    ext.check_device_errors()


@pytest.mark.parametrize("binding", ["compiled", "ctypes"])
@pytest.mark.parametrize("M,N", [(300, 136), (16, 256), (5, 1)])
def test_rows_that_lie_on_one_another(cuda_device, binding, M, N):
    """One row given as C for all of them is read as such, and an out whose rows are not apart is refused."""
    from infinite_dreams import infinite_dreams_ext as ext
    g = torch.Generator(device="cuda").manual_seed(M)
    A = torch.randn(M, 64, generator=g, device="cuda").half()
    B = torch.randn(64, N, generator=g, device="cuda").half()
    row = torch.randn(1, N, generator=g, device="cuda").half()
    keep, ext._fast = ext._fast, ext._fast if binding == "compiled" else None
    try:
        want = ext.gemm_ex(A, B, beta=1.0, C=row.expand(M, N).contiguous())
        assert torch.equal(ext.gemm_ex(A, B, beta=1.0, C=row.expand(M, N)), want)
        for out in (row.expand(M, N), torch.empty(M + N, dtype=torch.float16, device="cuda").as_strided((M, N), (0, 1))):
            with pytest.raises(RuntimeError, match="rows apart"):
                ext.gemm_ex(A, B, out=out)
    finally:
        ext._fast = keep
