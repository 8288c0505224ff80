"""lora_gemm's two launches beside what runs before them."""
import pytest
import torch

from grouped_helpers import check, randn, ref_lora, stacked

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    from infinite_dreams import infinite_dreams_ext as ext
    yield
    torch.cuda.synchronize()
    ext.check_device_errors()


@pytest.mark.parametrize("T", [5, 300])
@pytest.mark.parametrize("cut", [0, 1], ids=["in place", "repacked"])
def test_operands_written_right_before_the_call(T, cut):
    """Every operand is rewritten by the kernels before each call, with no sync between: the bits of a synced run."""
    from infinite_dreams import infinite_dreams_ext as ext
    K, N, L, R, dt = 512, 520, 6, 24, torch.float16
    made = []
    for i in range(4):
        big = randn((T, K + cut), dt, i), randn((K, N + cut), dt, 10 + i, 0.1), randn((L, K, R + cut), dt, 20 + i, 0.1)
        made.append((*big, randn((L, R, N + cut), dt, 30 + i), randn((N,), dt, 40 + i),
                     ((torch.arange(T, device="cuda") * (i + 1)) % (L + 1) - 1).int()))
    now = [torch.empty_like(m) for m in made[0]]

    def calls(sync):
        outs = []
        for turn in range(40):
            for to, of in zip(now, made[turn % 4]):
                to.copy_(of)
            x, W, down, up, bias, ids = now
            outs.append(ext.lora_gemm(x[:, :K], W[:, :N], down[..., :R], up[..., :N], ids, bias=bias))
            if sync:
                torch.cuda.synchronize()
        return outs

    want = calls(True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(calls(False), want))
    x, W, down, up, bias, ids = made[0]
    check(want[0], *ref_lora(x[:, :K], W[:, :N], down[..., :R], up[..., :N], ids, None, bias))
