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


def test_a_low_rank_half_longer_than_the_bounded_waits():
    """The product's waits give up after two seconds of its own, not of the kernel that it waits for (3.2 s here)."""
    from infinite_dreams import infinite_dreams_ext as ext
    T, K, N, L, R, dt = 400000, 8192, 64, 8, 1024, torch.bfloat16
    W = randn((K, N), dt, 1, K ** -0.5)
    # rows of 1025 elements: read one element at a time
    down, up = randn((L, K, R + 1), dt, 2, K ** -0.5)[..., :R], randn((L, R, N), dt, 3, R ** -0.5)
    x = torch.empty(T, K, dtype=dt, device="cuda")
    part = randn((T // 32, K), dt, 4)
    for i in range(32):
        x[i * (T // 32):(i + 1) * (T // 32)] = part
    ids = (torch.arange(T, device="cuda") % L).int()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    out = ext.lora_gemm(x, W, down, up, ids)
    end.record()
    torch.cuda.synchronize()
    ext.check_device_errors()
    assert start.elapsed_time(end) > 2000   # else this shows nothing: give it more rows
    for at in (slice(0, 300), slice(T // 2, T // 2 + 300), slice(T - 300, T)):
        check(out[at], *ref_lora(x[at], W, down, up, ids[at]))


@pytest.mark.parametrize("T,K,L,R", [(5000, 1024, 3, 16), (2100, 520, 4, 8), (4100, 264, 8, 32), (4100, 264, 9, 32),
                                     (5000, 512, 40, 64), (9000, 200, 300, 16), (3000, 328, 17, 100)])
@pytest.mark.parametrize("stored", ["kn", "nk"])
def test_many_rows_of_few_and_of_many_adapters(T, K, L, R, stored):
    """Both forms of the low-rank half past 2048 rows, on either side of the rule that picks one."""
    from infinite_dreams import infinite_dreams_ext as ext
    dt = torch.bfloat16
    x, W, down, up = (randn((T, K), dt, 1), stacked(1, K, 72, dt, 2, stored)[0], stacked(L, K, R, dt, 3, stored),
                      stacked(L, R, 72, dt, 4, stored))
    for ids in (torch.arange(T, device="cuda") * 7 % (L + 1) - 1, torch.arange(T, device="cuda") * L // T):
        check(ext.lora_gemm(x, W, down, up, ids), *ref_lora(x, W, down, up, ids))


def test_rows_that_each_pick_another_adapter_cost_no_pass_over_x_each():
    """8192 rows of 64 adapters of rank 16: about four times as long one by one as in runs (fourteen times where the
    low-rank half passed over a tile's rows once per adapter)."""
    from infinite_dreams import infinite_dreams_ext as ext
    T, K, N, L, R, dt = 8192, 4096, 128, 64, 16, torch.bfloat16
    x, W, down, up = (randn((T, K), dt, 1), randn((K, N), dt, 2), stacked(L, K, R, dt, 3), stacked(L, R, N, dt, 4))
    rows = torch.arange(T, device="cuda")

    def best(ids):
        times = []
        for _ in range(10):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            for _ in range(5):
                ext.lora_gemm(x, W, down, up, ids)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    assert best(rows * 7 % L) < 8 * best(rows * L // T)
