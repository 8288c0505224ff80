"""lora_gemm against a 64-bit reference, at the sizes, ranks and choices of adapters where it can go wrong."""
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


def _weights(K, N, L, R, dtype, stored="kn", seed=1):
    W = stacked(1, K, N, dtype, seed, stored)[0]
    return W, stacked(L, K, R, dtype, seed + 1, stored), stacked(L, R, N, dtype, seed + 2, stored)


def _ids(T, L, pattern, dtype=torch.int32):
    """Which adapter each row picks."""
    g = torch.Generator().manual_seed(T + L)
    if pattern == "random":
        ids = torch.randint(-1, L, (T,), generator=g)
    elif pattern == "runs":
        ids = torch.arange(T) * 5 // max(T, 1) % (L + 1) - 1
    elif pattern == "one":
        ids = torch.full((T,), L - 1)
    elif pattern == "none":
        ids = torch.full((T,), -1)
    return ids.to(dtype).cuda()


def _run(T, K, N, L, R, dtype, stored="kn", pattern="random", scale=True, bias=False, act="none", index=torch.int32):
    from infinite_dreams import infinite_dreams_ext as ext
    x, (W, down, up) = randn((T, K), dtype, 9), _weights(K, N, L, R, dtype, stored)
    ids = _ids(T, L, pattern, index)
    s = torch.rand(L, generator=torch.Generator().manual_seed(3)).cuda() + 0.5 if scale else None
    b = randn((N,), dtype, 11, 0.5) if bias else None
    out = ext.lora_gemm(x, W, down, up, ids, scale=s, bias=b, activation=act)
    ref, tol = ref_lora(x, W, down, up, ids, s, b, act)
    check(out, ref, tol, f"T={T} K={K} N={N} L={L} R={R} {pattern}")
    return x, W, down, up, ids, s, out


@pytest.mark.parametrize("T", [1, 2, 16, 17, 33, 63, 64, 65, 100, 256, 257, 700])
@pytest.mark.parametrize("pattern", ["random", "runs", "one", "none"])
@pytest.mark.parametrize("stored", ["kn", "nk"])
def test_rows(T, pattern, stored):
    _run(T, 192, 264, 5, 16, torch.float16, stored, pattern, index=torch.int64 if T % 2 else torch.int32)


@pytest.mark.parametrize("R", [1, 4, 8, 16, 24, 31, 32, 33, 48, 64, 65, 128, 200])
@pytest.mark.parametrize("T", [30, 150])
@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_ranks(R, T, stored, dtype):
    _run(T, 320, 256, 4, R, dtype, stored)


@pytest.mark.parametrize("K,N", [(1, 1), (8, 8), (33, 520), (777, 1023), (1000, 129), (4096, 128), (72, 2000)])
@pytest.mark.parametrize("T", [20, 200])
@pytest.mark.parametrize("stored", ["kn", "nk"])
def test_sizes(K, N, T, stored):
    _run(T, K, N, 3, 16, torch.float16, stored, bias=True, act="relu")


@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
@pytest.mark.parametrize("T", [20, 200])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_epilogue(act, T, dtype):
    _run(T, 256, 384, 4, 8, dtype, "nk", bias=True, act=act, scale=False)


def test_every_row_its_own_adapter():
    """256 adapters in a tile, more adapters than rows, and adapters scattered over the tiles."""
    from infinite_dreams import infinite_dreams_ext as ext
    for T, L in ((64, 64), (256, 300), (600, 600)):
        x, (W, down, up) = randn((T, 128), torch.bfloat16, 1), _weights(128, 256, L, 8, torch.bfloat16)
        ids = torch.randperm(L, generator=torch.Generator().manual_seed(1))[:T].to(torch.int32).cuda()
        check(ext.lora_gemm(x, W, down, up, ids), *ref_lora(x, W, down, up, ids))


@pytest.mark.parametrize("T,K,N,L,R", [(513, 64, 64, 3, 8), (700, 4096, 72, 5, 64), (1999, 320, 136, 4, 24),
                                       (2100, 2000, 64, 9, 130), (4700, 1032, 64, 3, 48), (5000, 4096, 128, 6, 16),
                                       (9000, 520, 64, 4, 200)])
@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("pattern", ["random", "runs"])
def test_many_rows(T, K, N, L, R, stored, pattern):
    """The low-rank half's two tiles, with K split over clusters and without."""
    _run(T, K, N, L, R, torch.float16 if T % 2 else torch.bfloat16, stored, pattern)


@pytest.mark.parametrize("T,K,N,L,R,pattern", [
    (20000, 64, 64, 2, 1024, "runs"), (20000, 200, 64, 40, 16, "random"),     # single CTAs
    (5120, 64, 1024, 40, 16, "random"), (21000, 328, 256, 3, 300, "runs")])   # pairs
def test_many_tiles_with_many_blocks(T, K, N, L, R, pattern):
    """CTAs that do several tiles, each with more adapter blocks than twice the ring's stages."""
    _run(T, K, N, L, R, torch.bfloat16, "nk", pattern, scale=False)


@pytest.mark.parametrize("T", [40, 300])
@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("where", ["up", "down", "x"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_one_request_does_not_reach_another(T, stored, where, bad):
    """inf or NaN in one adapter's weights or one request's rows: the others keep their bits, its own rows show it."""
    from infinite_dreams import infinite_dreams_ext as ext
    for R in (16, 72):
        x, (W, down, up) = randn((T, 128), torch.float16, 1), _weights(128, 264, 4, R, torch.float16, stored)
        ids = _ids(T, 4, "random")
        clean = ext.lora_gemm(x, W, down, up, ids)
        mine = ids == 2
        {"up": up[2, 5, 7:], "down": down[2, 3:], "x": x[mine]}[where][:] = bad
        if where == "x":
            x[mine] = bad
        got = ext.lora_gemm(x, W, down, up, ids)
        assert torch.equal(got[~mine], clean[~mine])
        if where == "up":     # one rank of some columns: h * bad there, the rest as before
            assert torch.equal(got[mine][:, :7], clean[mine][:, :7]) and not bool(got[mine][:, 7:].isfinite().any())
            if bad == float("inf"):
                h = x[mine].double() @ down[2, :, 5].double()
                assert torch.equal(got[mine][:, 7:].sign(), h.sign()[:, None].expand(-1, 257).to(got.dtype))
        else:
            assert not bool(got[mine].isfinite().any())


@pytest.mark.parametrize("T", [9, 90])
def test_strides(T):
    """Pitches, unaligned bases, weights cut out of larger ones, expanded and permuted ones; a strided output."""
    from infinite_dreams import infinite_dreams_ext as ext
    K, N, R, dt = 136, 144, 16, torch.bfloat16
    ids = _ids(T, 3, "random")
    big_x, big_w = randn((T, K + 24), dt, 1), randn((K + 8, N + 40), dt, 2, 0.1)
    big_d, big_u = randn((5, K + 8, R + 8), dt, 3, 0.1), randn((5, R + 2, N + 24), dt, 4, 0.1)
    out = torch.full((T, N + 16), 5.0, dtype=dt, device="cuda")
    for x, W, down, up in [
            (big_x[:, 8:8 + K], big_w[:K, 16:16 + N], big_d[:3, :K, :R], big_u[:3, :R, 8:8 + N]),
            (big_x[:, 3:3 + K], big_w[1:1 + K, 5:5 + N], big_d[::2, 1:1 + K, 3:3 + R], big_u[::2, 1:1 + R, 7:7 + N]),
            (randn((K, T), dt, 5).t(), randn((N, K), dt, 6, 0.1).t(), big_d[:1, :K, :R].expand(3, K, R),
             randn((R, 3, N), dt, 7, 0.1).transpose(0, 1)),
            (big_x[:1, :K].expand(T, K), big_w[:K, :N], randn((R, K, 3), dt, 8, 0.1).permute(2, 1, 0),
             randn((3, N, R + 1), dt, 9, 0.1)[:, :, 1:].transpose(1, 2))]:
        ref, tol = ref_lora(x, W, down, up, ids)
        check(ext.lora_gemm(x, W, down, up, ids, out=out[:, 8:8 + N]), ref, tol)
    assert bool((out[:, :8] == 5).all()) and bool((out[:, 8 + N:] == 5).all())


def test_without_adapters_it_is_the_projection():
    """Rows without an adapter get x @ W, whatever the others pick: gemm_ex's value, or the next one (one fp16 step,
    2^-10 of the value, where the two kernels' sums differ in the last bits)."""
    from infinite_dreams import infinite_dreams_ext as ext
    x, W, down, up, ids, s, out = _run(200, 512, 256, 4, 16, torch.float16)
    plain = ext.gemm_ex(x, W)
    none = ids < 0
    off = (out[none].float() - plain[none].float()).abs()
    assert bool(none.any()) and bool((off <= 2.0 ** -10 * plain[none].float().abs() + 2.0 ** -14).all())


def test_index_past_the_last_adapter():
    from infinite_dreams import infinite_dreams_ext as ext
    for T in (10, 100):
        x, (W, down, up) = randn((T, 64), torch.float16, 1), _weights(64, 128, 2, 8, torch.float16)
        ids = _ids(T, 2, "random")
        ids[3] = 2
        ids[7] = 1 << 30
        check(ext.lora_gemm(x, W, down, up, ids), *ref_lora(x, W, down, up, ids))
        with pytest.raises(RuntimeError, match="adapter index"):
            ext.check_device_errors()


def test_both_bindings_give_the_same_bits():
    from infinite_dreams import infinite_dreams_ext as ext
    x, W, down, up, ids, s, fast = _run(77, 100, 201, 3, 12, torch.bfloat16, "nk")
    keep, ext._fast = ext._fast, None
    try:
        slow = ext.lora_gemm(x, W, down, up, ids, scale=s)
    finally:
        ext._fast = keep
    assert torch.equal(fast.view(torch.int16), slow.view(torch.int16))


@pytest.mark.parametrize("T", [8, 300])
def test_chained_calls_and_another_stream(T):
    """Each call reads the one before, with no sync between them; the same bits as one at a time."""
    from infinite_dreams import infinite_dreams_ext as ext
    W, down, up = _weights(256, 256, 4, 16, torch.float16)
    ids, x0 = _ids(T, 4, "random"), randn((T, 256), torch.float16, 2)

    def chain(sync):
        x = x0
        for _ in range(8):
            x = ext.lora_gemm(x, W, down, up, ids)
            if sync:
                torch.cuda.synchronize()
        return x

    want = chain(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [chain(False) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_two_graphs_replayed_at_once():
    """Two graphs captured on one stream, replayed on two, with new adapter choices: the eager bits each time."""
    from infinite_dreams import infinite_dreams_ext as ext
    W, down, up = _weights(512, 1024, 6, 16, torch.float16)
    xs = [randn((48, 512), torch.float16, 5), randn((200, 512), torch.float16, 6)]
    ids = [_ids(48, 6, "random"), _ids(200, 6, "random")]
    ext.lora_gemm(xs[1], W, down, up, ids[1])
    torch.cuda.synchronize()
    side, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for x, i in zip(xs, ids):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side[0]):
            outs.append(ext.lora_gemm(x, W, down, up, i))
        graphs.append(g)
    for turn in range(3):
        want = [ext.lora_gemm(x, W, down, up, i) for x, i in zip(xs, ids)]
        for _ in range(5):
            torch.cuda.synchronize()
            for s, g in zip(side, graphs):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, w) for o, w in zip(outs, want)), turn
        for i in ids:
            i.copy_(i.roll(turn + 1))


def test_refuses_gradients():
    from infinite_dreams import infinite_dreams_ext as ext
    W, down, up = _weights(64, 64, 2, 8, torch.float16)
    with pytest.raises(RuntimeError, match="serving operator"):
        ext.lora_gemm(randn((4, 64), torch.float16, 1), W, down.requires_grad_(), up, _ids(4, 2, "one"))


def test_an_expert_layer_and_an_adapted_projection_together():
    """Rows through an adapted projection, then sorted by expert through the experts: the two operators in a row."""
    from infinite_dreams import infinite_dreams_ext as ext
    from grouped_helpers import counts_to_offsets, ref_grouped
    T, K, N, E, dt = 150, 256, 320, 5, torch.bfloat16
    x, (W, down, up) = randn((T, K), dt, 1), _weights(K, K, 3, 8, dt)
    ids, expert = _ids(T, 3, "random"), torch.randint(0, E, (T,), generator=torch.Generator().manual_seed(4)).cuda()
    order = expert.argsort(stable=True)
    off = counts_to_offsets(torch.bincount(expert, minlength=E).tolist())
    B = stacked(E, K, N, dt, 5)
    h = ext.lora_gemm(x, W, down, up, ids, activation="gelu")
    y = torch.empty((T, N), dtype=dt, device="cuda")
    y[order] = ext.grouped_gemm(h[order], B, off)
    check(h, *ref_lora(x, W, down, up, ids, act="gelu"))
    ref, tol = ref_grouped(h[order], B, off)
    check(y[order], ref, tol)
