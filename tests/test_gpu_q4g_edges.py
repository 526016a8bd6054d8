"""Group-scaled products and the gated half at the edges of what a caller may do."""
import numpy as np
import pytest

from test_gpu_q4g import bound, dense, make_weight, rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_cuda():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


@pytest.fixture(scope="module")
def ctx(torch_cuda):
    from mojostream_b200.runtime import Context
    c = Context(0)
    yield c
    c.close()


def test_sources_that_a_stream_still_writes(ctx, torch_cuda):
    """Pinned host sources filled by copies that wait, on a stream of their
    own, behind 100 ms of other work: the weight is made of what they bring."""
    torch = torch_cuda
    from mojostream_b200.runtime import Q4GroupWeight
    rng = np.random.default_rng(21)
    K, N, g = 256, 128, 64
    q, s, z = make_weight(rng, K, N, g, True)
    want = [torch.from_numpy(x).cuda() for x in (q, s, z)]
    host = [torch.zeros(x.shape, dtype=x.dtype).pin_memory() for x in want]
    a = rows(torch, rng, 3, K, 0, torch.float32)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        for h, x in zip(host, want):
            h.copy_(x, non_blocking=True)
    w = Q4GroupWeight(ctx, host[0], host[1], K, N, g, zeros=host[2])
    c = w.gemm(a, torch.empty((3, N), device="cuda"))
    ctx.sync(current=True)
    a64, wd = a.double().cpu().numpy(), dense(q, s, z, g)
    exact = a64 @ wd
    assert (np.abs(c.double().cpu().numpy() - exact) <= bound(torch, torch.float32, g, a64, wd, exact)).all()
    w.close()


def test_a_refused_weight_leaves_no_error_behind(ctx, torch_cuda):
    """A weight larger than the device is refused, and only that: the calls
    after it, whose launches also report errors, succeed."""
    import ctypes
    torch = torch_cuda
    from mojostream_b200 import _lib
    from mojostream_b200.runtime import LogitRules
    q, s = np.zeros(64, np.uint8), np.zeros(64, np.float16)
    h = ctypes.c_void_p()
    for _ in range(2):
        # 2^39 bytes: no allocation, so nothing of q or s is read
        status = _lib.lib().ms_q4g_weight_create(ctx.h, q.ctypes.data, s.ctypes.data, 2, None, 1 << 20,
                                                 1 << 20, 128, ctypes.byref(h))
        assert _lib.STATUS_NAMES[status] == "MS_ERR_OOM" and not h
        mask = torch.full((1, 2), 5, dtype=torch.int32, device="cuda")
        lg = torch.ones((1, 40), device="cuda")
        ctx.logit_rules(lg, LogitRules(mask=mask))
        assert torch.isfinite(lg).sum() == 4
    ctx.sync(current=True)


@pytest.mark.parametrize("M", [20, 50, 300])
@pytest.mark.parametrize("g", [32, 64])
def test_fp32_sums_of_many_rows_keep_their_last_bits(ctx, torch_cuda, M, g):
    """The error of all results together (2-norms).  An MMA of 16 k cuts its sum
    off: half a unit of 2^-23 on average of a partial sum, whose size after
    the j-th of a group's g / 16 is sqrt(16 j / g) of the group's.  That is if
    the limbs come smallest first; the smaller limbs after the largest would
    add 2 g / 16 cuts at full size.  Then K / g sums in fp32, each rounded by
    2^-24 / sqrt(3) (uniform) of a partial sum of sqrt(j g / K)."""
    torch = torch_cuda
    from mojostream_b200.runtime import Q4GroupWeight
    rng = np.random.default_rng(M + g)
    K, N = 256, 512
    q, s, z = make_weight(rng, K, N, g, True)
    w = Q4GroupWeight(ctx, q, s, K, N, g, zeros=z)
    a = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).cuda()
    c = w.gemm(a, torch.empty((M, N), device="cuda")).double().cpu().numpy()
    exact = a.double().cpu().numpy() @ dense(q, s, z, g)
    steps, groups = g // 16, K // g
    cuts = 0.5 * 2.0 ** -23 * sum(((j + 1) / steps) ** 0.5 for j in range(steps))
    limit = cuts + 2.0 ** -24 / 3 ** 0.5 * ((groups + 1) / 2) ** 0.5
    assert np.linalg.norm(c - exact) <= limit * np.linalg.norm(exact)
    w.close()


@pytest.mark.parametrize("M", [1, 2, 3, 5, 8, 9, 40])
@pytest.mark.parametrize("large", [1e4, 1e6])
def test_a_large_channel_of_weights_zero_takes_no_bits(ctx, torch_cuda, M, large):
    """Two channels of every group are `large` and meet weights that are 0, the
    rest are around 1: the error is that of fp32 sums of the rest, however many
    rows the call has.  With 2-norms and independent roundings (uniform,
    2^-24 / sqrt(3) each): a group's sum is converted, scaled and added (three),
    partial sums grow as sqrt(groups); of more rows the MMAs cut off half a
    unit of 2^-23 four times a group at most.  A value is held to 2^-45 of the
    largest: less than 2^-25 of 1."""
    torch = torch_cuda
    from mojostream_b200.runtime import Q4GroupWeight
    rng = np.random.default_rng(M)
    K, N, g = 256, 512, 64
    q, s, z = make_weight(rng, K, N, g, True)
    big = np.arange(K).reshape(-1, g)[:, [5, 40]].ravel()
    zz = np.repeat(z, g, 0)[big]
    q[big] = zz[:, 0::2] | (zz[:, 1::2] << 4)
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[:, big] *= large
    a = torch.from_numpy(x).cuda()
    w = Q4GroupWeight(ctx, q, s, K, N, g, zeros=z)
    c = w.gemm(a, torch.empty((M, N), device="cuda")).double().cpu().numpy()
    wd = dense(q, s, z, g)
    assert not wd[big].any()
    exact = x.astype(np.float64) @ wd
    limit = 2.0 ** -24 / 3 ** 0.5 * (3 ** 0.5 + ((K // g + 1) / 2) ** 0.5) + 2.0 ** -25
    if M > 8:
        limit += 0.5 * 2.0 ** -23 * 4
    assert np.linalg.norm(c - exact) <= limit * np.linalg.norm(exact)
    w.close()


def infinite_rows(torch, rng, K, dt):
    """Rows with infinities at random: two to six in one group of k, one in
    each of two groups, everywhere."""
    x = rng.standard_normal((8, K))
    for r in range(6):
        at = rng.choice(32, size=2 + r % 5, replace=False) + 32 * (r % (K // 32))
        x[r, at] = np.where(rng.random(len(at)) < 0.5, np.inf, -np.inf)
    x[6, [3, K - 1]] = np.inf, -np.inf
    x[7] = np.where(rng.random(K) < 0.5, np.inf, -np.inf)
    return torch.from_numpy(x.astype(np.float32)).cuda().to(dt)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("M", [8, 24])
@pytest.mark.parametrize("zeros,g,accumulate", [(False, 32, False), (True, 64, True), (True, 128, False)])
def test_several_infinities_of_a_row(ctx, torch_cuda, M, dtype, zeros, g, accumulate):
    """Infinities of opposite sign add up to NaN, of one sign to that infinity,
    and one that meets a weight of 0 is NaN: as the definition has it, of few
    rows and of many."""
    torch = torch_cuda
    from mojostream_b200.runtime import Q4GroupWeight
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(M + g)
    K, N = 384, 140
    q, s, z = make_weight(rng, K, N, g, zeros)
    s[:, 5::7] *= -1
    if not zeros:
        q[:, 20:60] = rng.choice([0x9a, 0xbc, 0xdf], size=(K, 40))  # one sign, no zeros
    w = Q4GroupWeight(ctx, q, s, K, N, g, zeros=z)
    x = torch.cat([infinite_rows(torch, rng, K, dt) for _ in range(M // 8)])
    c = torch.ones((M, N), dtype=dt, device="cuda")
    w.gemm(x, c, accumulate=accumulate)
    with np.errstate(invalid="ignore"):
        want = x.double().cpu().numpy() @ dense(q, s, z, g)
    got = c.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert np.isinf(want[fine]).all() and np.array_equal(got[fine], want[fine])
    assert zeros or np.isinf(want).any()
    w.close()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("M", [8, 24])
@pytest.mark.parametrize("same", [False, True])
def test_several_infinities_of_a_gated_row(ctx, torch_cuda, M, dtype, same):
    torch = torch_cuda
    from mojostream_b200.runtime import Q4GroupWeight
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(M)
    K, N, g = 256, 66, 64
    mats = [make_weight(rng, K, N, g, False) for _ in range(2)]
    for q, _, _ in mats:
        q[:, 8:] = rng.choice([0x9a, 0xbc, 0xdf], size=(K, N // 2 - 8))
    if same:
        mats[1] = mats[0]
    gate = Q4GroupWeight(ctx, *mats[0][:2], K, N, g)
    up = gate if same else Q4GroupWeight(ctx, *mats[1][:2], K, N, g)
    x = torch.cat([infinite_rows(torch, rng, K, dt) for _ in range(M // 8)])
    x[0] = x[0].abs()
    h = torch.empty((M, N), dtype=dt, device="cuda")
    gate.gated(up, x, h)
    a = x.double().cpu().numpy()
    with np.errstate(invalid="ignore", over="ignore"):
        v, u = (a @ dense(*m, g) for m in mats)
        want = v / (1 + np.exp(-v)) * u  # (NaN for a gate of -infinity)
    got = h.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert fine[0, 16:].all() and np.array_equal(got[fine], want[fine])


@pytest.mark.parametrize("M", [1, 4, 30])
def test_operands_that_share_memory(ctx, torch_cuda, M):
    """Products of A and C that share memory are refused and write nothing;
    column blocks of one buffer share none."""
    torch = torch_cuda
    from mojostream_b200 import MsError
    from mojostream_b200.runtime import Q4GroupWeight
    rng = np.random.default_rng(M)
    K, N, g = 128, 64, 64
    q, s, z = make_weight(rng, K, N, g, True)
    w = Q4GroupWeight(ctx, q, s, K, N, g, zeros=z)
    buf = torch.from_numpy(rng.standard_normal((M + 1, K + N)).astype(np.float32)).cuda()
    before = buf.clone()
    for c in (buf[:M, :N], buf[:M, K - 1:K - 1 + N], buf[1:, 5:5 + N] if M > 1 else buf[:M, 7:7 + N]):
        with pytest.raises(MsError, match="share memory"):
            w.gemm(buf[:M, :K], c)
        with pytest.raises(MsError, match="share memory"):
            w.gated(w, buf[:M, :K], c)
    assert torch.equal(buf, before)
    want = w.gemm(before[:M, :K], torch.empty((M, N), device="cuda"))
    w.gemm(buf[:M, :K], buf[:M, K:])
    assert torch.equal(buf[:M, K:], want) and torch.equal(buf[:, :K], before[:, :K])
    assert torch.equal(buf[M], before[M])
    w.close()


@pytest.mark.parametrize("M", [9, 20, 50, 300])
def test_fp32_sums_of_long_groups_keep_their_last_bits(ctx, torch_cuda, M):
    """A group of 128 as two sums of 64, each with the bound of the test before:
    one sum would cut the second half's small limbs off against the first half
    (eight more cuts of half a unit at 0.7 of the group's size)."""
    torch = torch_cuda
    from mojostream_b200.runtime import Q4GroupWeight
    rng = np.random.default_rng(M)
    K, N, g = 256, 512, 128
    q, s, z = make_weight(rng, K, N, g, True)
    w = Q4GroupWeight(ctx, q, s, K, N, g, zeros=z)
    a = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).cuda()
    c = w.gemm(a, torch.empty((M, N), device="cuda")).double().cpu().numpy()
    exact = a.double().cpu().numpy() @ dense(q, s, z, g)
    cuts = 0.5 * 2.0 ** -23 * sum(((j + 1) / 4) ** 0.5 for j in range(4))
    limit = cuts + 2.0 ** -24 / 3 ** 0.5 * ((K // 64 + 1) / 2) ** 0.5
    assert np.linalg.norm(c - exact) <= limit * np.linalg.norm(exact)
    w.close()
