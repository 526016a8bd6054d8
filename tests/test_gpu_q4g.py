"""Products with group-scaled 4-bit weights and the gated half on them
(ms_q4g_gemm, ms_q4g_gated) against their definition in 64 bits.

Bounds, with u = 2^-24 and S = sum_k |a w|; the larger of the two holds for
any number of rows.
  Integer digits (decode rows).  A value is held to half a step of its group's
scale: 2^-30 (fp32) or 2^-22 (16-bit types) of the group's largest value, at
least 2^-120.  Group sums of digits are exact; per digit the K / g groups are
scaled and added in fp32, the digits of a value add up to at most 2 |a| in
magnitude, and scale, factor, up to 16 + 8 partial sums and the digits cost
one rounding each:  2 (K / g + 32) u S.
  bfloat16 limbs (more rows).  Every product is exact; an MMA of 16 k adds to
an fp32 accumulator with an error of at most 4 u (alignment of the addends and
the final rounding) of the magnitudes that it adds, a group takes g / 16 MMAs
per limb, and the group and partial sums one rounding each:
(4 limbs g / 16 + K / g + 20) u S.
  Then half a step of the result's type.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
LIMBS = {"float32": 3, "float16": 2, "bfloat16": 1}


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


def make_weight(rng, K, N, g, zeros, scale=0.02, bf=False):
    q = rng.integers(0, 256, size=(K, N // 2), dtype=np.uint8)
    s = (scale * (0.5 + rng.random((K // g, N)))).astype(np.float16)
    z = rng.integers(0, 16, size=(K // g, N), dtype=np.uint8) if zeros else None
    return q, s, z


def dense(q, s, z, g):
    K, half = q.shape
    v = np.empty((K, 2 * half))
    v[:, 0::2] = q & 15
    v[:, 1::2] = q >> 4
    group = np.arange(K) // g
    return (v - (8.0 if z is None else z[group].astype(np.float64))) * s.astype(np.float64)[group]


def sums_bound(name, g, a64, wd):
    """Bound of |sum - exact| before the result is rounded."""
    K = wd.shape[0]
    mag = np.abs(a64) @ np.abs(wd)
    steps = max(4 * LIMBS[name] * g / 16 + K / g + 20, 2 * (K / g + 32))
    half = 2.0 ** -30 if name == "float32" else 2.0 ** -22
    top = np.abs(a64).reshape(len(a64), K // g, g).max(2)
    per_group = np.abs(wd).reshape(K // g, g, -1).sum(1)
    return steps * U * mag + np.maximum(half * top, 2.0 ** -120) @ per_group


def rounded(torch, dtype, tol, exact):
    """A bound after rounding to dtype (half a step, or of its smallest step near zero)."""
    half = torch.finfo(dtype).eps / 2
    return tol * (1 + half) + half * np.abs(exact) + torch.finfo(dtype).smallest_normal * half


def bound(torch, dtype, g, a64, wd, exact, c0=0.0):
    tol = sums_bound(str(dtype).replace("torch.", ""), g, a64, wd) + U * (np.abs(exact) + np.abs(c0))
    return rounded(torch, dtype, tol, exact)


def rows(torch, rng, M, K, pad, dtype):
    a = rng.standard_normal((M, K + pad)).astype(np.float32)
    a[:, rng.integers(0, K, size=max(1, K // 50))] *= 30
    t = torch.from_numpy(a).cuda().to(dtype)
    return t[:, :K]


def check(torch, ctx, M, K, N, g, zeros, dtype, pad, seed=0, accumulate=False):
    from mojostream_b200.runtime import Q4GroupWeight
    rng = np.random.default_rng(seed + M * 7 + K * 3 + N)
    q, s, z = make_weight(rng, K, N, g, zeros)
    w = Q4GroupWeight(ctx, q, s, K, N, g, zeros=z)
    a = rows(torch, rng, M, K, pad, dtype)
    buf = torch.full((M + 1, N + pad + 1), 7.0, dtype=dtype, device="cuda")
    c = buf[:M, :N]
    c0 = np.zeros((M, N))
    if accumulate:
        c.copy_(torch.from_numpy(rng.standard_normal((M, N))).to(dtype))
        c0 = c.double().cpu().numpy()
    out = w.gemm(a, c, accumulate=accumulate)
    ctx.sync(current=True)
    assert out is c
    a64, wd = a.double().cpu().numpy(), dense(q, s, z, g)
    exact = a64 @ wd + c0
    err, tol = np.abs(c.double().cpu().numpy() - exact), bound(torch, dtype, g, a64, wd, exact, c0)
    assert (err <= tol).all(), float((err / tol).max())
    # nothing beside the result is touched
    assert (buf[M] == 7).all() and (buf[:, N:] == 7).all()
    w.close()


DT = ["float32", "bfloat16", "float16"]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,K,N,g,zeros,pad", [
    (1, 32, 2, 32, False, 0),        # the smallest: one group, two columns
    (1, 64, 16, 64, True, 0),
    (1, 128, 64, 128, False, 0),
    (1, 2560, 2048, 32, False, 0),
    (2, 96, 30, 32, True, 1),        # k that ends inside a block, odd strides
    (3, 160, 66, 32, False, 3),
    (4, 10240, 256, 64, False, 0),   # a long k split over all warps
    (5, 192, 1030, 64, True, 8),
    (7, 2592, 1030, 32, True, 24),
    (8, 384, 130, 128, True, 0),
    (9, 256, 62, 128, False, 5),     # the second row width
    (16, 1280, 640, 64, True, 0),
    (17, 512, 96, 32, False, 0),     # a second block of rows with one row in it
    (33, 256, 128, 128, True, 2),
    (64, 1024, 320, 128, False, 0),
    (130, 640, 258, 64, True, 0),
    (257, 2560, 514, 32, False, 8),
])
def test_product(ctx, torch_cuda, M, K, N, g, zeros, pad, dtype):
    check(torch_cuda, ctx, M, K, N, g, zeros, getattr(torch_cuda, dtype), pad)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M", [1, 6, 20, 200])
def test_accumulate(ctx, torch_cuda, M, dtype):
    check(torch_cuda, ctx, M, 320, 100, 32, True, getattr(torch_cuda, dtype), 4, accumulate=True)


@pytest.mark.parametrize("M", [1, 12, 300])
def test_bf16_scales_and_device_sources(ctx, torch_cuda, M):
    torch = torch_cuda
    from mojostream_b200.runtime import Q4GroupWeight
    rng = np.random.default_rng(3)
    K, N, g = 256, 192, 64
    q, s, z = make_weight(rng, K, N, g, True)
    sb = torch.from_numpy(s.astype(np.float32) * 1e6).cuda().to(torch.bfloat16)  # beyond half's range
    w = Q4GroupWeight(ctx, torch.from_numpy(q).cuda(), sb, K, N, g, zeros=torch.from_numpy(z).cuda())
    a = rows(torch, rng, M, K, 0, torch.float32)
    c = torch.empty((M, N), device="cuda")
    w.gemm(a, c)
    a64, wd = a.double().cpu().numpy(), dense(q, sb.double().cpu().numpy(), z, g)
    exact = a64 @ wd
    assert (np.abs(c.double().cpu().numpy() - exact) <= bound(torch, torch.float32, g, a64, wd, exact)).all()
    assert w.nbytes >= K * N // 2


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M", [6, 40])
def test_infinities_and_nans_stay_in_their_rows(ctx, torch_cuda, dtype, M):
    torch = torch_cuda
    from mojostream_b200.runtime import Q4GroupWeight
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(5)
    K, N, g = 256, 48, 32
    q, s, z = make_weight(rng, K, N, g, False)
    w = Q4GroupWeight(ctx, q, s, K, N, g)
    a = rows(torch, rng, M, K, 0, dt)
    a[1, 37] = math.inf
    a[3, 200] = math.nan
    a[4, 5], a[4, 6] = math.inf, -math.inf
    a[5, 255] = torch.finfo(dt).max / 2.0 ** 12
    c = torch.empty((M, N), dtype=dt, device="cuda")
    w.gemm(a, c)
    got = c.double().cpu().numpy()
    wd = dense(q, s, z, g)
    a64 = a.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        exact = a64 @ wd
    want = exact[1]
    zero = wd[37] == 0  # infinity times a weight of zero
    assert np.isnan(got[1][zero]).all() and (got[1][~zero] == np.sign(wd[37][~zero]) * math.inf).all(), want
    assert np.isnan(got[3]).all()
    assert not np.isfinite(got[4]).any()
    fine = [r for r in range(M) if r not in (1, 3, 4)]
    assert (np.abs(got[fine] - exact[fine]) <= bound(torch, dt, g, a64[fine], wd, exact[fine])).all()


def gated_exact(a64, wg, wu, act):
    g, u = a64 @ wg, a64 @ wu
    if act == "silu":
        f = g / (1 + np.exp(-g))
    else:
        f = 0.5 * g * (1 + np.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
    return g, u, f, f * u


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M,K,N,g,zeros,pad", [
    (1, 32, 2, 32, False, 0), (1, 2560, 640, 32, False, 0), (3, 96, 66, 32, True, 3),
    (4, 1280, 1030, 64, True, 0), (8, 256, 128, 128, False, 0), (13, 640, 98, 128, True, 5),
    (64, 512, 322, 128, True, 0), (133, 2560, 258, 64, False, 8),
])
def test_gated(ctx, torch_cuda, M, K, N, g, zeros, pad, act, dtype):
    """|f'| <= 1.13 for both activations, so the error of act(g) u is at most
    1.13 dg (|u| + du) + |f| du; the activation itself (an exp of an argument
    below 100 where it matters, a division) costs at most 128 u of |f|."""
    torch = torch_cuda
    from mojostream_b200.runtime import Q4GroupWeight
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(M + K + N)
    mats = [make_weight(rng, K, N, g, zeros, scale=0.01) for _ in range(2)]
    wg, wu = (Q4GroupWeight(ctx, q, s, K, N, g, zeros=z) for q, s, z in mats)
    a = rows(torch, rng, M, K, pad, dt)
    buf = torch.full((M + 1, N + pad + 1), 7.0, dtype=dt, device="cuda")
    h = buf[:M, :N]
    assert wg.gated(wu, a, h, act=act) is h
    ctx.sync(current=True)
    a64 = a.double().cpu().numpy()
    dg, du = (dense(q, s, z, g) for q, s, z in mats)
    with np.errstate(over="ignore"):
        gx, ux, f, exact = gated_exact(a64, dg, du, act)
    eg, eu = sums_bound(dtype, g, a64, dg), sums_bound(dtype, g, a64, du)
    tol = 1.13 * eg * (np.abs(ux) + eu) + np.abs(f) * eu + 128 * U * np.abs(exact)
    tol = rounded(torch, dt, tol, exact) + 2.0 ** -126
    got = h.double().cpu().numpy()
    over = np.abs(exact) > 65000 if dtype == "float16" else np.zeros_like(exact, bool)
    assert (np.abs(got - exact) <= tol)[~over].all(), float((np.abs(got - exact) / tol)[~over].max())
    assert (buf[M] == 7).all() and (buf[:, N:] == 7).all()


@pytest.mark.parametrize("M,dtype", [(1, "float32"), (1, "bfloat16"), (5, "bfloat16"), (48, "float32"),
                                     (300, "bfloat16")])
def test_other_streams_graphs_and_repeats(ctx, torch_cuda, M, dtype):
    """The same bits on every call: on the default stream, on another one, and
    in a captured graph that is replayed with new inputs."""
    torch = torch_cuda
    from mojostream_b200.runtime import Q4GroupWeight
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(11)
    K, N, g = 640, 200, 64
    q, s, z = make_weight(rng, K, N, g, True)
    w = Q4GroupWeight(ctx, q, s, K, N, g, zeros=z)
    inputs = [rows(torch, rng, M, K, 0, dt) for _ in range(3)]
    want = [w.gemm(a, torch.empty((M, N), dtype=dt, device="cuda")).clone() for a in inputs]
    again = w.gemm(inputs[0], torch.empty((M, N), dtype=dt, device="cuda"))
    assert torch.equal(again, want[0])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c = w.gemm(inputs[1], torch.empty((M, N), dtype=dt, device="cuda"))
    side.synchronize()
    assert torch.equal(c, want[1])
    a, c = inputs[0].clone(), torch.empty((M, N), dtype=dt, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.gemm(a, c)
    for x, y in zip(inputs, want):
        a.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c, y)


def test_workspace_growth_inside_a_capture_is_refused(torch_cuda):
    torch = torch_cuda
    from mojostream_b200 import MsError
    from mojostream_b200.runtime import Context, Q4GroupWeight
    c2 = Context(0)
    rng = np.random.default_rng(2)
    K, N, g = 2560, 64, 64
    q, s, _ = make_weight(rng, K, N, g, False)
    w = Q4GroupWeight(c2, q, s, K, N, g)
    a = torch.randn((1000, K), device="cuda")
    c = torch.empty((1000, N), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(MsError, match="MS_ERR_STATE"):
        with torch.cuda.graph(graph):
            w.gemm(a, c)
    w.gemm(a, c)  # outside the capture it grows
    want = c.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.gemm(a, c)
    b = torch.randn((4000, K), device="cuda")
    w.gemm(b, torch.empty((4000, N), device="cuda"))  # grows again: the graph keeps its buffer
    c.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c, want)
    del graph
    w.close()
    c2.close()


def test_refusals(ctx, torch_cuda):
    torch = torch_cuda
    from mojostream_b200 import _lib
    from mojostream_b200 import MsError
    from mojostream_b200.runtime import Q4GroupWeight
    rng = np.random.default_rng(1)
    q, s, z = make_weight(rng, 128, 64, 32, True)
    bad = z.copy()
    bad[2, 5] = 16
    with pytest.raises(MsError, match="zero point above 15"):
        Q4GroupWeight(ctx, q, s, 128, 64, 32, zeros=bad)
    w = Q4GroupWeight(ctx, q, s, 128, 64, 32, zeros=z)
    plain = Q4GroupWeight(ctx, q, s, 128, 64, 32)
    a, c = torch.zeros((2, 128), device="cuda"), torch.zeros((2, 64), device="cuda")
    L = _lib.lib()

    def call(w=w.h, C=c.data_ptr(), ldc=64, A=a.data_ptr(), lda=128, dtype=0, M=2):
        return _lib.STATUS_NAMES[L.ms_q4g_gemm(ctx.h, w, C, ldc, A, lda, dtype, M, 0, None)]

    assert call() == "MS_OK"
    assert call(M=0) == call(M=-1) == call(lda=127) == call(ldc=63) == "MS_ERR_SHAPE"
    assert call(dtype=3) == call(w=None) == call(A=None) == call(C=None) == "MS_ERR_INVALID_ARG"
    assert call(A=a.data_ptr() + 2) == "MS_ERR_ALIGN"
    host = np.zeros((2, 128), np.float32)
    assert call(A=host.ctypes.data) == "MS_ERR_INVALID_ARG"
    h = torch.zeros((2, 64), device="cuda")
    with pytest.raises(MsError, match="MS_ERR_SHAPE"):
        w.gated(plain, a, h)  # one with zero points, one without
    with pytest.raises(ValueError, match="act"):
        w.gated(w, a, h, act="relu")
    assert _lib.STATUS_NAMES[L.ms_q4g_gated(ctx.h, w.h, w.h, 2, h.data_ptr(), 64, a.data_ptr(), 128, 0, 2,
                                            None)] == "MS_ERR_INVALID_ARG"
    ctx.sync()
