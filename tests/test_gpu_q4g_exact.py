"""Group-scaled products whose results are known to the last bit: what each of
the two forms, of few rows and of many, holds of a value.  Weights are +1 and
-1 (a scale of 1), or 0, so that a result is one value of its row."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
# values that a group's largest leaves exact, in powers of two below it, and
# what any other value is held to, of the largest (few rows)
EXACT = {"float32": 21, "float16": 19, "bfloat16": 22}
HELD = {"float32": 45, "float16": 30, "bfloat16": 30}
FEW = {"float32": [1, 2, 3, 4, 5, 6, 8], "float16": [1, 2, 5, 8, 9, 16], "bfloat16": [1, 2, 3, 5, 8]}
MANY = {"float32": [9, 20, 70, 130, 300], "float16": [17, 40, 130, 300], "bfloat16": [9, 40, 130, 400]}
BITS = {"float32": 24, "float16": 11, "bfloat16": 8}
ROWS = [(d, m) for d in BITS for m in FEW[d] + MANY[d]]


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


def pack(w, z):
    """Integer weights [K][N] as bytes, q = w + z."""
    q = (w + z).astype(np.uint8)
    return q[:, 0::2] | (q[:, 1::2] << 4)


def weight(ctx, w, g, zeros, rng):
    """A weight of the integers w, scale 1."""
    from mojostream_b200.runtime import Q4GroupWeight
    K, N = w.shape
    z = rng.integers(1, 15, size=(K // g, N), dtype=np.uint8) if zeros else None
    zz = np.repeat(z, g, 0).astype(np.int64) if zeros else 8
    return Q4GroupWeight(ctx, pack(w, zz), np.ones((K // g, N), np.float16), K, N, g, zeros=z)


def mantissas(rng, n, dtype):
    """Values in [1, 2) with all bits of the type, the lowest set, of either sign."""
    m = rng.integers(0, 2 ** (BITS[dtype] - 2), size=n) * 2 + 1
    return (1 + m * 2.0 ** (1 - BITS[dtype])) * rng.choice([-1.0, 1.0], n)


def tensor(torch, x, dtype):
    """x, exactly."""
    t = torch.from_numpy(x.astype(np.float32)).cuda().to(getattr(torch, dtype))
    assert (t.double().cpu().numpy() == x).all()
    return t


@pytest.mark.parametrize("dtype,M", ROWS)
@pytest.mark.parametrize("g,zeros", [(32, True), (64, False), (128, True)])
def test_one_value_a_row(ctx, torch_cuda, dtype, M, g, zeros):
    """A row with one value among zeros: every result is plus or minus it."""
    torch = torch_cuda
    rng = np.random.default_rng(M + g)
    K, N = 384, 72
    w = rng.choice([-1, 1], size=(K, N))
    x, at = np.zeros((M, K)), rng.integers(0, K, M)
    at[-1] = K - 1
    spread = 12 if dtype == "float16" else 40
    x[np.arange(M), at] = mantissas(rng, M, dtype) * 2.0 ** rng.integers(-spread, spread, M)
    h = weight(ctx, w, g, zeros, rng)
    c = h.gemm(tensor(torch, x, dtype), torch.empty((M, N), dtype=getattr(torch, dtype), device="cuda"))
    assert (c.double().cpu().numpy() == x[np.arange(M), at][:, None] * w[at]).all()
    h.close()


@pytest.mark.parametrize("dtype,M", ROWS)
@pytest.mark.parametrize("g,zeros", [(32, False), (64, True), (128, False)])
def test_a_small_value_beside_a_large_one(ctx, torch_cuda, dtype, M, g, zeros):
    """In every group a large value meets weights of 0, and one value of the
    row, `gap` powers of two below, meets 1 and -1."""
    torch = torch_cuda
    rng = np.random.default_rng(M + g)
    K, N = 256, 40
    few = M in FEW[dtype]
    for gap in (3, EXACT[dtype], EXACT[dtype] + 1, 27, 29, 31) + ((40, 44, 50) if dtype != "float16" else ()):
        w = rng.choice([-1, 1], size=(K, N))
        w[::32] = 0
        x = np.zeros((M, K))
        up = 14 if dtype == "float16" else 20
        # the large ones do not round up to the next power of two
        x[:, ::32] = 2.0 ** up * rng.choice([-1.0, 1.0, 1.5], (M, K // 32))
        at = rng.integers(0, K // 32, M) * 32 + rng.integers(1, 32, M)
        small = mantissas(rng, M, dtype) * 2.0 ** (up - gap)
        if dtype == "float16":  # (its least step: fewer bits where the value is below 2^-14)
            small = np.round(small * 2.0 ** 24) / 2.0 ** 24
        x[np.arange(M), at] = small
        h = weight(ctx, w, g, zeros, rng)
        c = h.gemm(tensor(torch, x, dtype), torch.empty((M, N), dtype=getattr(torch, dtype), device="cuda"))
        got, want = c.double().cpu().numpy(), small[:, None] * w[at]
        if gap <= EXACT[dtype] or not few:
            assert (got == want).all(), gap
        else:
            largest = np.abs(x[:, ::32].reshape(M, K // g, -1)).max(2)[np.arange(M), at // g]
            # and half a step of the result's type
            tol = 2.0 ** -HELD[dtype] * largest[:, None] + 2.0 ** -BITS[dtype] * np.abs(want)
            assert (np.abs(got - want) <= tol).all(), gap
        h.close()


@pytest.mark.parametrize("M", [1, 3, 8, 9, 24, 80, 200])
def test_tiny_fp32_values(ctx, torch_cuda, M):
    """Of few rows to half a step of 2^-126 where that is more than 2^-45 of the
    largest; of many cut off to multiples of 2^-133, exact from 2^-110 up."""
    torch = torch_cuda
    rng = np.random.default_rng(M)
    K, N = 128, 34
    w = rng.choice([-1, 1], size=(K, N))
    h = weight(ctx, w, 64, True, rng)
    for e in (-100, -110, -112, -118, -124):
        x, at = np.zeros((M, K)), rng.integers(0, K, M)
        x[np.arange(M), at] = mantissas(rng, M, "float32") * 2.0 ** e
        c = h.gemm(tensor(torch, x, "float32"), torch.empty((M, N), device="cuda")).double().cpu().numpy()
        want = x[np.arange(M), at][:, None] * w[at]
        err = np.abs(c - want)
        if M <= 8:
            assert (err <= np.maximum(2.0 ** -127, 2.0 ** -45 * np.abs(want))).all(), e
        else:
            assert (err < 2.0 ** -133).all() and (e < -110 or not err.any()), e
    h.close()


@pytest.mark.parametrize("dtype", list(BITS))
@pytest.mark.parametrize("M", [4, 64, 512])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_activations(ctx, torch_cuda, dtype, M, act):
    """Rows with one value v, gate and up weights of 1: results act(v) v for v
    over the range of the exponential.  Relative errors: the exponent x takes up
    to four roundings (|x| 2^-24 each, as |x| 2^-24 of e^x), exponential,
    sum and quotient 2^-21 together, the product one; then half a step."""
    torch = torch_cuda
    rng = np.random.default_rng(M)
    K, N = 64, 2
    dt = getattr(torch, dtype)
    top = 80.0 if act == "silu" else 9.0
    for low in (1e-3, 0.1, 1.0, top / 2):
        v = rng.choice([-1.0, 1.0], M) * np.exp(rng.uniform(np.log(low), np.log(top), M))
        a = torch.zeros((M, K), device="cuda", dtype=dt)
        a[torch.arange(M), torch.from_numpy(rng.integers(0, K, M)).cuda()] = torch.from_numpy(v).cuda().to(dt)
        v = a.sum(1).double().cpu().numpy()
        w = weight(ctx, np.ones((K, N), np.int64), 64, False, rng)
        got = w.gated(w, a, torch.empty((M, N), dtype=dt, device="cuda"), act=act).double().cpu().numpy()
        x = v if act == "silu" else 2 * np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)
        want = v / (1 + np.exp(-x)) * v
        rel = 4 * np.abs(x) * 2.0 ** -24 + 2.0 ** -21
        assert rel.max() <= 2.0 ** -15 and (rel[np.abs(x) <= 8] <= 2.0 ** -18).all()
        tol = np.abs(want) * (rel + 2.0 ** -BITS[dtype]) + torch.finfo(dt).smallest_normal * 2.0 ** -BITS[dtype]
        assert (np.abs(got - want[:, None]) <= tol[:, None]).all(), low
        w.close()
