"""The operators of a decode step as they follow one another: a model's rows,
a gated feed-forward and a head with group-scaled 4-bit weights, the rules on
the head's logits, the sampler.  And products of several sizes back to back."""
import numpy as np
import pytest

from mojostream_b200.model import small_spec, synth_weights
from rules_check import reference, words
from test_gpu_q4g import U, bound, check, dense, gated_exact, make_weight, rounded, sums_bound
from test_gpu_q4g import test_gated as gated_case

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


@pytest.mark.parametrize("V", [5, 9000, 262144])
@pytest.mark.parametrize("value", [-np.inf, np.nan])
def test_a_row_without_a_candidate_gives_its_first_id(ctx, torch_cuda, V, value):
    """A mask can leave no id: the greedy id is then 0, as a scan that keeps
    the first maximum finds; rows beside it are not touched by that."""
    torch = torch_cuda
    lg = torch.full((3, V), value, dtype=torch.float32, device="cuda")
    lg[1] = 0
    lg[1, V - 2] = 1
    for pen in (1.0, 1.3):
        out = ctx.sample(lg, [[1], [1], []], 0.0, pen, [0, 0, 0]).cpu().tolist()
        assert out == [0, V - 2, 0]
    out = ctx.sample(lg, [[], [], []], 0.7, 1.0, [1, 2, 3]).cpu()
    assert ((out >= 0) & (out < V)).all()


@pytest.mark.parametrize("M,dtype", [(3, "float32"), (3, "bfloat16"), (24, "float32"), (24, "bfloat16")])
def test_chain(ctx, torch_cuda, M, dtype):
    """Each step against its definition in 64 bits on the inputs that the step
    before it wrote, and the whole again from a captured graph."""
    torch = torch_cuda
    from mojostream_b200.runtime import KVCache, LogitRules, Model, Q4GroupWeight
    dt = getattr(torch, dtype)
    spec = small_spec(vocab=4096, n_layers=2, window=32)
    model = Model(ctx, spec, synth_weights(spec, seed=5, symmetric=True), max_rows=32)
    kv = KVCache(ctx, model, M, 64, slide_cap=64)
    rng = np.random.default_rng(M)
    ids = rng.integers(0, spec.vocab, size=M).tolist()
    x = model.forward(model.embed(ids), kv, list(range(M)), [0] * M)
    K, F, V, g = spec.hidden, 1024, 2050, 64
    mats = [make_weight(rng, K, F, g, True, scale=0.01), make_weight(rng, K, F, g, True, scale=0.01),
            make_weight(rng, F, K, g, True, scale=0.01), make_weight(rng, K, V, g, False)]
    shapes = [(K, F), (K, F), (F, K), (K, V)]
    gate, up, down, head = (Q4GroupWeight(ctx, q, s, k, n, g, zeros=z)
                            for (q, s, z), (k, n) in zip(mats, shapes))
    hist = [rng.integers(0, V, size=5 + r).astype(np.int32) for r in range(M)]
    off = np.concatenate([[0], np.cumsum([len(h) for h in hist])]).astype(np.int32)
    allowed = rng.random((2, V)) < 0.3
    allowed[1] = False  # row 1 may say nothing
    arrays = dict(hist=np.concatenate(hist), hist_off=off, repetition=np.full(M, 1.2, np.float32),
                  presence=np.full(M, 0.1, np.float32), frequency=np.full(M, 0.05, np.float32),
                  mask=words(allowed), mask_row=np.array([0, 1] + [-1] * (M - 2), np.int32))
    rules = LogitRules(**{k: torch.from_numpy(v).cuda() for k, v in arrays.items()})
    x0 = x.to(dt)
    h = torch.empty((M, F), dtype=dt, device="cuda")
    y, lg = x0.clone(), torch.empty((M, V), dtype=dt, device="cuda")
    ruled = torch.empty_like(lg)

    def step():
        y.copy_(x0)
        gate.gated(up, x0, h)
        down.gemm(h, y, accumulate=True)
        head.gemm(y, lg)
        ctx.logit_rules(lg, rules, out=ruled)

    step()
    picked = ctx.sample(ruled.float(), [[]] * M, 0.0, 1.0, [0] * M).cpu().numpy()
    n64 = lambda t: t.double().cpu().numpy()
    wg, wu, wd, wh = (dense(q, s, z, g) for q, s, z in mats)
    a = n64(x0)
    gx, ux, f, exact = gated_exact(a, wg, wu, "silu")
    eg, eu = sums_bound(dtype, g, a, wg), sums_bound(dtype, g, a, wu)
    tol = rounded(torch, dt, 1.13 * eg * (np.abs(ux) + eu) + np.abs(f) * eu + 128 * U * np.abs(exact), exact)
    assert (np.abs(n64(h) - exact) <= tol).all()
    exact = n64(h) @ wd + a
    assert (np.abs(n64(y) - exact) <= bound(torch, dt, g, n64(h), wd, exact, a)).all()
    exact = n64(y) @ wh
    assert (np.abs(n64(lg) - exact) <= bound(torch, dt, g, n64(y), wh, exact)).all()
    want = torch.from_numpy(reference(lg.float().cpu().numpy(), **arrays)).to(dt)
    assert torch.equal(ruled.cpu(), want)
    assert picked[1] == 0 and (picked == want.float().numpy().argmax(1)).all()

    results = [t.clone() for t in (h, y, lg, ruled)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t in (h, y, lg, ruled):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for t, r in zip((h, y, lg, ruled), results):
        assert torch.equal(t, r)
    del graph


@pytest.mark.parametrize("op,M,K,N,g,zeros,dtype", [
    ("gemm", 1100, 2560, 5120, 128, False, "bfloat16"),  # more tiles than an SM holds at once
    ("gemm", 1100, 1280, 5120, 32, True, "bfloat16"),
    ("gemm", 520, 1280, 5120, 64, False, "float32"),
    ("gemm", 300, 1280, 10208, 64, True, "float16"),     # a half-empty last tile
    ("gated", 400, 1280, 5088, 64, False, "bfloat16"),
    ("gemm", 40, 2560, 2560, 128, True, "bfloat16"),     # k shared by clusters
    ("gemm", 4, 10240, 512, 64, False, "float32"),
])
def test_back_to_back(ctx, torch_cuda, op, M, K, N, g, zeros, dtype):
    """Calls with nothing between them give what each gives alone, bit by bit
    (a copy that overtook its reader showed up only so)."""
    torch = torch_cuda
    from mojostream_b200.runtime import Q4GroupWeight
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(N)

    def weight():
        q, s, z = make_weight(rng, K, N, g, zeros)
        return Q4GroupWeight(ctx, q, s, K, N, g, zeros=z)

    pairs = [(weight(), weight() if op == "gated" else None) for _ in range(2)]
    a = [torch.randn((M, K), device="cuda").to(dt) for _ in range(2)]

    def call(i, c):
        w, up = pairs[i]
        return w.gated(up, a[i], c) if up else w.gemm(a[i], c)

    alone = []
    for i in range(2):
        c = torch.empty((M, N), dtype=dt, device="cuda")
        torch.cuda.synchronize()
        call(i, c)
        torch.cuda.synchronize()
        alone.append(c)
    for _ in range(6):
        cs = [torch.empty((M, N), dtype=dt, device="cuda") for _ in range(6)]
        torch.cuda.synchronize()
        for j, c in enumerate(cs):
            call(j % 2, c)
        torch.cuda.synchronize()
        for j, c in enumerate(cs):
            assert torch.equal(c, alone[j % 2]), j


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("pad,accumulate", [
    (7, False),  # rows of the result start on 16-byte boundaries
    (2, False),  # and do not
    (7, True),
])
def test_more_tiles_than_sms(ctx, torch_cuda, dtype, pad, accumulate):
    """A CTA makes several tiles: whole ones, one whose columns end inside it
    and rows that do, against the definition."""
    check(torch_cuda, ctx, 1100, 256, 5136, 64, not accumulate, getattr(torch_cuda, dtype), pad,
          accumulate=accumulate)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("N,pad", [(3000, 7), (3010, 2)])
def test_more_gated_tiles_than_sms(ctx, torch_cuda, dtype, N, pad):
    gated_case(ctx, torch_cuda, 700, 256, N, 32, True, pad, "silu", dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_whole_and_cut_tiles_in_turns(ctx, torch_cuda, dtype):
    """One group of k a tile, so that warps may be a tile apart, and every
    third tile's columns end inside it."""
    for seed in range(4):
        check(torch_cuda, ctx, 40000, 128, 328, 128, True, getattr(torch_cuda, dtype), 7, seed=seed)
