"""Rules on logits (ms_logit_rules_apply) against the same operations in NumPy
float32: every step is one IEEE-rounded operation, so the results are equal
bit for bit, and 16-bit logits are that value rounded once."""
import numpy as np
import pytest

from rules_check import reference, words

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


def make(rng, M, V, hist, bias, masks):
    x = {}
    if hist:
        lens = rng.integers(0, hist + 1, size=M)
        lens[0] = hist
        off = np.zeros(M + 1, np.int32)
        off[1:] = lens.cumsum()
        ids = (rng.random(off[-1]) ** 3 * V).astype(np.int32)
        ids[rng.random(len(ids)) < 0.05] = V + 7   # outside: skipped
        ids[rng.random(len(ids)) < 0.05] = -3
        x.update(hist=ids, hist_off=off, repetition=(1 + rng.random(M)).astype(np.float32),
                 presence=rng.random(M).astype(np.float32), frequency=rng.random(M).astype(np.float32))
    if bias:
        off = (np.arange(M + 1) * bias).astype(np.int32)
        ids = rng.integers(0, V, size=M * bias).astype(np.int32)
        val = (rng.random(M * bias) * 20 - 10).astype(np.float32)
        if bias > 3:  # an id listed twice, one outside, an infinite bias
            ids[1::bias] = ids[0::bias]
            ids[2::bias] = V
            val[3::bias] = -np.inf
        x.update(bias_id=ids, bias_val=val, bias_off=off)
    if masks:
        allowed = rng.random((masks, V)) < np.array([0.9, 0.01, 0.5, 0.0])[np.arange(masks) % 4][:, None]
        row = rng.integers(-1, masks, size=M).astype(np.int32)
        row[M // 2] = masks + 3  # no such mask: the row is free
        x.update(mask=words(allowed), mask_row=row)
    return x


def on_gpu(torch, x):
    from mojostream_b200.runtime import LogitRules
    return LogitRules(**{k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in x.items()})


def logits_of(torch, rng, M, V, pad, dtype):
    lg = (rng.standard_normal((M, V + pad)) * 4).astype(np.float32)
    t = torch.from_numpy(lg).cuda().to(dtype)
    v = t[:, :V]
    if V > 8:
        v[0, 1], v[0, 2], v[0, 3], v[0, 4] = np.inf, -np.inf, np.nan, 0.0
    return v


def same(torch, got, want32, dtype):
    want = torch.from_numpy(want32).to(dtype)
    g = got.cpu()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(g), nan)
    assert torch.equal(g[~nan], want[~nan])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("M,V,pad,hist,bias,masks", [
    (1, 1, 0, 3, 1, 1), (1, 31, 0, 5, 2, 2), (2, 33, 1, 0, 0, 3), (3, 1000, 0, 50, 0, 0),
    (5, 8192, 8, 0, 7, 0), (4, 8193, 0, 300, 5, 4), (37, 32003, 13, 700, 5, 9), (1, 262144, 0, 500, 8, 1),
    (9, 100001, 3, 5000, 60, 5), (2, 4096, 0, 0, 0, 0),
    # many columns: the stream and the lists in kernels of their own
    (64, 65536, 0, 300, 9, 7), (40, 70001, 5, 20000, 100, 3), (31, 100003, 1, 40, 0, 0),
    (70, 50000, 0, 0, 30, 2), (48, 60000, 0, 0, 0, 5),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_rules(ctx, torch_cuda, M, V, pad, hist, bias, masks, dtype, in_place):
    torch = torch_cuda
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(M * 3 + V)
    x = make(rng, M, V, hist, bias, masks)
    lg = logits_of(torch, rng, M, V, pad, dt)
    want = reference(lg.float().cpu().numpy(), **x)
    rules = on_gpu(torch, x)
    if in_place:
        got = ctx.logit_rules(lg, rules)
        assert got is lg
    else:
        before = lg.clone()
        buf = torch.full((M + 1, V + 5), 3.0, dtype=dt, device="cuda")
        got = ctx.logit_rules(lg, rules, out=buf[:M, :V])
        torch.cuda.synchronize()
        assert (buf[M] == 3).all() and (buf[:, V:] == 3).all()
        assert torch.equal(torch.nan_to_num(lg), torch.nan_to_num(before))
    same(torch, got, want, dt)


@pytest.mark.parametrize("M,V", [(6, 3000), (50, 60001)])
def test_each_part_alone_and_masks_by_row(ctx, torch_cuda, M, V):
    torch = torch_cuda
    rng = np.random.default_rng(4)
    x = make(rng, M, V, 100, 6, M)
    lg = logits_of(torch, rng, M, V, 0, torch.float32)
    for keep in (("hist", "hist_off"), ("hist", "hist_off", "repetition"),
                 ("hist", "hist_off", "presence"), ("hist", "hist_off", "frequency"),
                 ("bias_id", "bias_val", "bias_off"), ("mask",), ("mask", "mask_row")):
        part = {k: x[k] for k in keep}
        got = ctx.logit_rules(lg, on_gpu(torch, part), out=torch.empty_like(lg))
        same(torch, got, reference(lg.cpu().numpy(), **part), torch.float32)


@pytest.mark.parametrize("in_place", [False, True])
def test_more_distinct_ids_than_a_table_holds(ctx, torch_cuda, in_place):
    """Every id of a large vocabulary in one row's history, some often: each
    is penalised once, whatever tables the ids pass through."""
    torch = torch_cuda
    rng = np.random.default_rng(9)
    M, V = 20, 150000
    ids = [np.arange(V), rng.integers(0, V, 30000), np.repeat(rng.integers(0, V, 3), 70000),
           8 * rng.integers(0, V // 8, 20000), 16384 * rng.integers(0, V // 16384, 500)]
    ids += [rng.integers(0, V, 50) for _ in range(M - len(ids))]
    off = np.cumsum([0] + [len(i) for i in ids]).astype(np.int32)
    x = dict(hist=np.concatenate(ids).astype(np.int32), hist_off=off,
             repetition=np.full(M, 1.25, np.float32), presence=np.full(M, 0.5, np.float32),
             frequency=np.full(M, 0.125, np.float32),
             bias_id=np.tile(np.arange(0, V, 40, dtype=np.int32), M),
             bias_val=rng.random(M * (V // 40)).astype(np.float32),
             bias_off=(np.arange(M + 1) * (V // 40)).astype(np.int32))
    lg = logits_of(torch, rng, M, V, 0, torch.float32)
    want = reference(lg.cpu().numpy(), **x)
    got = ctx.logit_rules(lg, on_gpu(torch, x), out=None if in_place else torch.empty_like(lg))
    same(torch, got, want, torch.float32)


def test_offsets_are_clamped(ctx, torch_cuda):
    """Offsets that leave the lists (a host's mistake) read nothing outside."""
    torch = torch_cuda
    rng = np.random.default_rng(5)
    M, V = 4, 500
    x = make(rng, M, V, 40, 5, 0)
    n = len(x["hist"])
    x["hist_off"] = np.array([-5, n + 100, 3, 2, n], np.int32)
    x["bias_off"] = np.array([0, 1000, -7, 5, 20], np.int32)
    lg = logits_of(torch, rng, M, V, 0, torch.float32)
    got = ctx.logit_rules(lg, on_gpu(torch, x), out=torch.empty_like(lg))
    same(torch, got, reference(lg.cpu().numpy(), **x), torch.float32)


def test_replayed_graph_reads_the_lists_again(ctx, torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(6)
    M, V = 3, 9000
    x = make(rng, M, V, 200, 4, 3)
    rules = on_gpu(torch, x)
    lg = logits_of(torch, rng, M, V, 0, torch.float32)
    out = torch.empty_like(lg)
    ctx.logit_rules(lg, rules, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.logit_rules(lg, rules, out=out)
    x["mask_row"] = np.array([2, -1, 0], np.int32)
    x["hist"] = np.roll(x["hist"], 17)
    rules.tensors["mask_row"].copy_(torch.from_numpy(x["mask_row"]))
    rules.tensors["hist"].copy_(torch.from_numpy(x["hist"]))
    graph.replay()
    torch.cuda.synchronize()
    same(torch, out, reference(lg.cpu().numpy(), **x), torch.float32)


def test_refusals(ctx, torch_cuda):
    torch = torch_cuda
    from mojostream_b200 import MsError
    from mojostream_b200.runtime import LogitRules
    z = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
    lg = z(2, 64, dt=torch.float32)
    ok = LogitRules(mask=z(1, 2), mask_row=z(2))
    ctx.logit_rules(lg, ok)
    with pytest.raises(ValueError, match="words"):
        ctx.logit_rules(z(2, 65, dt=torch.float32), ok)
    with pytest.raises(ValueError, match="masks for 2 rows"):
        ctx.logit_rules(lg, LogitRules(mask=z(1, 2)))
    with pytest.raises(ValueError, match="offsets"):
        ctx.logit_rules(lg, LogitRules(hist=z(4), hist_off=z(4)))
    with pytest.raises(ValueError, match="go together"):
        LogitRules(hist=z(4))
    with pytest.raises(ValueError, match="penalties need"):
        LogitRules(presence=z(2, dt=torch.float32))
    with pytest.raises(ValueError, match="torch.int32"):
        LogitRules(hist=z(4, dt=torch.int64), hist_off=z(3))
    with pytest.raises(ValueError, match="values for 2 rows"):
        ctx.logit_rules(lg, LogitRules(hist=z(4), hist_off=z(3), presence=z(3, dt=torch.float32)))
    big = z(3, 64, dt=torch.float32)
    with pytest.raises(MsError, match="overlaps"):
        ctx.logit_rules(big[:2], ok, out=big[1:])
    with pytest.raises(ValueError, match="out"):
        ctx.logit_rules(lg, ok, out=z(2, 64, dt=torch.bfloat16))
    with pytest.raises(ValueError, match="shape"):
        ctx.logit_rules(lg, ok, out=z(2, 63, dt=torch.float32))
