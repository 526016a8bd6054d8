"""Group-scaled products on several streams and in several graphs at once: each
gives what it gives alone, bit by bit."""
import gc

import numpy as np
import pytest

from test_gpu_q4g import make_weight

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


# rows that are converted by a kernel of their own, and limb planes
CASES = [(7, 4096, 512, "float32"), (6, 5120, 256, "bfloat16"), (16, 2560, 256, "float16"),
         (40, 2560, 512, "bfloat16"), (300, 1280, 640, "float32")]


def jobs(torch, ctx, M, K, N, dtype, n):
    """n inputs, results and what each result is when nothing else runs."""
    from mojostream_b200.runtime import Q4GroupWeight
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(M)
    q, s, z = make_weight(rng, K, N, 64, True)
    w = Q4GroupWeight(ctx, q, s, K, N, 64, zeros=z)
    a = [torch.randn((M, K), device="cuda").to(dt) for _ in range(n)]
    alone = []
    for x in a:
        alone.append(w.gemm(x, torch.empty((M, N), dtype=dt, device="cuda")))
        torch.cuda.synchronize()
    return w, a, alone, [torch.empty_like(y) for y in alone]


@pytest.mark.parametrize("M,K,N,dtype", CASES)
def test_streams_at_once(ctx, torch_cuda, M, K, N, dtype):
    torch = torch_cuda
    w, a, alone, out = jobs(torch, ctx, M, K, N, dtype, 3)
    streams = [torch.cuda.Stream() for _ in a]
    for _ in range(30):
        for y in out:
            y.zero_()
        torch.cuda.synchronize()
        for _ in range(8):
            for s, x, y in zip(streams, a, out):
                with torch.cuda.stream(s):
                    w.gemm(x, y)
        torch.cuda.synchronize()
        for y, want in zip(out, alone):
            assert torch.equal(y, want)


@pytest.mark.parametrize("M,K,N,dtype", CASES)
def test_graphs_at_once(ctx, torch_cuda, M, K, N, dtype):
    """Two graphs, captured one after the other from one stream, run beside
    each other and beside calls outside of them."""
    torch = torch_cuda
    w, a, alone, out = jobs(torch, ctx, M, K, N, dtype, 3)
    graphs = []
    for x, y in zip(a[:2], out[:2]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(8):
                w.gemm(x, y)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in a]
    for _ in range(30):
        for y in out:
            y.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            for _ in range(8):
                w.gemm(a[2], out[2])
        torch.cuda.synchronize()
        for y, want in zip(out, alone):
            assert torch.equal(y, want)
    del graphs, g


def test_one_capture_over_two_streams(ctx, torch_cuda):
    torch = torch_cuda
    w, a, alone, out = jobs(torch, ctx, 7, 4096, 512, "float32", 2)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(8):
            w.gemm(a[0], out[0])
            with torch.cuda.stream(side):
                w.gemm(a[1], out[1])
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(30):
        for y in out:
            y.zero_()
        g.replay()
        torch.cuda.synchronize()
        for y, want in zip(out, alone):
            assert torch.equal(y, want)
    del g


def test_graphs_that_end_give_their_workspace_back(torch_cuda):
    torch = torch_cuda
    from mojostream_b200.runtime import Context, Q4GroupWeight
    c2 = Context(0)
    rng = np.random.default_rng(2)
    K, N = 5120, 64
    q, s, _ = make_weight(rng, K, N, 64, False)
    w = Q4GroupWeight(c2, q, s, K, N, 64)
    a, c = torch.randn((4000, K), device="cuda"), torch.empty((4000, N), device="cuda")
    want = w.gemm(a, c).clone()  # 120 MB of planes
    free = []
    for _ in range(40):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            w.gemm(a, c)
        c.zero_()
        g.replay()
        del g  # (its execution may still run)
        gc.collect()
        torch.cuda.synchronize()
        assert torch.equal(c, want)
        free.append(torch.cuda.mem_get_info()[0])
    assert free[-1] > free[3] - 300e6  # 36 graphs took 4.5 GB, if each kept its own
    w.close()
    c2.close()


def test_many_streams_share_a_few_workspaces(torch_cuda):
    """More streams than workspaces are kept for: the right results still."""
    torch = torch_cuda
    from mojostream_b200.runtime import Context
    c2 = Context(0)
    w, a, alone, out = jobs(torch, c2, 7, 4096, 512, "float32", 24)
    streams = [torch.cuda.Stream() for _ in a]
    for _ in range(3):
        for s, x, y in zip(streams, a, out):
            with torch.cuda.stream(s):
                w.gemm(x, y)
        torch.cuda.synchronize()
        for y, want in zip(out, alone):
            assert torch.equal(y, want)
            y.zero_()
    w.close()
    c2.close()


@pytest.mark.parametrize("M,K,N,dtype", [(1, 2560, 20480, "bfloat16"), (1, 5120, 4096, "float32"),
                                         (4, 10240, 2560, "bfloat16"), (3, 5120, 4096, "float32")])
def test_few_rows_beside_many(ctx, torch_cuda, M, K, N, dtype):
    """Decode calls while another stream's products of 64 rows keep the SMs'
    shared memory busy, so that loads from a ring's stages take longest when
    the stages are refilled."""
    torch = torch_cuda
    w, a, alone, out = jobs(torch, ctx, M, K, N, dtype, 2)
    w2, a2, alone2, out2 = jobs(torch, ctx, 64, 5120, 2048, "bfloat16", 1)
    one, other = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(30):
        for y in out + out2:
            y.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            for _ in range(10):
                w2.gemm(a2[0], out2[0])
        with torch.cuda.stream(one):
            for _ in range(8):
                for x, y in zip(a, out):
                    w.gemm(x, y)
        torch.cuda.synchronize()
        for y, want in zip(out + out2, alone + alone2):
            assert torch.equal(y, want)
