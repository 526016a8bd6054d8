"""Rules on logits at the edges of what a caller may do."""
import numpy as np
import pytest

from rules_check import reference
from test_gpu_rules import logits_of, make, on_gpu, same

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


@pytest.mark.parametrize("M,V", [(1, 500), (5, 3001), (40, 70001)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_column_blocks_of_one_buffer(ctx, torch_cuda, M, V, dtype):
    """Logits and results side by side in one buffer share no byte; one column
    less between them, and they do."""
    torch = torch_cuda
    from mojostream_b200 import MsError
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(V)
    x = make(rng, M, V, 50, 5, 3)
    rules = on_gpu(torch, x)
    buf = torch.zeros((M, 2 * V), dtype=dt, device="cuda")
    buf[:, :V] = logits_of(torch, rng, M, V, 0, dt)
    before = buf[:, :V].clone()
    want = reference(before.float().cpu().numpy(), **x)
    got = ctx.logit_rules(buf[:, :V], rules, out=buf[:, V:])
    same(torch, got, want, dt)
    assert torch.equal(torch.nan_to_num(buf[:, :V]), torch.nan_to_num(before))
    with pytest.raises(MsError, match="overlaps"):
        ctx.logit_rules(buf[:, :V], rules, out=buf[:, V - 1:2 * V - 1])


@pytest.mark.parametrize("length", ["n_hist", "n_bias"])
def test_lists_longer_than_their_walk_are_refused(ctx, torch_cuda, length):
    """Indices of such a list would pass 2^31 behind its end: refused before
    any launch, so nothing of the (short) list is read."""
    torch = torch_cuda
    from mojostream_b200 import MsError
    rng = np.random.default_rng(1)
    rules = on_gpu(torch, make(rng, 2, 100, 5, 5, 0))
    lg = torch.zeros((2, 100), device="cuda")
    for n in (2 ** 31 - 1, 2 ** 31 - 65536):
        setattr(rules.desc, length, n)
        with pytest.raises(MsError, match="MS_ERR_SHAPE.*list lengths"):
            ctx.logit_rules(lg, rules)
    assert not lg.any()
