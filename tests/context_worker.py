"""Contexts made by several threads at once, as the first thing of a process:
each thread's product, whose k a cluster shares, as a hash of its bits."""
import hashlib
import sys
import threading

import numpy as np
import torch

from mojostream_b200.runtime import Context, Q4GroupWeight


def main(n):
    torch.cuda.init()
    rng = np.random.default_rng(1)
    K, N, g, M = 13824, 640, 128, 16
    q = rng.integers(0, 256, size=(K, N // 2), dtype=np.uint8)
    s = (0.01 * (0.5 + rng.random((K // g, N)))).astype(np.float16)
    a = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).cuda().to(torch.bfloat16)
    torch.cuda.synchronize()
    start, found, errors = threading.Barrier(n), [None] * n, []

    def work(i):
        try:
            start.wait()
            ctx = Context(0)
            with torch.cuda.stream(torch.cuda.Stream()):
                w = Q4GroupWeight(ctx, q, s, K, N, g)
                c = w.gemm(a, torch.empty((M, N), dtype=torch.bfloat16, device="cuda"))
                ctx.sync(current=True)
            found[i] = hashlib.sha256(c.float().cpu().numpy().tobytes()).hexdigest()
            w.close()
            ctx.close()
        except Exception as e:  # reported by the parent
            errors.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    print(" ".join(found))


if __name__ == "__main__":
    main(int(sys.argv[1]))
