"""Cases for the operators between a hidden row and a token id: products with 4-bit weights that
have a scale (and a zero point) per group of k, the gated feed-forward half on two such weights,
and the rules on logits (repetition, presence and frequency penalties, biases, grammar masks).

Weights are bytes [K][N / 2], low nibble = even column, w[k][n] = (q - z) * s with s (and z) of the
group k // g; without zero points z = 8.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token through a hybrid layer's query projection: the smallest product, latency counts
        {"name": "product 1 row, query", "op": "product", "M": 1, "K": 2560, "N": 2048, "g": 32,
         "zeros": False, "dtype": "f32", "pad": 0},
        # four sequences through a down projection
        {"name": "product 4 rows, down", "op": "product", "M": 4, "K": 10240, "N": 2560, "g": 64,
         "zeros": False, "dtype": "f32", "pad": 0},
        # one token's logits from a 4-bit head
        {"name": "product 1 row, head", "op": "product", "M": 1, "K": 2560, "N": 262144, "g": 128,
         "zeros": False, "dtype": "bf16", "pad": 0},
        # a decode batch through a larger model's down projection, with zero points
        {"name": "product 16 rows, zeros", "op": "product", "M": 16, "K": 13824, "N": 5120, "g": 128,
         "zeros": True, "dtype": "bf16", "pad": 0},
        # odd sizes: k that ends inside a 64-k piece, columns that end inside a tile, strided rows
        {"name": "product 7 rows, odd", "op": "product", "M": 7, "K": 2592, "N": 1030, "g": 32,
         "zeros": True, "dtype": "f16", "pad": 24},
        # a prompt chunk through the gate projection
        {"name": "product 2048 rows", "op": "product", "M": 2048, "K": 2560, "N": 10240, "g": 128,
         "zeros": False, "dtype": "bf16", "pad": 0},
        # one token through a feed-forward block's first half
        {"name": "gated 1 row", "op": "gated", "M": 1, "K": 2560, "N": 10240, "g": 32,
         "zeros": False, "dtype": "f32", "pad": 0, "act": "silu"},
        # the batch-64 decode step of the larger model
        {"name": "gated 64 rows", "op": "gated", "M": 64, "K": 5120, "N": 13824, "g": 128,
         "zeros": True, "dtype": "bf16", "pad": 0, "act": "gelu_tanh"},
        # a ragged prompt
        {"name": "gated 519 rows, ragged", "op": "gated", "M": 519, "K": 2560, "N": 10240, "g": 64,
         "zeros": False, "dtype": "bf16", "pad": 0, "act": "silu"},
        # one request: a short history, a few biases, one grammar state
        {"name": "rules 1 row", "op": "rules", "M": 1, "V": 262144, "hist": 500, "bias": 8,
         "masks": 1, "dtype": "f32", "pad": 0},
        # a full decode batch with long histories
        {"name": "rules 64 rows", "op": "rules", "M": 64, "V": 262144, "hist": 4096, "bias": 32,
         "masks": 16, "dtype": "f32", "pad": 0},
        # an odd vocabulary in 16 bits, rows of another stride, a mask that leaves a row empty
        {"name": "rules 37 rows, odd", "op": "rules", "M": 37, "V": 32003, "hist": 700, "bias": 5,
         "masks": 9, "dtype": "bf16", "pad": 13},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["product", "product", "gated", "rules"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    pad = rng.choice([0, 0, 8, 13])
    if op == "rules":
        M = _log_int(rng, 1, 128)
        V = _log_int(rng, 1000, 262144)
        return {"op": op, "M": M, "V": min(V, 16000000 // M), "hist": _log_int(rng, 1, 4096),
                "bias": rng.randrange(0, 64), "masks": rng.randrange(0, 20), "dtype": dtype, "pad": pad}
    g = rng.choice([32, 64, 128])
    K = g * max(1, _log_int(rng, 256, 13824) // g)
    N = 2 * _log_int(rng, 64, 16384)
    M = _log_int(rng, 1, 2048)
    if rng.random() < 0.5:
        M = rng.randrange(1, 17)
    M = max(1, min(M, 50_000_000_000 // (K * N * (2 if op == "gated" else 1))))
    case = {"op": op, "M": M, "K": K, "N": N, "g": g, "zeros": rng.random() < 0.5, "dtype": dtype, "pad": pad}
    if op == "gated":
        case["act"] = rng.choice(["silu", "gelu_tanh"])
    return case


# ------------------------------------------------------------------- inputs --

def _weight_inputs(case, gen):
    """Bytes, group scales and zero points of one weight, as a checkpoint holds them: values of
    unit variance over sqrt(K) spread over 16 levels, zero points around the middle."""
    K, N, g = case["K"], case["N"], case["g"]
    q = torch.randint(0, 256, (K, N // 2), dtype=torch.uint8, device="cuda", generator=gen)
    s = (0.5 + torch.rand((K // g, N), device="cuda", generator=gen)) * (0.2 / math.sqrt(K))
    z = None
    if case["zeros"]:
        z = torch.randint(4, 13, (K // g, N), dtype=torch.uint8, device="cuda", generator=gen)
    return q, s.to(torch.float16), z


def _product_inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    M, K, N, pad = case["M"], case["K"], case["N"], case["pad"]
    dt = _TYPES[case["dtype"]]
    a = torch.randn((M, K + pad), device="cuda", generator=gen)
    # a few channels are much larger than the rest, as hidden rows have them
    big = torch.randint(0, K, (max(1, K // 256),), device="cuda", generator=gen)
    a[:, big] *= 20.0
    a = a.to(dt)[:, :K]
    out = torch.empty((M, N + pad), dtype=dt, device="cuda")[:, :N]
    weights = [_weight_inputs(case, gen) for _ in range(2 if case["op"] == "gated" else 1)]
    return a, out, weights


def _rules_inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    M, V, pad = case["M"], case["V"], case["pad"]
    dt = _TYPES[case["dtype"]]
    r = lambda *shape: torch.rand(shape, device="cuda", generator=gen)  # noqa: E731
    logits = (torch.randn((M, V + pad), device="cuda", generator=gen) * 3.0).to(dt)[:, :V]
    out = torch.empty((M, V + pad), dtype=dt, device="cuda")[:, :V]
    lens = (r(M) * case["hist"]).to(torch.int64) + 1
    if M > 2:
        lens[1] = 0  # a request with no history yet
    off = torch.zeros(M + 1, dtype=torch.int64, device="cuda")
    off[1:] = lens.cumsum(0)
    # ids repeat as words do: a power of a uniform number crowds the low ids
    hist = (r(int(off[-1])) ** 4 * V).to(torch.int32).clamp_(0, V - 1)
    nb = case["bias"]
    x = {"logits": logits, "out": out, "hist": hist, "hist_off": off.to(torch.int32),
         "repetition": 1.0 + 0.3 * r(M), "presence": r(M), "frequency": 0.5 * r(M),
         "bias_id": None, "bias_val": None, "bias_off": None, "mask": None, "mask_row": None}
    if nb:
        x["bias_id"] = (r(M * nb) * V).to(torch.int32).clamp_(0, V - 1)
        x["bias_val"] = r(M * nb) * 20.0 - 10.0
        x["bias_off"] = torch.arange(M + 1, dtype=torch.int32, device="cuda") * nb
    n = case["masks"]
    if n:
        words = (V + 31) // 32
        mask = torch.empty((n, words), dtype=torch.int32, device="cuda")
        for i in range(n):
            # a state inside a string allows most ids, one between tokens very few
            keep = (0.95, 0.002, 0.3, 0.0)[i % 4]
            bits = (r(words, 32) < keep).to(torch.int64) << torch.arange(32, device="cuda")
            mask[i] = bits.sum(1).to(torch.int32)
        x["mask"] = mask
        # several rows share a state; every fifth row is free
        row = (r(M) * n).to(torch.int32).clamp_(0, n - 1)
        row[4::5] = -1
        x["mask_row"] = row
    return x


_context = None


def _ctx():
    global _context
    if _context is None:
        from mojostream_b200.runtime import Context
        _context = Context(0)
    return _context


def prepare(case, seed):
    if case["op"] == "rules":
        state = {"case": case, **_rules_inputs(case, seed)}
        if own:
            from mojostream_b200.runtime import LogitRules
            state["ctx"] = _ctx()
            state["rules"] = LogitRules(**{k: state[k] for k in (
                "hist", "hist_off", "repetition", "presence", "frequency", "bias_id", "bias_val",
                "bias_off", "mask", "mask_row")})
        return state
    a, out, weights = _product_inputs(case, seed)
    state = {"case": case, "a": a, "out": out, "weights": weights}
    if own:
        from mojostream_b200.runtime import Q4GroupWeight
        state["handles"] = [Q4GroupWeight(_ctx(), q, s, case["K"], case["N"], case["g"], zeros=z)
                            for q, s, z in weights]
    return state


# -------------------------------------------------------------- plain forms --

def _dequant(q, s, z, g):
    K, half = q.shape
    v = torch.stack((q & 15, q >> 4), dim=2).view(K // g, g, 2 * half).float()
    v -= 8.0 if z is None else z.float().unsqueeze(1)
    v *= s.float().unsqueeze(1)
    return v.view(K, 2 * half)


def _plain_product(state):
    q, s, z = state["weights"][0]
    return (state["a"].float() @ _dequant(q, s, z, state["case"]["g"])).to(state["a"].dtype)


def _plain_gated(state):
    a, g = state["a"].float(), state["case"]["g"]
    gate, up = (a @ _dequant(q, s, z, g) for q, s, z in state["weights"])
    if state["case"]["act"] == "silu":
        act = gate / (1.0 + torch.exp(-gate))
    else:
        act = 0.5 * gate * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate * gate * gate)))
    return (act * up).to(state["a"].dtype)


def _rows(off, n):
    M = off.numel() - 1
    return torch.repeat_interleave(torch.arange(M, device=off.device), (off[1:] - off[:-1]).long(), output_size=n)


def _plain_rules(state):
    logits = state["logits"]
    M, V = logits.shape
    v = logits.float()
    hist = state["hist"]
    count = torch.zeros((M, V), device=v.device)
    count.view(-1).index_add_(0, _rows(state["hist_off"], hist.numel()) * V + hist,
                              torch.ones(hist.numel(), device=v.device))
    rep, pres, freq = (state[k].unsqueeze(1) for k in ("repetition", "presence", "frequency"))
    seen = count > 0
    v = torch.where(seen, torch.where(v > 0, v / rep, v * rep) - (pres + freq * count), v)
    if state["bias_id"] is not None:
        n = state["bias_id"].numel()
        at = torch.full((M * V,), -1, dtype=torch.int64, device=v.device)
        at.scatter_reduce_(0, _rows(state["bias_off"], n) * V + state["bias_id"],
                           torch.arange(n, device=v.device), "amax")
        at = at.view(M, V)
        v = torch.where(at >= 0, v + state["bias_val"][at.clamp(min=0)], v)
    if state["mask"] is not None:
        words, row = state["mask"], state["mask_row"].long()
        bits = (words.unsqueeze(2) >> torch.arange(32, dtype=torch.int32, device=v.device)) & 1
        allowed = bits.view(words.shape[0], -1)[row.clamp(min=0), :V].bool() | (row < 0).unsqueeze(1)
        v = torch.where(allowed, v, torch.full_like(v, -math.inf))
    return v.to(logits.dtype)


def run(state):
    op = state["case"]["op"]
    if own:
        if op == "product":
            return state["handles"][0].gemm(state["a"], state["out"])
        if op == "gated":
            gate, up = state["handles"]
            return gate.gated(up, state["a"], state["out"], act=state["case"]["act"])
        return state["ctx"].logit_rules(state["logits"], state["rules"], out=state["out"])
    return {"product": _plain_product, "gated": _plain_gated, "rules": _plain_rules}[op](state)


# -------------------------------------------------------------- definitions --

def _exact_product(a, weight, g):
    """sum_k a[m,k] (q[k,n] - z) s, in 64 bits, 4096 columns at a time."""
    q, s, z = weight
    K, N = q.shape[0], 2 * q.shape[1]
    group = torch.arange(K, device=q.device) // g
    a64, parts = a.double(), []
    for n0 in range(0, N, 4096):
        cols = torch.arange(n0, min(N, n0 + 4096), device=q.device)
        byte = q[:, cols // 2].long()
        value = (byte // (1 + 15 * (cols % 2))) % 16
        zero = 8.0 if z is None else z[:, cols][group].double()
        parts.append(a64 @ ((value.double() - zero) * s[:, cols].double()[group]))
    return torch.cat(parts, dim=1)


def exact(case, seed):
    if case["op"] == "rules":
        x = _rules_inputs(case, seed)
        y = x["logits"].double().cpu().numpy().copy()
        M, V = y.shape
        host = {k: (None if t is None else t.cpu().numpy()) for k, t in x.items() if k not in ("logits", "out")}
        for r in range(M):
            ids = host["hist"][host["hist_off"][r]:host["hist_off"][r + 1]]
            seen = {}
            for j in ids.tolist():
                seen[j] = seen.get(j, 0) + 1
            rep, pres, freq = (float(host[k][r]) for k in ("repetition", "presence", "frequency"))
            for j, c in seen.items():
                v = y[r, j]
                y[r, j] = (v / rep if v > 0 else v * rep) - (pres + freq * c)
            if host["bias_id"] is not None:
                span = slice(host["bias_off"][r], host["bias_off"][r + 1])
                for j, b in dict(zip(host["bias_id"][span].tolist(), host["bias_val"][span].tolist())).items():
                    y[r, j] += b
            if host["mask"] is not None and host["mask_row"][r] >= 0:
                bits = host["mask"][host["mask_row"][r]].view("uint32")
                for b in range(32):
                    cols = y[r, b::32]
                    cols[(bits[:cols.size] >> b) % 2 == 0] = -math.inf
        return torch.from_numpy(y)
    a, _, weights = _product_inputs(case, seed)
    y = [_exact_product(a, w, case["g"]) for w in weights]
    if case["op"] == "product":
        return y[0]
    gate, up = y
    if case["act"] == "silu":
        return gate * torch.sigmoid(gate) * up
    c = math.sqrt(2.0 / math.pi)
    return gate * torch.sigmoid(2.0 * c * (gate + 0.044715 * gate ** 3)) * up


def work(case):
    M = case["M"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rules":
        V, n = case["V"], case["masks"]
        # a fifth of the rows is free, the rest keeps what the masks keep
        share = 1.0
        if n:
            kept = sum((0.95, 0.002, 0.3, 0.0)[i % 4] for i in range(n)) / n
            share = kept if M < 5 else 0.2 + 0.8 * kept
        read = share * M * V * size + n * 4 * ((V + 31) // 32) + M * (2 * case["hist"] + 8 * case["bias"] + 12)
        return {"bytes": read + M * V * size, "flops": M * V}
    K, N = case["K"], case["N"]
    many = 2 if case["op"] == "gated" else 1
    weights = many * (K * N // 2 + (3 if case["zeros"] else 2) * (K // case["g"]) * N)
    return {"bytes": weights + M * (K + N) * size, "flops": 2 * M * K * N * many}
