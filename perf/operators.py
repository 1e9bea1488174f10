"""The 8-bit activation path and the mixture-of-experts layer, as workloads to measure.

Four operators, each in its plain form (elementary torch operations) and, with ``own`` set, as this framework's
calls: the RMSNorm with the residual's addition (8-bit or 16-bit output), SwiGLU with an 8-bit output, the product of
8-bit rows with int8 weights, and a whole mixture-of-experts layer for a few tokens.
"""

import torch

own = False

EPS = 1e-6


def listed():
    return [
        # one token of a decoder of width 4096: launch latency
        {"name": "norm int8 1x4096", "op": "norm", "M": 1, "K": 4096, "dtype": "float16", "int8": True, "pad": 0},
        # a prompt of 2048 tokens in front of the 8-bit gate/up product
        {"name": "norm int8 2048x4096", "op": "norm", "M": 2048, "K": 4096, "dtype": "float16", "int8": True, "pad": 0},
        # the 16-bit output in bf16, a width that no vector divides, rows that are slices of a wider buffer
        {"name": "norm bf16 333x4100", "op": "norm", "M": 333, "K": 4100, "dtype": "bfloat16", "int8": False, "pad": 12},
        # a decode batch of 16 between the gate/up and the down product
        {"name": "swiglu int8 16x11008", "op": "swiglu", "M": 16, "N": 11008, "dtype": "float16"},
        # the same place in a prompt of 2048 tokens
        {"name": "swiglu int8 2048x11008", "op": "swiglu", "M": 2048, "N": 11008, "dtype": "float16"},
        # one token through an attention projection
        {"name": "w8a8 1x4096x4096", "op": "w8a8", "M": 1, "N": 4096, "K": 4096, "bias": False},
        # a decode batch of 16 through an up projection
        {"name": "w8a8 16x14336x4096", "op": "w8a8", "M": 16, "N": 14336, "K": 4096, "bias": False},
        # a ragged prompt and a ragged layer with a bias (a classifier's head, a column shard)
        {"name": "w8a8 333x1001x4112", "op": "w8a8", "M": 333, "N": 1001, "K": 4112, "bias": True},
        # a long prompt through the largest projection of the benchmark's configurations
        {"name": "w8a8 4096x28672x8192", "op": "w8a8", "M": 4096, "N": 28672, "K": 8192, "bias": False},
        # one token, few large experts
        {"name": "moe 1 token 2 of 8", "op": "moe", "T": 1, "H": 4096, "I": 14336, "E": 8, "k": 2, "renorm": True},
        # a decode batch of 16, many small experts
        {"name": "moe 16 tokens 8 of 64", "op": "moe", "T": 16, "H": 2048, "I": 1024, "E": 64, "k": 8, "renorm": True},
        # the largest batch but a few, an odd number of experts, odd widths, probabilities kept as they are
        {"name": "moe 27 tokens 4 of 60", "op": "moe", "T": 27, "H": 2064, "I": 720, "E": 60, "k": 4, "renorm": False},
    ]


def _log(rng, low, high):
    return min(high, int(round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["norm", "swiglu", "w8a8", "w8a8", "moe", "moe"])
    if op == "norm":
        K = _log(rng, 64, 16384)
        K = K if rng.random() < 0.3 else max(64, K // 64 * 64)
        return {"op": op, "M": _log(rng, 1, 4096), "K": K, "dtype": rng.choice(["float16", "bfloat16"]),
                "int8": rng.random() < 0.7, "pad": rng.choice([0, 0, 0, 8, 5])}
    if op == "swiglu":
        N = _log(rng, 64, 28672)
        N = N if rng.random() < 0.3 else max(64, N // 64 * 64)
        return {"op": op, "M": _log(rng, 1, 2048), "N": N, "dtype": rng.choice(["float16", "bfloat16"])}
    if op == "w8a8":
        N, K = _log(rng, 256, 28672), _log(rng, 256, 28672)
        K = K if rng.random() < 0.15 else K // 16 * 16 if rng.random() < 0.4 else K // 128 * 128
        N = N if rng.random() < 0.3 else N // 64 * 64
        most = 4096 * 28672 * 8192 // (N * K)
        return {"op": op, "M": _log(rng, 1, max(1, min(4096, most))), "N": N, "K": K, "bias": rng.random() < 0.5}
    H, I = _log(rng, 256, 4096) // 16 * 16, _log(rng, 128, 14336) // 16 * 16
    E = _log(rng, 4, 128)
    E = max(4, min(E, 8 * 4096 * 14336 // (H * I)))
    k = rng.randint(1, min(E, 8))
    T = _log(rng, 1, 32)
    T = max(1, min(T, 64 * 4096 * 14336 // (k * H * I)))
    return {"op": op, "T": T, "H": H, "I": I, "E": E, "k": k, "renorm": rng.random() < 0.5}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _rows_int8(v):
    """Rows of v as int8 values and one 32-bit scale each."""
    scale = v.abs().amax(-1) / 127
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return torch.round(v / scale.unsqueeze(-1)).clamp(-128, 127).to(torch.int8), scale


def _weight(g, *shape):
    """An int8 weight of N(0, 0.02) values with a scale for each output channel."""
    return _rows_int8(torch.randn(*shape, generator=g, device="cuda").mul_(0.02))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "norm":
        dtype, M, K = getattr(torch, case["dtype"]), case["M"], case["K"]
        wide = torch.randn(M, K + case["pad"], generator=g, device="cuda").to(dtype)
        # a residual stream's channels differ in size, a few by much
        channel = torch.exp(torch.randn(K, generator=g, device="cuda"))
        residual = (torch.randn(M, K, generator=g, device="cuda") * channel).to(dtype)
        weight = torch.rand(K, generator=g, device="cuda") + 0.5
        return dict(case, x=wide[:, :K], residual=residual, weight=weight)
    if op == "swiglu":
        dtype, M, N = getattr(torch, case["dtype"]), case["M"], case["N"]
        gate = (torch.randn(M, N, generator=g, device="cuda") * 1.3).to(dtype)
        return dict(case, gate=gate, up=(torch.randn(M, N, generator=g, device="cuda") * 1.3).to(dtype))
    if op == "w8a8":
        M, N, K = case["M"], case["N"], case["K"]
        q, sx = _rows_int8(torch.randn(M, K, generator=g, device="cuda"))
        w, sw = _weight(g, N, K)
        bias = (torch.randn(N, generator=g, device="cuda") * 0.1).half() if case["bias"] else None
        return dict(case, q=q, sx=sx, w=w, sw=sw, bias=bias)
    T, H, I, E = case["T"], case["H"], case["I"], case["E"]
    s = dict(case, x=torch.randn(T, H, generator=g, device="cuda").half())
    s["router"] = (torch.randn(E, H, generator=g, device="cuda") * (1.5 / H ** 0.5)).half()
    s["gate"], s["s_gate"] = _weight(g, E, I, H)
    s["up"], s["s_up"] = _weight(g, E, I, H)
    s["down"], s["s_down"] = _weight(g, E, H, I)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def _values(q, scale):
    """What int8 rows stand for, in 16 bits."""
    return torch.mul(q, scale.unsqueeze(-1), out=torch.empty(q.shape, dtype=torch.float16, device=q.device))


def _plain_norm(s):
    x, residual = s["x"], s["residual"]
    h = (x.float() + residual.float()).to(x.dtype)
    f = h.float()
    v = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * s["weight"]
    if not s["int8"]:
        return {"y": v.to(x.dtype), "h": h}
    q, scale = _rows_int8(v)
    return {"values": _values(q, scale), "scale": scale, "h": h}


def _plain_swiglu(s):
    gate = s["gate"].float()
    q, scale = _rows_int8(gate / (1 + torch.exp(-gate)) * s["up"].float())
    return {"values": _values(q, scale), "scale": scale}


def _plain_w8a8(s):
    y = (s["q"].float() @ s["w"].float().t()) * s["sx"].unsqueeze(1) * s["sw"]
    return (y if s["bias"] is None else y + s["bias"].float()).half()


def _plain_moe(s):
    T, k = s["T"], s["k"]
    # a choice between two experts is a border: its logits in 64 bits
    logits = s["x"].double() @ s["router"].double().t()
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    chosen, ids = torch.sort(p, dim=-1, descending=True, stable=True)
    chosen, ids = chosen[:, :k], ids[:, :k].reshape(-1)
    if s["renorm"]:
        chosen = chosen / chosen.sum(-1, keepdim=True)
    x = s["x"].float().repeat_interleave(k, 0).unsqueeze(-1)
    gate = (s["gate"][ids].float() @ x).squeeze(-1) * s["s_gate"][ids]
    up = (s["up"][ids].float() @ x).squeeze(-1) * s["s_up"][ids]
    a = gate / (1 + torch.exp(-gate)) * up
    y = (s["down"][ids].float() @ a.unsqueeze(-1)).squeeze(-1) * s["s_down"][ids]
    return (y.view(T, k, -1) * chosen.float().unsqueeze(-1)).sum(1).half()


def _own(s):
    import rotalabs_accel_b200 as ra
    op = s["op"]
    if op == "norm":
        if not s["int8"]:
            y, h = ra.add_rmsnorm(s["x"], s["residual"], s["weight"], EPS)
            return {"y": y, "h": h}
        q, scale, h = ra.add_rmsnorm_int8(s["x"], s["residual"], s["weight"], EPS)
        return {"values": _values(q, scale), "scale": scale, "h": h}
    if op == "swiglu":
        q, scale = ra.swiglu_int8(s["gate"], s["up"])
        return {"values": _values(q, scale), "scale": scale}
    if op == "w8a8":
        return ra.int8_gemm_w8a8(s["q"], s["sx"], s["w"], s["sw"], s["bias"])
    return ra.int8_moe(s["x"], s["router"], s["gate"], s["s_gate"], s["up"], s["s_up"], s["down"], s["s_down"],
                       top_k=s["k"], renormalize=s["renorm"])


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "swiglu": _plain_swiglu, "w8a8": _plain_w8a8, "moe": _plain_moe}[state["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "norm":
        M, K = case["M"], case["K"]
        return {"bytes": M * K * (2 + 2 + 2 + (1 if case["int8"] else 2)) + 4 * K + (4 * M if case["int8"] else 0),
                "flops": 8 * M * K}
    if op == "swiglu":
        M, N = case["M"], case["N"]
        return {"bytes": M * N * 5 + 4 * M, "flops": 8 * M * N}
    if op == "w8a8":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * K + N * K + 4 * M + 4 * N + (2 * N if case["bias"] else 0) + 2 * M * N,
                "flops": 2 * M * N * K}
    T, H, I, E, k = (case[n] for n in ("T", "H", "I", "E", "k"))
    active = E * (1 - (1 - k / E) ** T)  # experts that some token chose, on average
    return {"bytes": 2 * E * H + active * (3 * I * H + 4 * (2 * I + H)) + 4 * T * H,
            "flops": 2 * T * E * H + 6 * T * k * I * H}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def _exact_int8(v):
    top = v.abs().max(dim=-1).values
    step = torch.where(top > 0, top / 127, torch.ones_like(top))
    return (v / step[:, None]).round() * step[:, None], step


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = (s["x"].double() + s["residual"].double()).to(s["x"].dtype)
        d = h.double()
        v = d / (d.pow(2).sum(-1, keepdim=True) / case["K"] + EPS).sqrt() * s["weight"].double()
        if not case["int8"]:
            return {"y": v, "h": h.double()}
        values, step = _exact_int8(v)
        return {"values": values, "scale": step, "h": h.double()}
    if op == "swiglu":
        gate = s["gate"].double()
        values, step = _exact_int8(gate * torch.sigmoid(gate) * s["up"].double())
        return {"values": values, "scale": step}
    if op == "w8a8":
        x = s["q"].double() * s["sx"].double()[:, None]
        w = s["w"].double() * s["sw"].double()[:, None]
        y = torch.einsum("mk,nk->mn", x, w)
        return y if s["bias"] is None else y + s["bias"].double()[None, :]
    y = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
    p = torch.softmax(torch.einsum("th,eh->te", s["x"].double(), s["router"].double()), -1).tolist()
    for t, row in enumerate(p):
        best = sorted(range(case["E"]), key=lambda e: (-row[e], e))[:case["k"]]
        total = sum(row[e] for e in best) if case["renorm"] else 1.0
        x = s["x"][t].double()
        for e in best:
            gate = torch.mv(s["gate"][e].double(), x) * s["s_gate"][e].double()
            up = torch.mv(s["up"][e].double(), x) * s["s_up"][e].double()
            y[t] += row[e] / total * s["s_down"][e].double() * torch.mv(s["down"][e].double(), gate * torch.sigmoid(gate) * up)
    return y
