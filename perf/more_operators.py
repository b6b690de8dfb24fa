"""Sizes, inputs and plain forms of the routing of tokens to experts (with its
gradient), 8-bit floating point quantisation in blocks of 128, and the products
with 8-bit weights, dense and grouped by expert (with the gradient of their
rows).

``run(state)`` is one pass through an operator: with ``own`` false in
elementary torch operations (32 bits, 64 for the values that decide an order,
one rounding at the end), with ``own`` true through the package's entry points.
``exact(case, seed)`` evaluates the operator's definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BLOCK = 128  # elements that share a scale


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding token of the Mixtral-shaped layer chooses two of eight experts: launch latency
        {"name": "route_token", "op": "route", "T": 1, "E": 8, "k": 2, "score": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "group_top": 1, "renorm": True, "scale": 1.0, "dtype": "f32"},
        # the layer bench's batch (16384 tokens, 64 experts, top-6), logits of a bf16 projection
        {"name": "route_prefill", "op": "route", "T": 16384, "E": 64, "k": 6, "score": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "group_top": 1, "renorm": False, "scale": 1.0, "dtype": "bf16"},
        # the most experts, sigmoid scores with a balance bias, four of eight groups, an odd token count
        {"name": "route_groups", "op": "route", "T": 16383, "E": 256, "k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_top": 2, "renorm": True, "scale": 2.5, "dtype": "f32"},
        # training: the gradient that reaches every logit (softmax over all experts)
        {"name": "route_grad", "op": "route_grad", "T": 16384, "E": 64, "k": 6, "score": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "group_top": 1, "renorm": False, "scale": 1.0, "dtype": "bf16"},
        # training with sigmoid scores and renormalised weights, a padded batch
        {"name": "route_grad_groups", "op": "route_grad", "T": 16383, "E": 256, "k": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "group_top": 2, "renorm": True, "scale": 2.5, "dtype": "f32"},
        # the layer bench's dispatched rows are quantised once for all their experts' products
        {"name": "quantize_rows", "op": "quantize", "M": 98304, "K": 2048, "dtype": "bf16"},
        # a dense projection is quantised when a model is loaded
        {"name": "quantize_weight", "op": "quantize_weight", "K": 4096, "N": 14336, "dtype": "f32"},
        # one decoding token through one up projection of the dense GEMM suite's size
        {"name": "fp8_token", "op": "fp8", "M": 1, "K": 4096, "N": 14336, "dtype": "bf16"},
        # a prompt through the same projection: the tensor cores' rate
        {"name": "fp8_prefill", "op": "fp8", "M": 4096, "K": 4096, "N": 14336, "dtype": "bf16"},
        # training: the gradient of an odd number of float32 rows
        {"name": "fp8_grad", "op": "fp8_grad", "M": 2047, "K": 4096, "N": 14336, "dtype": "f32"},
        # a decoding batch over the 64 experts of the layer bench: a few rows for each expert
        {"name": "experts_batch", "op": "experts", "T": 64, "k": 6, "E": 64, "K": 2048, "N": 1408, "dtype": "bf16"},
        # the layer bench's batch through its experts' up projection
        {"name": "experts_prefill", "op": "experts", "T": 16384, "k": 6, "E": 64, "K": 2048, "N": 1408,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "route", "route_grad", "route_grad", "quantize", "quantize_weight", "fp8", "fp8",
                     "fp8_grad", "experts", "experts", "experts_grad"])
    c = {"op": op, "dtype": rng.choice(["bf16", "f32"])}
    if op in ("route", "route_grad"):
        groups, size = rng.choice([(1, 4), (1, 8), (1, 17), (1, 60), (1, 64), (1, 128), (1, 160), (1, 256), (4, 8),
                                   (4, 15), (8, 8), (8, 16), (8, 20), (8, 32), (16, 16)])
        E = groups * size
        top = 1 if groups == 1 else rng.randint(2, groups - 1)
        k = rng.randint(1, min(8, top * size))
        c.update(T=_log(rng, 1, 16383), E=E, k=k, score=rng.choice(["softmax", "sigmoid"]),
                 bias=rng.random() < 0.5, groups=groups, top_groups=top,
                 group_top=1 if groups == 1 else rng.choice([1, 2]), renorm=k > 1 and rng.random() < 0.5,
                 scale=rng.choice([1.0, 2.5]))
    elif op == "quantize":
        K = _log(rng, 64, 14336)
        K = max(64, K // 64 * 64) if rng.random() < 0.75 else K
        c.update(K=K, M=_log(rng, 1, 98304 * 2048 // (K * (1 if c["dtype"] == "bf16" else 2))))
    else:
        K = _log(rng, 64, 14336)
        N = _log(rng, 64, max(64, min(14336, 4096 * 14336 // K)))
        if rng.random() < 0.75:
            K = max(64, K // 64 * 64)
        if rng.random() < 0.75:
            N = max(64, N // 64 * 64)
        if op == "fp8_grad" and rng.random() < 0.5:
            K, N = N, K
        if op in ("fp8", "fp8_grad"):
            c["M"] = _log(rng, 1, 4096)
        elif op != "quantize_weight":
            E = rng.choice([4, 8, 16, 17, 60, 64, 128, 256])
            k = rng.randint(1, min(8, E))
            N = max(64, min(N, 64 * 2048 * 1408 // (E * K)))
            # no more operations than the largest listed case has, no more rows than it moves
            most = min(98304 * 2048 * 1408 // (K * N), 98304 * 2048 // max(K, N))
            c.update(E=E, k=k, T=_log(rng, 1, max(1, min(16384, most // k))))
        c.update(K=K, N=N)
    return c


# ------------------------------------------------------------------ inputs
def _logits(T, E, g, dt):
    """A trained router's logits: experts more and less popular, standard deviation of about 1.5."""
    popular = -0.3 * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    return (1.5 * torch.randn(T, E, device="cuda", generator=g) + popular).to(dt)


def _dispatched(T, k, E, g):
    """Rows [starts[e], starts[e+1]) of each expert, for T tokens with k choices each."""
    ids = torch.topk(_logits(T, E, g, torch.float32), k, dim=1).indices.reshape(-1)
    return torch.searchsorted(torch.sort(ids).values, torch.arange(E + 1, device="cuda")).to(torch.int32)


def _weights(G, K, N, g):
    """G e4m3 weights [K, N] and their scales, as normally distributed ones quantise to."""
    q = torch.randn(G, K, N, device="cuda", generator=g).mul_(448 / 4.2).clamp_(-448, 448).to(torch.float8_e4m3fn)
    s = torch.rand(G, -(-K // BLOCK), -(-N // BLOCK), device="cuda", generator=g) + 0.5
    return q, s * (4.2 / 448 / math.sqrt(K))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op, dt = case["op"], DTYPES[case["dtype"]]
    st = {"case": case}

    def rand(*shape):  # rows of their own sizes, as activations and gradients have
        x = torch.randn(*shape, device="cuda", generator=g)
        return (x * (0.5 + torch.rand(shape[0], 1, device="cuda", generator=g))).to(dt)

    if op in ("route", "route_grad"):
        T, E, k = case["T"], case["E"], case["k"]
        st["logits"] = _logits(T, E, g, dt)
        # the bias evens popular and rare experts out
        st["bias"] = 0.02 * torch.randn(E, device="cuda", generator=g) if case["bias"] else None
        if op == "route_grad":
            st["ids"] = _choice(st, case)[0].to(torch.int32)
            st["grad"] = torch.randn(T, k, device="cuda", generator=g)
        return st
    if op == "quantize":
        st["x"] = rand(case["M"], case["K"])
        return st
    K, N = case["K"], case["N"]
    if op == "quantize_weight":
        st["w"] = rand(K, N) * 0.02
        return st
    G = case.get("E", 1)
    q, s = _weights(G, K, N, g)
    if "E" in case:
        st["starts"] = _dispatched(case["T"], case["k"], G, g)
        st["most"] = int(st["starts"].diff().max())  # rows of the largest expert: the plain form's padding
    rows = case["M"] if "M" in case else case["T"] * case["k"]
    st["x"] = rand(rows, N if op.endswith("grad") else K)
    if own:  # weights are packed once, when they are loaded
        from aethermoe_b200 import fp8
        st["w"] = fp8.Fp8Weight(q, s)
    else:
        st["q"], st["s"] = q, s
    return st


# ------------------------------------------------------------------ one pass
def _choice(st, c):
    """(ids [T, k], score in 64 bits): the experts by score + bias; without a bias by the logits,
    whose order is the scores'."""
    x = st["logits"].double()
    s = torch.softmax(x, 1) if c["score"] == "softmax" else torch.sigmoid(x)
    key = s + st["bias"].double() if st["bias"] is not None else x
    if c["groups"] > 1:
        T, G = x.shape[0], c["groups"]
        by = key if st["bias"] is not None or c["group_top"] == 1 else s
        value = by.reshape(T, G, -1).sort(2, descending=True).values[:, :, :c["group_top"]].sum(2)
        kept = torch.argsort(value, dim=1, descending=True, stable=True)[:, :c["top_groups"]]
        on = torch.zeros(T, G, device="cuda", dtype=torch.bool).scatter(1, kept, True)
        key = torch.where(on.repeat_interleave(x.shape[1] // G, 1), key, -math.inf)
    return torch.argsort(key, dim=1, descending=True, stable=True)[:, :c["k"]], s


def _quantized(x):
    """(e4m3 values, scales) of rows in blocks of 128 along the last dimension."""
    M, K = x.shape
    kb = -(-K // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - K)).reshape(M, kb, BLOCK)
    a = x.abs().amax(2)
    s = torch.clamp(a / torch.full_like(a, 448.0), min=2.0 ** -126)
    return (x / s[:, :, None]).to(torch.float8_e4m3fn).reshape(M, kb * BLOCK)[:, :K], s


def _dequantized(q, s):
    M, K = q.shape
    return q.float() * s.repeat_interleave(BLOCK, 1)[:, :K]


def run(st):
    c = st["case"]
    if own:
        return _own(st, c)
    op = c["op"]
    if op == "route":
        ids, s = _choice(st, c)
        v = s.gather(1, ids).float()
        if c["renorm"]:
            v = v / (v.sum(1, keepdim=True) + 1e-20)
        return {"ids": ids.to(torch.int32), "weights": v * c["scale"]}
    if op == "route_grad":
        x, at, g = st["logits"].float(), st["ids"].long(), st["grad"] * c["scale"]
        s = torch.softmax(x, 1) if c["score"] == "softmax" else torch.sigmoid(x)
        v = s.gather(1, at)
        if c["renorm"]:  # of the chosen scores
            total = v.sum(1, keepdim=True) + 1e-20
            g = (g - (g * v / total).sum(1, keepdim=True)) / total
        gs = torch.zeros_like(s).scatter(1, at, g)
        gx = s * (gs - (gs * s).sum(1, keepdim=True)) if c["score"] == "softmax" else gs * s * torch.sigmoid(-x)
        return gx.to(st["logits"].dtype)
    if op == "quantize":
        q, s = _quantized(st["x"])
        return {"q": q, "scale": s}
    if op == "quantize_weight":
        K, N = c["K"], c["N"]
        kb, nb = -(-K // BLOCK), -(-N // BLOCK)
        w = torch.nn.functional.pad(st["w"].float(), (0, nb * BLOCK - N, 0, kb * BLOCK - K))
        a = w.abs().reshape(kb, BLOCK, nb, BLOCK).amax((1, 3))
        s = torch.clamp(a / torch.full_like(a, 448.0), min=2.0 ** -126)
        q = (w.reshape(kb, BLOCK, nb, BLOCK) / s[:, None, :, None]).to(torch.float8_e4m3fn)
        return {"q": q.reshape(kb * BLOCK, nb * BLOCK)[:K, :N], "scale": s}
    x = _dequantized(*_quantized(st["x"]))
    w = st["q"].float()
    w *= st["s"].repeat_interleave(BLOCK, 1)[:, :c["K"]].repeat_interleave(BLOCK, 2)[:, :, :c["N"]]
    if op.endswith("grad"):
        w = w.transpose(1, 2)
    if "E" not in c:
        return (x @ w[0]).to(st["x"].dtype)
    # every expert's rows, padded to the largest expert's number
    starts = st["starts"].long()
    at = starts[:-1, None] + torch.arange(st["most"], device="cuda")
    xe = torch.where((at < starts[1:, None])[:, :, None], x[at.clamp(max=x.shape[0] - 1)], 0.0)
    y = torch.bmm(xe, w)
    row = torch.arange(x.shape[0], device="cuda")
    of = torch.searchsorted(starts, row, right=True) - 1
    y = y[of, row - starts[of]]
    return (torch.relu(y) if op == "experts" else y).to(st["x"].dtype)


def _own(st, c):
    op = c["op"]
    from aethermoe_b200 import fp8, routing
    if op in ("route", "route_grad"):
        how = dict(score=c["score"], renormalize=c["renorm"], scale=c["scale"])
        if op == "route_grad":
            return routing.route_tokens_backward(st["grad"], st["logits"], st["ids"], **how)
        ids, weights = routing.route_tokens(st["logits"], c["k"], bias=st["bias"], groups=c["groups"],
                                            top_groups=c["top_groups"], group_top=c["group_top"], **how)
        return {"ids": ids, "weights": weights}
    if op == "quantize":
        rows = fp8.quantize_fp8(st["x"])
        return {"q": rows.q, "scale": rows.scale}
    if op == "quantize_weight":
        q, s = fp8.quantize_fp8_weight(st["w"])
        return {"q": q, "scale": s}
    if op == "fp8":
        return fp8.fp8_matmul(st["x"], st["w"])
    if op == "fp8_grad":
        return fp8.fp8_matmul_backward(st["x"], st["w"])
    if op == "experts":
        return fp8.grouped_fp8_matmul(st["x"], st["w"], st["starts"], relu=True)
    return fp8.grouped_fp8_matmul_backward(st["x"], st["w"], st["starts"])


# ------------------------------------------------------------------ work and definition
def work(case):
    """Bytes that have to cross memory once, and the products' operations."""
    op, es = case["op"], 2 if case["dtype"] == "bf16" else 4
    if op in ("route", "route_grad"):
        T, E, k = case["T"], case["E"], case["k"]
        if op == "route":
            return {"bytes": T * E * es + 8 * T * k, "flops": 4 * T * E}
        read = T * E if case["score"] == "softmax" and not case["renorm"] else T * k
        return {"bytes": (read + T * E) * es + 8 * T * k, "flops": 4 * read}
    K = case["K"]
    if op == "quantize":
        M = case["M"]
        return {"bytes": M * K * (es + 1) + 4 * M * -(-K // BLOCK), "flops": 2 * M * K}
    N = case["N"]
    scales = 4 * -(-K // BLOCK) * -(-N // BLOCK)
    if op == "quantize_weight":
        return {"bytes": K * N * (es + 1) + scales, "flops": 2 * K * N}
    M = case["M"] if "M" in case else case["T"] * case["k"]
    reached = 1.0
    if "E" in case:  # experts that a batch reaches, on average, popular ones more often
        pop = [(e + 1) ** -0.3 for e in range(case["E"])]
        reached = sum(1 - (1 - min(1.0, case["k"] * p / sum(pop))) ** case["T"] for p in pop)
        reached = max(reached, case["k"])
    return {"bytes": reached * (K * N + scales) + M * (K + N) * es, "flops": 2 * M * K * N}


def exact(case, seed):
    global own
    kept, own = own, False  # the inputs as tensors, whatever run() is about to use
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    if op in ("route", "route_grad"):
        x = st["logits"].double()
        if case["score"] == "softmax":
            e = torch.exp(x - x.amax(1, keepdim=True))
            s = e / e.sum(1, keepdim=True)
        else:
            s = 1 / (1 + torch.exp(-x))
        if op == "route":
            k, G, b = case["k"], case["groups"], st["bias"]
            by = s if b is None else s + b.double()
            left = by.clone()
            if G > 1:  # the groups' values, one largest expert after the other
                part, value = by.reshape(x.shape[0], G, -1).clone(), 0.0
                for _ in range(case["group_top"]):
                    top = part.max(2)
                    value = value + top.values
                    part.scatter_(2, top.indices[:, :, None], -math.inf)
                dropped = torch.ones_like(value, dtype=torch.bool)
                for _ in range(case["top_groups"]):
                    first = value.argmax(1, keepdim=True)
                    dropped.scatter_(1, first, False)
                    value = value.scatter(1, first, -math.inf)
                left[dropped.repeat_interleave(x.shape[1] // G, 1)] = -math.inf
            v = []
            for _ in range(k):
                top = left.max(1, keepdim=True)
                v.append(s.gather(1, top.indices))
                left.scatter_(1, top.indices, -math.inf)
            v = torch.cat(v, 1)
            if case["renorm"]:
                v = v / (v.sum(1, keepdim=True) + 1e-20)
            return {"ids": None, "weights": v * case["scale"]}
        # dw_j / dx_e, summed over the slots
        at, g = st["ids"].long(), st["grad"].double() * case["scale"]
        v = s.gather(1, at)
        if case["renorm"]:
            total = v.sum(1, keepdim=True) + 1e-20
            g = g / total - (g * v).sum(1, keepdim=True) / total ** 2
        out = torch.zeros_like(s)
        if case["score"] == "softmax":
            out -= s * (g * v).sum(1, keepdim=True)
            return out.scatter_add_(1, at, g * v)
        return out.scatter_add_(1, at, g * v / (1 + torch.exp(x.gather(1, at))))
    if op == "quantize":
        s = [st["x"][:, a:a + BLOCK].double().abs().amax(1) for a in range(0, case["K"], BLOCK)]
        return {"q": None, "scale": torch.stack(s, 1) / 448}
    K, N = case["K"], case["N"]
    if op == "quantize_weight":
        s = [torch.stack([st["w"][a:a + BLOCK, b:b + BLOCK].double().abs().amax() for b in range(0, N, BLOCK)])
             for a in range(0, K, BLOCK)]
        return {"q": None, "scale": torch.stack(s) / 448}
    # quantisation is part of the definition: a float32 scale, e4m3 values of the float32 quotient
    x, grad = st["x"], op.endswith("grad")
    R, C = x.shape
    vals = torch.empty(R, C, device="cuda", dtype=torch.float64)
    for a in range(0, C, BLOCK):
        part = x[:, a:a + BLOCK].float()
        sc = (part.abs().amax(1, keepdim=True) / torch.tensor(448.0, device="cuda")).clamp(min=2.0 ** -126)
        vals[:, a:a + BLOCK] = (part / sc).to(torch.float8_e4m3fn).double() * sc.double()
    bounds = st["starts"].tolist() if "E" in case else [0, R]
    out = torch.zeros(R, K if grad else N, device="cuda", dtype=torch.float64)
    for e in range(len(bounds) - 1):
        if bounds[e] == bounds[e + 1]:
            continue
        w = st["q"][e].double()
        for i, a in enumerate(range(0, K, BLOCK)):
            w[a:a + BLOCK] *= st["s"][e, i].double().repeat_interleave(BLOCK)[:N]
        out[bounds[e]:bounds[e + 1]] = vals[bounds[e]:bounds[e + 1]] @ (w.t() if grad else w)
    return out.clamp(min=0) if op == "experts" else out
