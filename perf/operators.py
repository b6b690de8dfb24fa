"""Sizes, inputs and plain forms of the expert operators: token dispatch and
combine (with their gradients), 4-bit group quantisation, and the products
with 4-bit weights, dense and grouped by expert.

``run(state)`` is one pass through an operator: with ``own`` false in
elementary torch operations (32 bits, one rounding at the end), with ``own``
true through the package's entry points.  ``exact(case, seed)`` evaluates the
operator's definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding token of the Mixtral-shaped layer goes to its two experts: launch latency
        {"name": "dispatch_token", "op": "dispatch", "T": 1, "k": 2, "E": 8, "d": 4096,
         "dtype": "bf16", "padded": 0.0},
        # the layer bench's batch (16384 tokens, 64 experts, top-6): the largest copy
        {"name": "dispatch_prefill", "op": "dispatch", "T": 16384, "k": 6, "E": 64, "d": 2048,
         "dtype": "bf16", "padded": 0.0},
        # training step of a padded float32 batch: gradient of the dispatch, an odd token count
        {"name": "dispatch_grad", "op": "dispatch_grad", "T": 4095, "k": 6, "E": 64, "d": 2048,
         "dtype": "f32", "padded": 0.1},
        # the same batch's way back: k expert rows of a token weighted and summed
        {"name": "combine_prefill", "op": "combine", "T": 16384, "k": 6, "E": 64, "d": 2048,
         "dtype": "bf16", "padded": 0.0},
        # training: gradients of the expert rows and of the gate weights, a padded batch
        {"name": "combine_grad", "op": "combine_grad", "T": 8191, "k": 6, "E": 64, "d": 2048,
         "dtype": "bf16", "padded": 0.05},
        # one decoding token through one up projection of the dense GEMM suite's size
        {"name": "q4_token", "op": "q4", "M": 1, "K": 4096, "N": 14336, "gs": 128,
         "dtype": "bf16", "scale": "bf16"},
        # eight float32 rows, the activation type of the host-array interface, finest groups
        {"name": "q4_rows_f32", "op": "q4", "M": 8, "K": 4096, "N": 14336, "gs": 32,
         "dtype": "f32", "scale": "f32"},
        # the largest decoding batch, through a down projection
        {"name": "q4_batch", "op": "q4", "M": 64, "K": 14336, "N": 4096, "gs": 64,
         "dtype": "bf16", "scale": "bf16"},
        # one decoding token of the Mixtral-shaped layer: two of eight experts are read
        {"name": "experts_token", "op": "experts", "T": 1, "k": 2, "E": 8, "K": 4096, "N": 14336,
         "gs": 128, "dtype": "bf16", "scale": "bf16"},
        # a decoding batch over the 64 experts of the layer bench: a few rows for each expert
        {"name": "experts_batch", "op": "experts", "T": 64, "k": 6, "E": 64, "K": 2048, "N": 1408,
         "gs": 32, "dtype": "bf16", "scale": "f32"},
        # one expert's projection of the layer bench is quantised: a small matrix
        {"name": "quantize_expert", "op": "quantize", "K": 2048, "N": 1408, "gs": 32,
         "dtype": "f32", "scale": "f32"},
        # a whole dense projection is quantised when a model is loaded
        {"name": "quantize_dense", "op": "quantize", "K": 14336, "N": 4096, "gs": 128,
         "dtype": "f32", "scale": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["dispatch", "dispatch_grad", "combine", "combine_grad", "q4", "q4", "experts",
                     "experts", "quantize"])
    c = {"op": op, "dtype": rng.choice(["bf16", "f32"])}
    if op in ("dispatch", "dispatch_grad", "combine", "combine_grad"):
        E = rng.choice([4, 8, 16, 17, 60, 64, 128, 256])
        k = rng.randint(1, min(8, E))
        d = _log(rng, 64, 8192)
        if rng.random() < 0.75:
            d = max(8, d // 8 * 8)
        # at most the bytes of the largest listed case, less for the gradient that moves more
        most = 16384 * 6 * 2048 // (2 if c["dtype"] == "f32" else 1) // (2 if op == "combine_grad" else 1)
        T = _log(rng, 1, max(1, min(32768, most // (k * d))))
        c.update(T=T, k=k, E=E, d=d, padded=rng.choice([0.0, 0.0, 0.03, 0.3]))
    else:
        c["gs"] = rng.choice([32, 64, 128])
        c["scale"] = rng.choice(["bf16", "f32"])
        K = _log(rng, 64, 14336)
        if rng.random() < 0.75:
            K = max(64, K // 64 * 64)
        N = _log(rng, 16, max(16, min(14336, 4096 * 14336 // K)))
        if rng.random() < 0.5:
            N = max(16, N // 16 * 16)
        c.update(K=K, N=N)
        if op == "q4":
            c["M"] = _log(rng, 1, 64 if c["dtype"] == "bf16" else 21)
        elif op == "experts":
            E = rng.choice([4, 8, 16, 17, 60, 64, 128, 256])
            c["E"] = E
            c["k"] = rng.randint(1, min(8, E))
            c["T"] = _log(rng, 1, 64)
            c["N"] = max(16, min(N, 64 * 2048 * 1408 // (E * K)))
    return c


# ------------------------------------------------------------------ inputs
def _routing(T, k, E, padded, g):
    """Gating's answer for T tokens: ids [T, k (+1)] int32 with popular and rare
    experts, softmax weights [T, k], and -1 ids for the padded tokens."""
    popular = -1.1 * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    logits = torch.randn(T, E, device="cuda", generator=g) + popular
    val, idx = torch.topk(logits, min(k + 1, E), dim=1)
    idx = idx.to(torch.int32)
    if padded:
        idx[T - int(T * padded):] = -1
    return idx[:, :k], torch.softmax(val[:, :k], dim=1)


def _sorted(ids, E):
    """Stable order of the (token, slot) units by expert, units without one last."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    ranked, order = torch.sort(key, stable=True)
    starts = torch.searchsorted(ranked, torch.arange(E + 1, device=ids.device))
    place = torch.arange(flat.numel(), device=ids.device)
    rank = torch.empty_like(order)
    rank[order] = place
    row_of = torch.where(key < E, rank, -1).reshape(ids.shape)
    unit_of = torch.where(place < starts[E], order, -1)
    return starts.to(torch.int32), row_of.to(torch.int32), unit_of.to(torch.int32)


def _weights(E, K, N, gs, scale, g):
    """E groups of 4-bit weights with the scales of normally distributed ones."""
    q = torch.randint(-7, 8, (E, K, N), device="cuda", dtype=torch.int8, generator=g)
    s = torch.rand(E, -(-K // gs), N, device="cuda", generator=g) + 0.5
    return q, (s * (0.6 / math.sqrt(K))).to(DTYPES[scale])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op, dt = case["op"], DTYPES[case["dtype"]]
    st = {"op": op, "case": case}

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(dt)

    if op in ("dispatch", "dispatch_grad", "combine", "combine_grad"):
        T, k, E, d = (case[n] for n in "TkEd")
        ids, st["weights"] = _routing(T, k, E, case["padded"], g)
        st["ids"] = ids
        if op == "dispatch":
            st["x"] = rand(T, d)
            return st
        st["starts"], st["row_of"], st["unit_of"] = _sorted(ids, E)
        st["rows"] = rand(T * k, d)  # expert rows, or their gradient
        if op == "combine_grad":
            st["grad_out"] = rand(T, d)
        if own:  # the order that the dispatch of the same step returned
            from aethermoe_b200 import dispatch as D
            st["order"] = D.TokenOrder(st["starts"], st["row_of"], st["unit_of"])
        return st
    K, N, gs = case["K"], case["N"], case["gs"]
    if op == "quantize":
        st["w"] = rand(K, N) * 0.02
        return st
    E = case.get("E", 1)
    q, s = _weights(E, K, N, gs, case["scale"], g)
    if op == "q4":
        st["x"] = rand(case["M"], K)
    else:
        ids, _ = _routing(case["T"], case["k"], E, 0.0, g)
        st["starts"] = _sorted(ids, E)[0]
        st["x"] = rand(case["T"] * case["k"], K)
    if own:  # weights are packed once, when they are loaded
        from aethermoe_b200 import q4
        st["w"] = q4.Q4Weight(q, s, gs)
    else:
        st["q"], st["s"] = q, s
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    c = st["case"]
    if own:
        return _own(st, c)
    op = st["op"]
    if op == "dispatch":
        starts, row_of, unit_of = _sorted(st["ids"], c["E"])
        rows = st["x"][unit_of.clamp(min=0).long() // c["k"]]
        rows = torch.where((unit_of >= 0)[:, None], rows, torch.zeros((), dtype=rows.dtype, device="cuda"))
        return {"rows": rows, "starts": starts, "row_of": row_of}
    if op in ("dispatch_grad", "combine"):
        at = st["row_of"].long()
        r = st["rows"][at.clamp(min=0)].float()
        if op == "combine":
            r = r * st["weights"][:, :, None]
        r = torch.where((at >= 0)[:, :, None], r, 0.0)
        return r.sum(1).to(st["rows"].dtype)
    if op == "combine_grad":
        at, unit = st["row_of"].long(), st["unit_of"].long()
        go = st["grad_out"].float()
        gw = (st["rows"][at.clamp(min=0)].float() * go[:, None, :]).sum(2)
        gw = torch.where(at >= 0, gw, 0.0)
        u = unit.clamp(min=0)
        gr = st["weights"].reshape(-1)[u][:, None] * go[u // c["k"]]
        gr = torch.where((unit >= 0)[:, None], gr, 0.0)
        return {"grad_rows": gr.to(st["rows"].dtype), "grad_weights": gw}
    if op == "quantize":
        K, N, gs = c["K"], c["N"], c["gs"]
        w = st["w"].float()
        kg = -(-K // gs)
        a = torch.nn.functional.pad(w.abs(), (0, 0, 0, kg * gs - K)).reshape(kg, gs, N).amax(1)
        s = torch.clamp(a / torch.full_like(a, 7.0), min=1e-12).to(DTYPES[c["scale"]])
        full = s.float().repeat_interleave(gs, 0)[:K]
        return {"q": torch.clamp(torch.round(w / full), -7, 7).to(torch.int8), "scale": s}
    w = st["q"].float() * st["s"].float().repeat_interleave(c["gs"], 1)[:, :c["K"]]
    x = st["x"].float()
    if op == "q4":
        return (x @ w[0]).to(st["x"].dtype)
    row = torch.arange(x.shape[0], device="cuda")
    of = torch.searchsorted(st["starts"].long(), row, right=True) - 1
    mine = of[None, :] == torch.arange(c["E"], device="cuda")[:, None]
    xe = torch.where(mine[:, :, None], x[None], 0.0)  # [E, rows, K], other experts' rows zero
    return torch.relu(torch.bmm(xe, w).sum(0)).to(st["x"].dtype)


def _own(st, c):
    op = st["op"]
    from aethermoe_b200 import dispatch as D
    from aethermoe_b200 import q4
    if op == "dispatch":
        rows, order = D.dispatch(st["x"], st["ids"], c["E"])
        return {"rows": rows, "starts": order.starts, "row_of": order.row_of}
    if op == "dispatch_grad":
        return D.dispatch_backward(st["rows"], st["order"])
    if op == "combine":
        return D.combine(st["rows"], st["weights"], st["order"])
    if op == "combine_grad":
        gr, gw = D.combine_backward(st["grad_out"], st["rows"], st["weights"], st["order"])
        return {"grad_rows": gr, "grad_weights": gw}
    if op == "quantize":
        q, s = q4.quantize_q4(st["w"], c["gs"], scale_dtype=DTYPES[c["scale"]])
        return {"q": q, "scale": s}
    if op == "q4":
        return q4.q4_matmul(st["x"], st["w"], out_dtype=st["x"].dtype)
    return q4.grouped_q4_matmul(st["x"], st["w"], st["starts"], relu=True, out_dtype=st["x"].dtype)


# ------------------------------------------------------------------ work and definition
def work(case):
    """Bytes that have to cross memory once, and the products' operations."""
    op, es = case["op"], 2 if case["dtype"] == "bf16" else 4
    if op in ("dispatch", "dispatch_grad", "combine", "combine_grad"):
        T, k, E, d = (case[n] for n in "TkEd")
        U = (T - int(T * case["padded"])) * k
        b = {"dispatch": (T + T * k) * d * es + 4 * T * k * 2 + 4 * (E + 1),
             "dispatch_grad": (U + T) * d * es + 4 * T * k,
             "combine": (U + T) * d * es + 8 * T * k,
             "combine_grad": (T + U + T * k) * d * es + 12 * T * k}[op]
        f = {"dispatch": 0, "dispatch_grad": 1, "combine": 2, "combine_grad": 3}[op] * U * d
        return {"bytes": b, "flops": f}
    K, N, gs = case["K"], case["N"], case["gs"]
    ss = 2 if case["scale"] == "bf16" else 4
    kg = -(-K // gs)
    if op == "quantize":
        return {"bytes": K * N * (es + 1) + kg * N * ss, "flops": 2 * K * N}
    M = case["M"] if op == "q4" else case["T"] * case["k"]
    reached = 1.0
    if op == "experts":  # experts that a batch reaches, on average, popular ones more often
        pop = [(e + 1) ** -1.1 for e in range(case["E"])]
        reached = sum(1 - (1 - min(1.0, case["k"] * p / sum(pop))) ** case["T"] for p in pop)
        reached = max(reached, case["k"])
    return {"bytes": reached * (K * N / 2 + kg * N * ss) + M * (K + N) * es, "flops": 2 * M * K * N}


def exact(case, seed):
    st = None
    global own
    kept, own = own, False  # the inputs as tensors, whatever run() is about to use
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    if op in ("dispatch", "dispatch_grad", "combine", "combine_grad"):
        T, k, E, d = (case[n] for n in "TkEd")
        ids = st["ids"]
        # experts in turn: the units that name expert e, in the order of the tokens
        units = torch.cat([torch.nonzero(ids.reshape(-1) == e)[:, 0] for e in range(E)])
        tok, n = units // k, units.numel()
        if op == "dispatch":
            rows = torch.zeros(T * k, d, device="cuda", dtype=torch.float64)
            rows[:n] = st["x"].double()[tok]
            return {"rows": rows, "starts": None, "row_of": None}
        w = st["weights"].double().reshape(-1)[units]
        if op == "combine_grad":
            go = st["grad_out"].double()[tok]
            gr = torch.zeros(T * k, d, device="cuda", dtype=torch.float64)
            gr[:n] = go * w[:, None]
            gw = torch.zeros(T * k, device="cuda", dtype=torch.float64)
            gw[units] = torch.einsum("rd,rd->r", go, st["rows"][:n].double())
            return {"grad_rows": gr, "grad_weights": gw.reshape(T, k)}
        r = st["rows"][:n].double()
        if op == "combine":
            r = r * w[:, None]
        return torch.zeros(T, d, device="cuda", dtype=torch.float64).index_add_(0, tok, r)
    K, gs = case["K"], case["gs"]
    if op == "quantize":
        s = torch.stack([st["w"][a:a + gs].double().abs().amax(0) for a in range(0, K, gs)]) / 7
        return {"q": None, "scale": s}
    x, out = st["x"].double(), []
    bounds = [0, case["M"]] if op == "q4" else st["starts"].tolist()
    for e in range(len(bounds) - 1):
        xe = x[bounds[e]:bounds[e + 1]]
        y = torch.zeros(xe.shape[0], case["N"], device="cuda", dtype=torch.float64)
        if xe.shape[0]:
            for i, a in enumerate(range(0, K, gs)):  # one group of K after the other
                y += (xe[:, a:a + gs] @ st["q"][e, a:a + gs].double()) * st["s"][e, i].double()
        out.append(y if op == "q4" else y.clamp(min=0))
    return torch.cat(out)
