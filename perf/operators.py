"""Workloads of the FP8 block-scaled products, their row quantiser and the router's balance loss.

Sizes are those of the framework's own configurations (hidden 7168, intermediate 2048, gate and up
fused to 4096 columns, 256 experts with 8 per token, 8192^3, N = 4096 / K = 8192) and generic odd
ones. `own = False` computes each operator from elementary torch operations in FP32; `own = True`
makes the calls a user of the package makes.
"""
import math

import numpy as np
import torch

own = False

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -60
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # one token through a fused gate/up projection kept in FP8
        {"name": "gemm one token", "op": "gemm", "m": 1, "n": 4096, "k": 7168, "out": "bf16"},
        # a small ragged batch, last tiles ragged in every dimension
        {"name": "gemm ragged 77", "op": "gemm", "m": 77, "n": 1000, "k": 1040, "out": "fp16"},
        # a batch of decoding requests
        {"name": "gemm batch 128", "op": "gemm", "m": 128, "n": 4096, "k": 8192, "out": "fp16"},
        # prompt processing, the square problem of the GEMM benchmark
        {"name": "gemm 8192 cubed", "op": "gemm", "m": 8192, "n": 8192, "k": 8192, "out": "bf16"},
        # a few rows over small experts, some of them empty
        {"name": "grouped small odd", "op": "grouped", "groups": 8, "rows": 130, "n": 520, "k": 656, "skew": 0.5,
         "out": "fp16"},
        # decoding: 64 tokens x 8 experts on one of eight ranks' 32 experts
        {"name": "grouped decode", "op": "grouped", "groups": 32, "rows": 64, "n": 4096, "k": 7168, "skew": 4.0,
         "out": "fp16"},
        # prompt processing: 4096 tokens x 8 slots, 32 local experts
        {"name": "grouped prefill", "op": "grouped", "groups": 32, "rows": 32768, "n": 4096, "k": 7168, "skew": 8.0,
         "out": "bf16"},
        # activations of a decoding batch in front of a product
        {"name": "quantize decode", "op": "quantize", "rows": 16, "k": 7168, "dtype": "bf16", "swiglu": False},
        # between the two expert products: SiLU(gate) * up of all routed rows
        {"name": "quantize swiglu", "op": "quantize", "rows": 32768, "k": 2048, "dtype": "fp16", "swiglu": True},
        # one micro-batch of a small router, loss and gradient
        {"name": "router step small", "op": "router_step", "tokens": 120, "experts": 64, "topk": 6, "sequences": 3,
         "dtype": "fp32"},
        # balance loss and counts of a training batch, 32 packed sequences
        {"name": "router loss", "op": "router_loss", "tokens": 65536, "experts": 256, "topk": 8, "sequences": 32,
         "dtype": "fp32"},
        # gradient through the weights and the loss, half-precision logits of an odd number of experts
        {"name": "router gradient", "op": "router_grad", "tokens": 131072, "experts": 160, "topk": 6, "sequences": 24,
         "dtype": "bf16"},
    ]


def _log_int(rng, low, high, step=1):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, v // step * step if v >= step else step))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "grouped", "grouped", "quantize", "router_step", "router_loss", "router_grad"])
    if op == "gemm":
        return {"op": op, "m": _log_int(rng, 1, 8192), "n": _log_int(rng, 64, 8192, 8), "k": _log_int(rng, 64, 8192, 16),
                "out": rng.choice(["fp16", "bf16", "fp32"])}
    if op == "grouped":
        c = {"op": op, "groups": _log_int(rng, 1, 128), "rows": _log_int(rng, 1, 32768), "n": _log_int(rng, 64, 7168, 8),
             "k": _log_int(rng, 64, 7168, 16), "skew": rng.choice([0.5, 4.0, 8.0]),
             "out": rng.choice(["fp16", "bf16", "fp32"])}
        while c["groups"] * c["n"] * c["k"] > 32 * 4096 * 7168 or c["rows"] * c["n"] * c["k"] > 32768 * 4096 * 7168:
            c["n"] = max(64, c["n"] // 16 * 8)
        return c
    if op == "quantize":
        swiglu = rng.random() < 0.5
        return {"op": op, "rows": _log_int(rng, 1, 32768), "k": _log_int(rng, 64, 2048 if swiglu else 4096, 16),
                "dtype": rng.choice(["fp16", "bf16"] + ([] if swiglu else ["fp32"])), "swiglu": swiglu}
    e = _log_int(rng, 8, 512)
    tokens = _log_int(rng, 1, 65536 if op == "router_loss" else 131072)
    return {"op": op, "tokens": min(tokens, (16 << 20) // e), "experts": e,
            "topk": rng.randint(1, min(16, e)), "sequences": _log_int(rng, 1, 64), "dtype": rng.choice(["fp32", "bf16", "fp16"])}


# ------------------------------------------------------------------------------------ inputs


def _blocks(k):
    return (k + 127) // 128


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, rows, k):
    """Rows of different magnitude with a few large channels, as hidden states have."""
    x = torch.randn((rows, k), device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn((rows, 1), device="cuda", generator=g))
    return x * torch.where(torch.rand((1, k), device="cuda", generator=g) < 0.01, 20.0, 1.0)


def _quantize_rows(x):
    rows, k = x.shape
    pad = torch.zeros((rows, _blocks(k) * 128), device=x.device)
    pad[:, :k] = x
    blocks = pad.view(rows, -1, 128)
    scale = blocks.abs().amax(-1).clamp(min=AMAX_FLOOR) / E4M3_MAX
    q = (blocks / scale.unsqueeze(-1)).view(rows, -1)[:, :k]
    return q.to(E4M3).contiguous(), scale


def _fp8_weight(g, n, k):
    """A weight matrix as an FP8 checkpoint holds it: e4m3 codes, one FP32 scale per 128 x 128 block."""
    nb, kb = _blocks(n), _blocks(k)
    w = torch.zeros((nb * 128, kb * 128), device="cuda")
    w[:n, :k] = 0.02 * torch.randn((n, k), device="cuda", generator=g)
    blocks = w.view(nb, 128, kb, 128)
    scale = blocks.abs().amax((1, 3)).clamp(min=AMAX_FLOOR) / E4M3_MAX
    q = (blocks / scale.view(nb, 1, kb, 1)).view(nb * 128, kb * 128)[:n, :k]
    return q.to(E4M3).contiguous(), scale


def _row_counts(seed, case):
    """Rows per expert: multinomial over Dirichlet proportions (a small `skew` leaves experts empty)."""
    rng = np.random.default_rng(seed)
    return rng.multinomial(case["rows"], rng.dirichlet(np.full(case["groups"], case["skew"]))).astype(np.int32)


def _sequence_starts(seed, tokens, sequences):
    """Packed sequences of ragged lengths, some of them empty; the last tokens are padding of the batch."""
    rng = np.random.default_rng(seed)
    end = tokens - (tokens // 50 if tokens >= 50 else 0)
    inner = np.sort(rng.integers(0, end + 1, sequences - 1))
    return np.concatenate([[0], inner, [end]]).astype(np.int32)


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    if case["op"] == "gemm":
        state["a"], state["a_scale"] = _quantize_rows(_activations(g, case["m"], case["k"]))
        state["b"], state["b_scale"] = _fp8_weight(g, case["n"], case["k"])
    elif case["op"] == "grouped":
        counts = _row_counts(seed, case)
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        state["x"], state["x_scale"] = _quantize_rows(_activations(g, case["rows"], case["k"]))
        n, k, groups = case["n"], case["k"], case["groups"]
        state["w"] = torch.empty((groups, n, k), device="cuda", dtype=E4M3)
        state["w_scale"] = torch.empty((groups, _blocks(n), _blocks(k)), device="cuda")
        for e in range(groups):
            state["w"][e], state["w_scale"][e] = _fp8_weight(g, n, k)
        state["starts"] = starts.tolist()
        state["seqlens"] = torch.from_numpy(counts).cuda()
        state["cu_seqlens"] = torch.from_numpy(starts).cuda()
    elif case["op"] == "quantize":
        state["x"] = _activations(g, case["rows"], case["k"] * (2 if case["swiglu"] else 1)).to(TYPES[case["dtype"]])
    else:
        t, e, k = case["tokens"], case["experts"], case["topk"]
        logits = torch.randn((t, e), device="cuda", generator=g) + 0.5 * torch.randn((1, e), device="cuda", generator=g)
        state["logits"] = logits.to(TYPES[case["dtype"]])
        ids = state["logits"].float().topk(k, dim=1).indices
        scores = torch.sigmoid(torch.gather(state["logits"].float(), 1, ids))
        state["weights"] = scores / scores.sum(1, keepdim=True)
        # every 64th token is masked: it goes to no expert
        state["ids"] = torch.where((torch.arange(t, device="cuda") % 64 == 63).unsqueeze(1), -1, ids).to(torch.int32)
        state["weights"] = torch.where(state["ids"] < 0, 0.0, state["weights"])
        state["cu_seqlens"] = torch.from_numpy(_sequence_starts(seed, t, case["sequences"])).cuda()
        state["grad_weights"] = torch.randn((t, k), device="cuda", generator=g)
        state["grad_loss"] = 0.5 + torch.rand((), device="cuda", generator=g)
        state["alpha"] = 0.001
        if case["op"] == "router_grad":
            # what the forward pass of the same step left behind
            state["slope"] = _plain_router_loss(state)[2]
    return state


# ------------------------------------------------------------------------------- plain forms


def _expand_rows(scale, k):
    return scale.repeat_interleave(128, dim=1)[:, :k]


def _plain_product(a, a_scale, b, b_scale):
    n, k = b.shape
    wide = b_scale.repeat_interleave(128, dim=0)[:n].repeat_interleave(128, dim=1)[:, :k]
    return (a.float() * _expand_rows(a_scale, k)) @ (b.float() * wide).t()


def _plain_grouped(state, out_type):
    starts = state["starts"]
    out = torch.empty((state["x"].shape[0], state["w"].shape[1]), device="cuda", dtype=out_type)
    for e in range(len(starts) - 1):
        lo, hi = starts[e], starts[e + 1]
        if hi > lo:
            out[lo:hi] = _plain_product(state["x"][lo:hi], state["x_scale"][lo:hi], state["w"][e],
                                        state["w_scale"][e]).to(out_type)
    return out


def _plain_quantize(x, swiglu):
    x = x.float()
    if swiglu:
        gate, up = x.chunk(2, dim=1)
        x = gate / (1.0 + torch.exp(-gate)) * up
    return _quantize_rows(x)


def _sequence_of_token(state):
    """Index of each token's sequence and whether the token counts: inside a sequence, with an expert."""
    cu, ids = state["cu_seqlens"], state["ids"]
    token = torch.arange(ids.shape[0], device="cuda", dtype=torch.int32)
    live = (token >= cu[0]) & (token < cu[-1]) & (ids >= 0).any(1)
    seq = torch.searchsorted(cu[1:].contiguous(), token, right=True).clamp(max=cu.shape[0] - 2)
    return seq, live


def _probabilities(logits):
    score = 1.0 / (1.0 + torch.exp(-logits.float()))
    return score, score / score.sum(1, keepdim=True)


def _plain_router_loss(state):
    logits, ids = state["logits"], state["ids"]
    e, k, sequences = logits.shape[1], ids.shape[1], state["cu_seqlens"].shape[0] - 1
    seq, live = _sequence_of_token(state)
    p = torch.where(live.unsqueeze(1), _probabilities(logits)[1], 0.0)
    total = torch.zeros((sequences, e), device="cuda", dtype=torch.float64).index_add_(0, seq, p.double())
    slot = (seq.unsqueeze(1) * e + ids.clamp(min=0)).reshape(-1)
    valid = ((ids >= 0) & live.unsqueeze(1)).reshape(-1)
    counts = torch.zeros(sequences * e, device="cuda", dtype=torch.int32)
    counts = counts.index_add_(0, slot, valid.to(torch.int32)).view(sequences, e)
    tokens = torch.zeros(sequences, device="cuda", dtype=torch.int32).index_add_(0, seq, live.to(torch.int32))
    n = tokens.double().clamp(min=1.0).unsqueeze(1)
    filled = (tokens > 0).sum().double().clamp(min=1.0)
    slope = state["alpha"] * e * counts.double() / (k * n * n * filled)
    return (slope * total).sum().float(), counts, slope.float()


def _plain_router_grad(state, slope):
    logits, ids, weights, gw = state["logits"], state["ids"], state["weights"], state["grad_weights"]
    seq, live = _sequence_of_token(state)
    score, p = _probabilities(logits)
    d = slope[seq]
    grad = state["grad_loss"] * p * (1.0 - score) * (d - (d * p).sum(1, keepdim=True))
    grad = torch.where(live.unsqueeze(1), grad, 0.0)
    at = ids.clamp(min=0).long()
    gw = torch.where(ids >= 0, gw, 0.0)
    dw = weights * (1.0 - torch.gather(score, 1, at)) * (gw - (gw * weights).sum(1, keepdim=True))
    grad = grad.scatter_add(1, at, torch.where(ids >= 0, dw, 0.0))
    return grad.to(logits.dtype)


def _run_plain(state):
    case = state["case"]
    if case["op"] == "gemm":
        return _plain_product(state["a"], state["a_scale"], state["b"], state["b_scale"]).to(TYPES[case["out"]])
    if case["op"] == "grouped":
        return _plain_grouped(state, TYPES[case["out"]])
    if case["op"] == "quantize":
        return _plain_quantize(state["x"], case["swiglu"])
    if case["op"] == "router_loss":
        return _plain_router_loss(state)
    if case["op"] == "router_grad":
        return _plain_router_grad(state, state["slope"])
    loss, counts, slope = _plain_router_loss(state)
    return loss, counts, slope, _plain_router_grad(state, slope)


def _run_own(state):
    import sm120_nvfp4_b200 as ops

    case = state["case"]
    if case["op"] == "gemm":
        return ops.fp8_gemm(state["a"], state["b"], state["a_scale"], state["b_scale"], out_dtype=TYPES[case["out"]])
    if case["op"] == "grouped":
        return ops.fp8_grouped_gemm(state["x"], state["w"], state["seqlens"], state["cu_seqlens"], state["x_scale"],
                                    state["w_scale"], out_dtype=TYPES[case["out"]])
    if case["op"] == "quantize":
        return ops.quantize_fp8(state["x"], swiglu=case["swiglu"])
    if case["op"] != "router_grad":
        loss, counts, slope = ops.router_balance_loss(state["logits"], state["ids"], cu_seqlens=state["cu_seqlens"],
                                                      alpha=state["alpha"])
        if case["op"] == "router_loss":
            return loss, counts, slope
    else:
        slope = state["slope"]
    grad = ops.router_backward(state["logits"], state["ids"], topk_weights=state["weights"],
                               grad_weights=state["grad_weights"], slope=slope, grad_loss=state["grad_loss"],
                               cu_seqlens=state["cu_seqlens"])
    return grad if case["op"] == "router_grad" else (loss, counts, slope, grad)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------- work and truth


def work(case):
    if case["op"] in ("gemm", "grouped"):
        m = case["m"] if case["op"] == "gemm" else case["rows"]
        groups = 1 if case["op"] == "gemm" else min(case["groups"], case["rows"])
        n, k = case["n"], case["k"]
        scales = 4 * _blocks(k) * (m + groups * _blocks(n))
        return {"bytes": m * k + groups * n * k + scales + m * n * BYTES[case["out"]], "flops": 2.0 * m * n * k}
    if case["op"] == "quantize":
        r, k = case["rows"], case["k"]
        return {"bytes": r * k * BYTES[case["dtype"]] * (2 if case["swiglu"] else 1) + r * k + 4 * r * _blocks(k),
                "flops": (8.0 if case["swiglu"] else 3.0) * r * k}
    t, e, k, s = case["tokens"], case["experts"], case["topk"], case["sequences"]
    forward = t * e * BYTES[case["dtype"]] + 4 * t * k + 8 * s * e
    backward = 2 * t * e * BYTES[case["dtype"]] + 12 * t * k + 4 * s * e
    return {"bytes": {"router_loss": forward, "router_grad": backward, "router_step": forward + backward}[case["op"]],
            "flops": {"router_loss": 5.0, "router_grad": 9.0, "router_step": 14.0}[case["op"]] * t * e}


def _exact_product(a, a_scale, b, b_scale):
    """Block by block, as the operator is defined: exact sums of a block's products, then its two scales."""
    out = torch.zeros((a.shape[0], b.shape[0]), device=a.device, dtype=torch.float64)
    column = torch.arange(b.shape[0], device=a.device) // 128
    for j in range(a_scale.shape[1]):
        part = a[:, j * 128:(j + 1) * 128].double() @ b[:, j * 128:(j + 1) * 128].double().t()
        out += part * a_scale[:, j].double().unsqueeze(1) * b_scale[column, j].double().unsqueeze(0)
    return out


def _exact_quantize(x, swiglu):
    x = x.double()
    if swiglu:
        gate, up = x[:, :x.shape[1] // 2], x[:, x.shape[1] // 2:]
        x = gate * torch.sigmoid(gate) * up
    codes, scales = torch.empty_like(x), []
    for j in range(0, x.shape[1], 128):
        block = x[:, j:j + 128]
        scale = block.abs().amax(1).clamp(min=AMAX_FLOOR) / E4M3_MAX
        codes[:, j:j + 128] = (block / scale.unsqueeze(1)).float().to(E4M3).double()
        scales.append(scale)
    return codes, torch.stack(scales, 1)


def _exact_router(state):
    """(loss, counts, slope, gradient) sequence by sequence in FP64."""
    z, ids, cu = state["logits"].double(), state["ids"], state["cu_seqlens"].tolist()
    t, e = z.shape
    k, sequences = ids.shape[1], len(cu) - 1
    alive = (ids >= 0).any(1)
    s = torch.sigmoid(z)
    p = s / s.sum(1, keepdim=True)
    filled = max(1, sum(bool(alive[a:b].any()) for a, b in zip(cu, cu[1:])))
    loss = torch.zeros((), device="cuda", dtype=torch.float64)
    counts = torch.zeros((sequences, e), device="cuda", dtype=torch.int32)
    slope = torch.zeros((sequences, e), device="cuda", dtype=torch.float64)
    grad = torch.zeros_like(z)
    for i in range(sequences):
        rows = torch.arange(cu[i], cu[i + 1], device="cuda")[alive[cu[i]:cu[i + 1]]]
        if rows.numel() == 0:
            continue
        chosen = ids[rows].reshape(-1)
        counts[i] = torch.bincount(chosen[chosen >= 0], minlength=e)
        share = counts[i].double() * e / (k * rows.numel())
        slope[i] = state["alpha"] * share / (rows.numel() * filled)
        loss += (slope[i] * p[rows].sum(0)).sum()
        d = state["slope"][i].double() if "slope" in state else slope[i]
        centre = (p[rows] * d).sum(1, keepdim=True)
        grad[rows] = state["grad_loss"].double() * p[rows] * (1.0 - s[rows]) * (d - centre)
    w, gw = state["weights"].double(), state["grad_weights"].double()
    valid = ids >= 0
    mean = torch.where(valid, gw * w, 0.0).sum(1, keepdim=True)
    at = ids.clamp(min=0).long()
    grad.scatter_add_(1, at, torch.where(valid, w * (1.0 - s.gather(1, at)) * (gw - mean), 0.0))
    return loss, counts, slope, grad


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "gemm":
        return _exact_product(state["a"], state["a_scale"], state["b"], state["b_scale"])
    if case["op"] == "grouped":
        starts = state["starts"]
        return torch.cat([_exact_product(state["x"][a:b], state["x_scale"][a:b], state["w"][i], state["w_scale"][i])
                          for i, (a, b) in enumerate(zip(starts, starts[1:]))])
    if case["op"] == "quantize":
        return _exact_quantize(state["x"], case["swiglu"])
    values = _exact_router(state)
    if case["op"] == "router_step":
        return values
    return values[:3] if case["op"] == "router_loss" else values[3]
