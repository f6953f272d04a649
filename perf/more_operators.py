"""A layer in 8-bit integers and its experts, as cases to time.

Five operators, each in its plain form (elementary torch operations) and, with
``own`` set, through the framework's entry points on the same inputs:

  norm      the residual's addition (of one addend, or of several with weights: what a token's
            experts give), RMS norm, and rows of 8 bits with a scale for each token
  quantize  rows in 8 bits with a scale for each token, of rows or of silu(gate) * up
  matmul    8-bit rows times packed 8-bit weights, a scale for each token and for each channel
  route     each token's experts and weights from its logits, and the tokens in expert order
  grouped   the same product by expert, over ragged groups of rows: rows gathered from the
            tokens (the first product of the experts) or results scattered to them (the second)

A row of 8 bits is q = rne(127 y / max|y|) with the scale max|y| / 127. Weights lie in tiles
[N / 32][K / 16][32][16], zeros past N and K, and for several experts one after the other.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 2.0**-20


def listed():
    return [
        # One token of a decode step between two layers.
        {"name": "norm_f16_1", "op": "norm", "type": "f16", "tokens": 1, "dim": 4096, "addends": 1, "weighted": False},
        # A prompt of an odd length.
        {"name": "norm_bf16_4099", "op": "norm", "type": "bf16", "tokens": 4099, "dim": 4096, "addends": 1,
         "weighted": False},
        # The eight experts of every token of a prompt added up with their weights.
        {"name": "norm_bf16_2048x8", "op": "norm", "type": "bf16", "tokens": 2048, "dim": 4096, "addends": 8,
         "weighted": True},
        # 33 sequences decode: what attention left, an odd number of elements.
        {"name": "quantize_f16_33x5001", "op": "quantize", "type": "f16", "rows": 33, "cols": 5001, "gated": False},
        # The gate of a large feed-forward block over a prompt.
        {"name": "quantize_bf16_2048_gated", "op": "quantize", "type": "bf16", "rows": 2048, "cols": 14336, "gated": True},
        # One token against the weights of a feed-forward block: their bytes are all that counts.
        {"name": "matmul_f16_1", "op": "matmul", "type": "f16", "m": 1, "n": 14336, "k": 4096, "bias": False},
        # A few hundred tokens, a long sum, few columns, with a bias.
        {"name": "matmul_bf16_500", "op": "matmul", "type": "bf16", "m": 500, "n": 4096, "k": 14336, "bias": True},
        # A prompt of 4096 tokens.
        {"name": "matmul_bf16_4096", "op": "matmul", "type": "bf16", "m": 4096, "n": 4096, "k": 4096, "bias": False},
        # A decode step of 32 sequences.
        {"name": "route_bf16_32", "op": "route", "type": "bf16", "tokens": 32, "experts": 64, "top": 8, "renorm": True,
         "padding": False},
        # A prompt of an odd length, a part of it padding, logits in f32.
        {"name": "route_f32_8191", "op": "route", "type": "f32", "tokens": 8191, "experts": 128, "top": 8, "renorm": False,
         "padding": True},
        # The experts' second product in a decode step of 32 sequences: 4 rows to an expert.
        {"name": "grouped_f16_32", "op": "grouped", "type": "f16", "tokens": 32, "experts": 64, "top": 8, "n": 4096,
         "k": 1792, "scatter": True, "padding": False},
        # The experts' first product over a prompt: gate and up, 512 rows to an expert.
        {"name": "grouped_bf16_4096", "op": "grouped", "type": "bf16", "tokens": 4096, "experts": 64, "top": 8, "n": 3584,
         "k": 4096, "scatter": False, "padding": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of a tensor: whole 64s more often than not, else any."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.4 else max(64, n // 64 * 64)


def draw(rng):
    op = rng.choice(("norm", "norm", "quantize", "matmul", "matmul", "matmul", "route", "grouped", "grouped", "grouped"))
    kind = rng.choice(("f16", "bf16"))
    if op == "norm":
        dim, addends = _size(rng, 64, 16384), rng.choice((1, 1, 1, rng.randint(2, 8)))
        return {"op": op, "type": kind, "tokens": _log(rng, 1, 8192 * 4096 // (dim * (addends + 2))), "dim": dim,
                "addends": addends, "weighted": addends > 1}
    if op == "quantize":
        cols = _size(rng, 64, 28672)
        return {"op": op, "type": kind, "rows": _log(rng, 1, 2048 * 14336 // cols), "cols": cols,
                "gated": rng.random() < 0.6}
    if rng.random() < 0.2:
        kind = "f32"
    if op == "matmul":
        m, n, k = _log(rng, 1, 4096), _size(rng, 64, 14336), _size(rng, 64, 14336)
        while m * n * k > 4096**3:
            m = max(1, m // 2)
        return {"op": op, "type": kind, "m": m, "n": n, "k": k, "bias": rng.random() < 0.4}
    experts, padding = rng.choice((8, 16, 60, 64, 128, 256)), rng.random() < 0.3
    top = rng.randint(1, min(8, experts))
    if op == "route":
        return {"op": op, "type": kind, "tokens": _log(rng, 1, 16384), "experts": experts, "top": top,
                "renorm": rng.random() < 0.5, "padding": padding}
    n, k = _size(rng, 64, 4096), _size(rng, 64, 4096)
    while experts * n * k > 2**29:
        n, k = max(64, n // 2), max(64, k // 2)
    tokens = _log(rng, 1, 4096)
    while tokens * top * n * k > 2**38 or experts * tokens * top * max(n, k) > 2**35:
        tokens = max(1, tokens // 2)
    return {"op": op, "type": kind, "tokens": tokens, "experts": experts, "top": top, "n": n, "k": k,
            "scatter": rng.random() < 0.5, "padding": padding}


def _padded(n, to):
    return -(-n // to) * to


def _tokens_with_experts(case):
    """Of a prompt with padding, the last eighth has none."""
    return case["tokens"] - (case["tokens"] // 8 if case["padding"] else 0)


def work(case):
    op = case["op"]
    if op == "norm":
        t, d, a = case["tokens"], case["dim"], case["addends"]
        # addends, residual and the sum in 16 bits, the rows in 8, scales, the norm's weight
        return {"bytes": t * d * (2 * a + 5) + 4 * t + 2 * d + (4 * t * a if case["weighted"] else 0),
                "flops": t * d * (2 * a + 5)}
    if op == "quantize":
        r, c = case["rows"], case["cols"]
        return {"bytes": r * c * (5 if case["gated"] else 3) + 4 * r, "flops": r * c * (8 if case["gated"] else 3)}
    out = 4 if case["type"] == "f32" else 2
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + out * m * n + 4 * (m + n + (n if case["bias"] else 0)), "flops": 2 * m * n * k}
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["top"]
        return {"bytes": t * e * out + t * k * 12 + 4 * (e + 1), "flops": t * e * 4}
    # Of the experts' weights those that some token takes; as if the choices were independent of each other.
    e, n, k, rows = case["experts"], case["n"], case["k"], _tokens_with_experts(case) * case["top"]
    taken = e * (1 - (1 - case["top"] / e) ** _tokens_with_experts(case))
    lhs = rows if case["scatter"] else _tokens_with_experts(case)
    return {"bytes": int(taken * n * (k + 4)) + lhs * (k + 4) + rows * (n * out + 4), "flops": 2 * rows * n * k}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    def codes(*shape):
        """Rows of 8 bits as quantised normal values have them."""
        return normal(*shape).mul_(32).round_().clamp_(-127, 127).to(torch.int8)

    def empty(*shape, dtype=dtype):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    # (a few channels are many times as large as the others, as in trained models)
    def channels(n):
        return torch.where(torch.arange(n, device="cuda") % 97 == 5, 12.0, 1.0)

    state = {"case": case}
    if op == "norm":
        t, d, a = case["tokens"], case["dim"], case["addends"]
        state["x"] = (normal(t, a, d) * channels(d)).to(dtype)
        state["residual"] = (normal(t, d) * channels(d) * 3).to(dtype)
        state["weight"] = (1 + 0.2 * normal(d)).to(dtype)
        state["addend_weights"] = torch.softmax(normal(t, a), -1).contiguous() if case["weighted"] else None
        state["sum"], state["q"], state["scale"] = empty(t, d), empty(t, d, dtype=torch.int8), empty(t, dtype=torch.float32)
        return state
    if op == "quantize":
        r, c = case["rows"], case["cols"]
        # (gate and up are the two halves of one product's rows)
        state["x"] = (normal(r, 2 * c if case["gated"] else c) * 1.5).to(dtype)
        state["q"], state["scale"] = empty(r, c, dtype=torch.int8), empty(r, dtype=torch.float32)
        return state
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["top"]
        state["logits"] = _logits(case, normal).to(dtype)
        state["ids"], state["weights"] = empty(t, k, dtype=torch.int32), empty(t, k, dtype=torch.float32)
        state["offsets"], state["rows"] = empty(e + 1, dtype=torch.int32), empty(t * k, dtype=torch.int32)
        return state

    experts = case["experts"] if op == "grouped" else 1
    n, k = case["n"], case["k"]
    wide, high = _padded(k, 16), _padded(n, 32)
    weights = torch.zeros(experts, high, wide, dtype=torch.int8, device="cuda")
    for e in range(experts):
        weights[e, :n, :k] = codes(n, k)
    state["packed"] = weights.view(experts, high // 32, 32, wide // 16, 16).transpose(2, 3).contiguous()
    state["weights"] = weights[:, :n, :k].contiguous()
    state["rhs_scale"] = (normal(experts, n).abs() + 0.5).mul_(1 / 4096)
    if op == "matmul":
        lhs = case["m"]
        state["bias"] = normal(n) if case["bias"] else None
        state["out"] = empty(lhs, n)
    else:
        ids = _choose(_logits(case, normal), case["top"])
        order = torch.argsort(ids.flatten(), stable=True)
        count = torch.bincount(ids.flatten(), minlength=experts + 1)[:experts]
        state["offsets"] = torch.cat((count.new_zeros(1), count.cumsum(0))).int()
        state["rows"] = order.int()
        state["rows"][int(state["offsets"][-1]):] = -1
        state["most"] = int(count.max())
        positions = case["tokens"] * case["top"]
        lhs = positions if case["scatter"] else case["tokens"]
        state["positions"], state["lhs_rows"], state["out"] = positions, lhs, empty(positions, n)
    state["lhs"] = torch.zeros(lhs, wide, dtype=torch.int8, device="cuda")
    state["lhs"][:, :k] = codes(lhs, k)
    state["lhs_scale"] = (normal(lhs).abs() + 0.5).mul_(1 / 32)
    return state


def _logits(case, normal):
    """Some experts are more popular than others; a token that is padding has no expert."""
    logits = normal(case["tokens"], case["experts"]) * 1.5 + normal(case["experts"]) * 0.4
    logits[_tokens_with_experts(case):] = -math.inf
    return logits


def _choose(logits, top):
    """The experts of every token, the number of experts in the place of one that there is not."""
    values, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    return torch.where(values[:, :top] > -math.inf, ids[:, :top], logits.shape[1])


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _plain_codes(y):
    """Rows (64 bits: a value next to the border between two codes has to fall on the right side) in 8 bits; their largest."""
    top = y.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, torch.round(y * 127 / top), torch.zeros_like(y))
    return q.to(torch.int8), top[..., 0]


def _plain_norm(s):
    x, weights = s["x"].double(), s["addend_weights"]
    if weights is not None:
        x = x * weights.double()[..., None]
    total = (s["residual"].double() + x.sum(1)).to(s["x"].dtype)
    wide = total.double()
    rate = torch.rsqrt((wide * wide).mean(-1) + EPS)
    q, top = _plain_codes(wide * s["weight"].double())
    return total, q, (top * rate / 127).float()


def _plain_quantize(s):
    c, x = s["case"], s["x"].double()
    if c["gated"]:
        gate, up = x[:, :c["cols"]], x[:, c["cols"]:]
        x = gate / (1 + torch.exp(-gate)) * up
    q, top = _plain_codes(x)
    return q, (top / 127).float()


def _plain_matmul(s):
    k = s["case"]["k"]
    y = s["lhs"][:, :k].float() @ s["weights"][0].float().T
    y = y * s["lhs_scale"][:, None] * s["rhs_scale"][0]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["out"].dtype)


def _plain_route(s):
    c = s["case"]
    e, k = c["experts"], c["top"]
    logits = s["logits"].float()
    ids = _choose(logits, k)
    there = ids < e
    top = logits.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(logits - top)
    mine = torch.where(there, torch.gather(p, 1, ids.clamp(max=e - 1)), torch.zeros_like(p[:, :k]))
    total = mine.sum(-1, keepdim=True) if c["renorm"] else p.sum(-1, keepdim=True)
    weights = torch.where(there, mine / total, torch.zeros_like(mine))
    flat = ids.flatten()
    order = torch.sort(flat, stable=True).indices
    count = (flat[:, None] == torch.arange(e, device=flat.device)).sum(0)
    offsets = torch.cat((count.new_zeros(1), count.cumsum(0)))
    rows = torch.where(torch.arange(flat.numel(), device=flat.device) < offsets[-1], order, -1)
    return torch.where(there, ids, -1).int(), weights, offsets.int(), rows.int()


def _plain_grouped(s):
    c = s["case"]
    offsets, rows = s["offsets"].long(), s["rows"].long()
    # every expert's positions side by side, as many as the most popular has
    at = offsets[:-1, None] + torch.arange(s["most"], device=rows.device)
    there = at < offsets[1:, None]
    at = torch.where(there, at, 0)
    source = at if c["scatter"] else (rows[at] // c["top"]).clamp(min=0)
    lhs = s["lhs"][:, :c["k"]][source].float()
    y = torch.bmm(lhs, s["weights"].float().transpose(1, 2).contiguous())
    y = y * s["lhs_scale"][source][..., None] * s["rhs_scale"][:, None]
    out = torch.zeros_like(s["out"])
    target = rows[at] if c["scatter"] else at
    out[target[there]] = y[there].to(out.dtype)
    return out


def run(state):
    c = state["case"]
    op = c["op"]
    if own:
        import iree_amd
        from iree_amd import flags as F
        kind = {"f16": F.ROWS_TYPE_F16, "bf16": F.ROWS_TYPE_BF16, "f32": F.ROWS_TYPE_F32}[c["type"]]
        if op == "norm":
            iree_amd.rms_norm_quantize(state["x"], state["q"], state["scale"], c["tokens"], c["dim"], kind,
                                       weight=state["weight"], eps=EPS, residual=state["residual"], sum_out=state["sum"],
                                       addends=c["addends"], addend_weights=state["addend_weights"])
            return state["sum"], state["q"], state["scale"]
        if op == "quantize":
            if c["gated"]:
                iree_amd.quantize_rows(state["x"], state["q"], state["scale"], c["rows"], c["cols"], kind,
                                       up=state["x"][:, c["cols"]:], x_stride0=2 * c["cols"], up_stride0=2 * c["cols"])
            else:
                iree_amd.quantize_rows(state["x"], state["q"], state["scale"], c["rows"], c["cols"], kind)
            return state["q"], state["scale"]
        if op == "matmul":
            iree_amd.matmul_w8a8(state["lhs"], state["packed"], state["out"], state["lhs_scale"], state["rhs_scale"],
                                 c["m"], c["n"], c["k"], kind, bias=state["bias"])
            return state["out"]
        if op == "route":
            iree_amd.moe_route(state["logits"], state["ids"], state["weights"], state["offsets"], state["rows"],
                               c["tokens"], c["experts"], c["top"], kind | (F.ROUTE_RENORMALIZE if c["renorm"] else 0))
            return state["ids"], state["weights"], state["offsets"], state["rows"]
        move = F.GROUPED_SCATTER if c["scatter"] else F.GROUPED_GATHER
        iree_amd.grouped_matmul_w8a8(state["lhs"], state["packed"], state["out"], state["lhs_scale"], state["rhs_scale"],
                                     state["offsets"], state["positions"], c["experts"], c["n"], c["k"], kind | move,
                                     lhs_rows=state["lhs_rows"], rows=state["rows"], rows_per_token=c["top"])
        return state["out"]
    return {"norm": _plain_norm, "quantize": _plain_quantize, "matmul": _plain_matmul, "route": _plain_route,
            "grouped": _plain_grouped}[op](state)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        total = s["residual"].double()
        for j in range(case["addends"]):
            total = total + s["x"][:, j].double() * (1.0 if s["addend_weights"] is None else s["addend_weights"][:, j, None].double())
        # (the norm is that of the sum as it is kept)
        kept = total.to(s["x"].dtype).double()
        y = s["weight"].double() * kept / (kept.square().sum(-1, keepdim=True) / case["dim"] + EPS).sqrt()
        return total, None, y.abs().max(-1).values / 127
    if op == "quantize":
        x = s["x"].double()
        if case["gated"]:
            gate, up = x.split(case["cols"], 1)
            x = torch.sigmoid(gate) * gate * up
        return None, x.abs().max(-1).values / 127
    if op == "route":
        logits = s["logits"].double()
        p = torch.softmax(logits, -1).nan_to_num(nan=0.0)
        best = torch.topk(p, case["top"], -1).values
        return None, best / best.sum(-1, keepdim=True).clamp(min=1e-300) if case["renorm"] else best, None, None
    k = case["k"]
    if op == "matmul":
        lhs = s["lhs"][:, :k].double() * s["lhs_scale"].double()[:, None]
        y = torch.mm(lhs, (s["weights"][0].double() * s["rhs_scale"][0].double()[:, None]).T.contiguous())
        return y if s["bias"] is None else y + s["bias"].double()
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    rows, ends = s["rows"].tolist(), s["offsets"].tolist()
    for e in range(case["experts"]):
        mine = range(ends[e], ends[e + 1])
        if not len(mine):
            continue
        source = torch.tensor([p if case["scatter"] else rows[p] // case["top"] for p in mine], device="cuda")
        target = torch.tensor([rows[p] if case["scatter"] else p for p in mine], device="cuda")
        product = s["lhs"][source, :k].double() @ s["weights"][e].double().T.contiguous()
        out[target] = product * s["lhs_scale"][source].double()[:, None] * s["rhs_scale"][e].double()
    return out
