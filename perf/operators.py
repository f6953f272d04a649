"""The attention block of a language model on a cache held in 4 bits, as cases to time.

Four operators, each in its plain form (elementary torch operations) and, with
``own`` set, through the framework's entry points on the same inputs:

  rope       RMS norm of every query and key head and their position rotation, rows to rows
  append     the same with K and V going to a paged 4-bit cache, and the rows read back
  attention  attention over the paged cache: decode steps and prompts, sliding windows, sinks
  pages      pages of a cache copied inside their pool: forks, a compaction

The cache. A page holds ``page`` tokens of every kv head, one block of page * (D + 8)
bytes per head: the K codes [page][D / 2] (two per byte, even d in the low nibble), the V
codes as dwords [page / 4][D / 8][4 tokens] (a dword: 8 consecutive d of one token), then
scale and offset (f16 each) of every token's K row and of every V row. A code c stands
for c * scale + offset, scale = (max - min) / 15 and offset = min of the row, both in f16.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One sequence decodes one token: 32 query and 8 key heads of 128, a few microseconds.
        {"name": "rope_f16_1", "op": "rope", "type": "f16", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False},
        # A prompt of an odd length whose heads rotate only their first half, pairs side by side.
        {"name": "rope_bf16_4099", "op": "rope", "type": "bf16", "tokens": 4099, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 64, "interleaved": True},
        # 33 sequences decode a token each into the cache, small heads.
        {"name": "append_f16_33", "op": "append", "type": "f16", "tokens": 33, "heads": 16, "kv_heads": 4, "dim": 64,
         "rotary": 64, "interleaved": False, "page": 16},
        # A long prompt goes into the cache.
        {"name": "append_bf16_8191", "op": "append", "type": "bf16", "tokens": 8191, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "page": 32},
        # The latency of one short sequence's decode step.
        {"name": "decode_f16_1x300", "op": "attention", "type": "f16", "batch": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 300,
         "kv_hi": 300, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "sinks": 0},
        # A serving batch of 32 sequences of different lengths.
        {"name": "decode_f16_32x8192", "op": "attention", "type": "f16", "batch": 32, "q_lo": 1, "q_hi": 1,
         "kv_lo": 1000, "kv_hi": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "window": 0, "sinks": 0},
        # 64 long chats, each sees its last 1024 positions and its first 4.
        {"name": "decode_bf16_window", "op": "attention", "type": "bf16", "batch": 64, "q_lo": 1, "q_hi": 1,
         "kv_lo": 4001, "kv_hi": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 1024, "sinks": 4},
        # Two very long documents: the work is split over their length.
        {"name": "decode_f16_2x131072", "op": "attention", "type": "f16", "batch": 2, "q_lo": 1, "q_hi": 1,
         "kv_lo": 100001, "kv_hi": 131072, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "sinks": 0},
        # A ragged batch of prompts, some continued, small heads, a window and sinks.
        {"name": "prompt_bf16_ragged", "op": "attention", "type": "bf16", "batch": 5, "q_lo": 1, "q_hi": 1500,
         "kv_lo": 77, "kv_hi": 3001, "heads": 16, "kv_heads": 2, "dim": 64, "page": 16, "window": 512, "sinks": 8},
        # One prompt of 4096 tokens.
        {"name": "prompt_f16_4096", "op": "attention", "type": "f16", "batch": 1, "q_lo": 4096, "q_hi": 4096,
         "kv_lo": 4096, "kv_hi": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "window": 0, "sinks": 0},
        # Eight sequences fork: the last, partly filled page of each is copied. 32 layers a page.
        {"name": "pages_fork_8", "op": "pages", "pages": 64, "moves": 8, "page": 16, "kv_heads": 8, "dim": 128,
         "layers": 32},
        # A pool is compacted: 600 pages move to the front.
        {"name": "pages_compact_600", "op": "pages", "pages": 1400, "moves": 600, "page": 16, "kv_heads": 8, "dim": 128,
         "layers": 32},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope", "append", "attention", "attention", "attention", "attention", "pages"))
    kind = rng.choice(("f16", "bf16"))
    if op in ("rope", "append"):
        dim = rng.choice((64, 128, 256))
        kv_heads = rng.randint(1, 1024 // dim)
        heads = kv_heads * rng.randint(1, 32 // max(kv_heads, 4))
        case = {"op": op, "type": kind, "tokens": _log(rng, 1, 8191 * 48 * 128 // ((heads + 2 * kv_heads) * dim) // 4),
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rng.choice((dim, dim // 2)),
                "interleaved": rng.random() < 0.5}
        if op == "append":
            case["page"] = rng.choice((16, 32, 64, 128))
        return case
    if op == "pages":
        pages = _log(rng, 24, 1400)
        return {"op": op, "pages": pages, "moves": rng.randint(1, pages * 3 // 7), "page": rng.choice((16, 32)),
                "kv_heads": rng.randint(1, 8), "dim": rng.choice((64, 128)), "layers": rng.randint(1, 16)}
    dim = rng.choice((64, 128, 128, 256))
    kv_heads = rng.randint(1, 1024 // dim)
    heads = kv_heads * rng.randint(1, 16 // max(kv_heads, 2))
    case = {"op": op, "type": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": rng.choice((16, 32, 64, 128)), "window": 0, "sinks": 0}
    if rng.random() < 0.6:      # a decode step, or a few drafted tokens at once
        case["batch"] = _log(rng, 1, 64)
        case["kv_hi"] = _log(rng, 1, min(65536, 262144 // case["batch"]))
        case["q_hi"] = rng.choice((1, 1, 1, rng.randint(2, 9)))
    else:
        case["batch"] = _log(rng, 1, 6)
        case["q_hi"] = _log(rng, 10, 2048 // case["batch"])
        case["kv_hi"] = case["q_hi"] + rng.choice((0, _log(rng, 1, 2048)))
    case["kv_hi"] = max(case["kv_hi"], case["q_hi"])
    case["q_lo"] = rng.randint(1, case["q_hi"])
    case["kv_lo"] = rng.randint(1, case["kv_hi"])
    if rng.random() < 0.4:
        case["window"] = _log(rng, 1, max(2, case["kv_hi"]))
        case["sinks"] = rng.choice((0, 1, 4, 37))
    return case


def _spread(n, lo, hi):
    """n whole numbers from hi to lo, evenly spread and in a mixed order."""
    order = sorted(range(n), key=lambda i: i * 2654435761 % 2**32)
    return [hi - (hi - lo) * i // max(n - 1, 1) for i in order]


def _lengths(case):
    """Query tokens and cached tokens (the queries' own among them) of every sequence."""
    q = _spread(case["batch"], case["q_lo"], case["q_hi"])
    kv = _spread(case["batch"], case["kv_lo"], case["kv_hi"])[::-1]
    return q, [max(a, b) for a, b in zip(q, kv)]


def _block_bytes(page, dim):
    return page * (dim + 8)


def _visible(first, last, window, sinks):
    """Keys that at least one query at positions first..last sees, and the pairs that are visible."""
    if not window:
        return last + 1, (last + 1) * (last + 2) // 2 - first * (first + 1) // 2
    lo = max(0, first - window + 1)
    keys = last + 1 - lo + min(sinks, lo)
    pairs = sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(first, last + 1))
    return keys, pairs


def work(case):
    if case["op"] == "pages":
        return {"bytes": 2 * case["moves"] * case["layers"] * case["kv_heads"] * _block_bytes(case["page"], case["dim"]),
                "flops": 0}
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] in ("rope", "append"):
        t = case["tokens"]
        rows = h + (2 if case["op"] == "append" else 1) * kv
        out = 2 * t * (h + kv) * d if case["op"] == "rope" else 2 * t * h * d + 2 * t * kv * (d + 8) + 4 * t * kv * d
        return {"bytes": 2 * t * rows * d + 4 * t * case["rotary"] + out, "flops": 8 * t * (h + kv) * d}
    keys = pairs = rows = 0
    for q, n in zip(*_lengths(case)):
        k, p = _visible(n - q, n - 1, case["window"], case["sinks"])
        keys, pairs, rows = keys + k, pairs + p, rows + q
    return {"bytes": keys * kv * (d + 8) + 4 * rows * h * d, "flops": 4 * pairs * h * d}


def _quantise(x):
    """Codes (uint8), scale and offset (f16) of rows of f16 or bf16 values, in 64 bits up to the code."""
    x = x.double()
    low, high = x.amin(-1), x.amax(-1)
    offset, scale = low.half(), ((high - low) / 15).half()
    s, m = scale.double()[..., None], offset.double()[..., None]
    codes = torch.where(s > 0, torch.round((x - m) / s), torch.zeros_like(x)).clamp(0, 15)
    return codes.to(torch.uint8), scale, offset


def _store(k, v, page):
    """K and V rows [pages][kv heads][page][D] (f16) as the bytes of a cache [pages][kv heads * block]."""
    pages, heads, _, dim = k.shape
    parts, params = [], []
    for rows, is_v in ((k, False), (v, True)):
        codes, scale, offset = _quantise(rows)
        codes = codes.view(pages, heads, page, dim // 2, 2)
        packed = codes[..., 0] | (codes[..., 1] << 4)
        if is_v:
            packed = packed.view(pages, heads, page // 4, 4, dim // 8, 4).transpose(3, 4)
        parts.append(packed.reshape(pages, heads, -1))
        params.append(torch.stack((scale, offset), -1).view(torch.uint8).reshape(pages, heads, -1))
    return torch.cat(parts + params, -1).reshape(pages, -1).contiguous()


def _angles(rows, rotary):
    """cos and sin of every position's rotation [rows][rotary], f32: the table a model keeps."""
    rate = 10000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * rate
    return torch.cat((angle.cos(), angle.sin()), -1).float().contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    def order(n):
        return torch.randperm(n, generator=gen, device="cuda")

    if case["op"] == "pages":
        nbytes = case["layers"] * case["kv_heads"] * _block_bytes(case["page"], case["dim"])
        pool = torch.randint(-2**31, 2**31 - 1, (case["pages"], nbytes // 4), generator=gen, device="cuda",
                             dtype=torch.int32)
        perm = order(case["pages"]).int().cpu()
        return {"case": case, "pool": pool, "src": perm[:case["moves"]].contiguous(),
                "dst": perm[case["moves"]:2 * case["moves"]].contiguous(), "nbytes": nbytes}

    h, kv, d, dtype = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["type"]]
    # (a few channels of keys are several times as large as the others, as in trained models)
    channels = torch.where(torch.arange(d, device="cuda") % 29 == 3, 4.0, 1.0)
    if case["op"] in ("rope", "append"):
        t = case["tokens"]
        qkv = normal(t, (h + 2 * kv) * d).mul_(2.0)
        qkv[:, h * d:(h + kv) * d].view(t, kv, d).mul_(channels)
        state = {"case": case, "qkv": qkv.to(dtype), "table": _angles(32768, case["rotary"]),
                 "positions": torch.randint(0, 32768, (t,), generator=gen, device="cuda", dtype=torch.int32),
                 "q_weight": (1 + 0.1 * normal(d)).to(dtype), "k_weight": (1 + 0.1 * normal(d)).to(dtype),
                 "q_out": torch.empty(t, h, d, dtype=dtype, device="cuda"),
                 "k_out": torch.empty(t, kv, d, dtype=dtype, device="cuda")}
        if case["op"] == "append":
            pages = -(-t // case["page"]) + 3
            state["v_out"] = torch.empty_like(state["k_out"])
            state["pages"] = pages
            state["cache"] = torch.zeros(pages, kv * _block_bytes(case["page"], d), dtype=torch.uint8, device="cuda")
            # (the prompt's pages lie anywhere in the pool, its tokens in order inside them)
            where = order(pages)[torch.arange(t, device="cuda") // case["page"]]
            state["slots"] = (where * case["page"] + torch.arange(t, device="cuda") % case["page"]).long()
        return state

    q_lens, kv_lens = _lengths(case)
    page, batch = case["page"], case["batch"]
    need = [-(-n // page) for n in kv_lens]
    most, pages = max(need), sum(need) + 2
    table = torch.full((batch, most), -1, dtype=torch.int32)
    perm, at = order(pages).int().cpu(), 0
    for b, n in enumerate(need):
        table[b, :n], at = perm[at:at + n], at + n
    cache = torch.empty(pages, kv * _block_bytes(page, d), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (kv * page * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        cache[p:p + n] = _store((normal(n, kv, page, d) * channels).half(), normal(n, kv, page, d).half(), page)
    starts = [0]
    for n in q_lens:
        starts.append(starts[-1] + n)
    tokens = starts[-1]
    return {"case": case, "cache": cache, "pages": pages, "table": table.cuda(), "tokens": tokens, "most": most,
            "q": normal(tokens, h, d).to(dtype), "out": torch.empty(tokens, h, d, dtype=dtype, device="cuda"),
            "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
            "kv_lens": torch.tensor(kv_lens, dtype=torch.int32, device="cuda"),
            "q_most": max(q_lens), "kv_most": max(kv_lens)}


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _norm_rotate(x, weight, table, positions, interleaved, wide):
    """Rows [tokens][heads][D] normed and rotated, in the type `wide`."""
    x = x.to(wide)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 2.0**-20) * weight.to(wide)
    rotary = table.shape[1]
    angles = table[positions.long()].to(wide)[:, None]
    cos, sin = angles[..., :rotary // 2], angles[..., rotary // 2:]
    part = x[..., :rotary]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., :rotary // 2], part[..., rotary // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rotary:]), -1)


def _plain_rope(s):
    c, qkv = s["case"], s["qkv"]
    h, kv, d, t = c["heads"], c["kv_heads"], c["dim"], c["tokens"]
    # (a key next to the border between two codes has to fall on the right side of it)
    wide = torch.float64 if c["op"] == "append" else torch.float32
    q, k = qkv[:, :h * d].view(t, h, d), qkv[:, h * d:(h + kv) * d].view(t, kv, d)
    q = _norm_rotate(q, s["q_weight"], s["table"], s["positions"], c["interleaved"], torch.float32).to(qkv.dtype)
    k = _norm_rotate(k, s["k_weight"], s["table"], s["positions"], c["interleaved"], wide).to(qkv.dtype)
    if c["op"] == "rope":
        return q, k
    v = qkv[:, (h + kv) * d:].view(t, kv, d)
    return (q,) + tuple(_as_cached(x) for x in (k, v))


def _as_cached(x):
    codes, scale, offset = _quantise(x)
    return (codes.float() * scale.float()[..., None] + offset.float()[..., None]).to(x.dtype)


def _plain_attention(s):
    c = s["case"]
    h, kv, d, page, batch = c["heads"], c["kv_heads"], c["dim"], c["page"], c["batch"]
    group, most, dev = h // kv, s["most"] * page, s["q"].device
    blocks = s["cache"].view(s["pages"], kv, -1)[s["table"].long().clamp(min=0)].transpose(1, 2)
    half = page * d // 2

    def params(at):
        both = blocks[..., at:at + 4 * page].contiguous().view(torch.float16).float()
        return both.view(batch, kv, most, 2)

    def values(nibbles, at):
        low_high = torch.stack((nibbles & 15, nibbles >> 4), -1).reshape(batch, kv, most, d).float()
        both = params(at)
        return low_high * both[..., :1] + both[..., 1:]

    k = values(blocks[..., :half].reshape(batch, kv, most, d // 2), 2 * half)
    v = blocks[..., half:2 * half].reshape(batch, kv, most // 4, d // 8, 4, 4).transpose(3, 4)
    v = values(v.reshape(batch, kv, most, d // 2), 2 * half + 4 * page)

    # queries as a dense [batch][longest]: rows past a sequence's own repeat its last one
    starts, lens = s["starts"].long(), s["kv_lens"].long()
    count = starts[1:] - starts[:-1]
    at = torch.arange(s["q_most"], device=dev)
    rows = starts[:-1, None] + torch.minimum(at[None], count[:, None] - 1)
    q = s["q"].float()[rows].view(batch, s["q_most"], kv, group, d).permute(0, 2, 3, 1, 4)
    scores = q.reshape(batch, kv, group * s["q_most"], d) @ k.transpose(-1, -2)
    scores = scores.view(batch, kv, group, s["q_most"], most) / math.sqrt(d)
    pos = (lens - count)[:, None] + at[None]
    key = torch.arange(most, device=dev)
    seen = (key[None, None] <= pos[..., None]) & (key[None, None] < lens[:, None, None])
    if c["window"]:
        seen &= (key[None, None] > pos[..., None] - c["window"]) | (key[None, None] < c["sinks"])
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where((key[None] < lens[:, None])[:, None, :, None], v, torch.zeros_like(v))
    o = p.view(batch, kv, group * s["q_most"], most) @ v
    o = o.view(batch, kv, group, s["q_most"], d) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, s["q_most"], h, d)
    return o[at[None] < count[:, None]].to(s["q"].dtype)


def run(state):
    c = state["case"]
    if own:
        import iree_amd
        from iree_amd import flags as F
        if c["op"] == "pages":
            iree_amd.copy_pages(state["pool"], c["pages"], state["nbytes"], state["src"], state["dst"])
            return state["pool"]
        h, kv, d = c["heads"], c["kv_heads"], c["dim"]
        kind = F.ATTENTION_TYPE_F16 if c["type"] == "f16" else F.ATTENTION_TYPE_BF16
        if c["op"] == "attention":
            iree_amd.attention_kv4(state["q"], state["out"], state["cache"], state["pages"], c["page"], state["table"],
                                   state["starts"], state["kv_lens"], state["tokens"], c["batch"], h, kv, d,
                                   state["most"], kind, scale=1 / math.sqrt(d), window=c["window"], sinks=c["sinks"],
                                   max_kv_len=state["kv_most"])
            return state["out"]
        t, row = c["tokens"], (h + 2 * kv) * d
        flags = kind | (F.ATTENTION_ROPE_INTERLEAVED if c["interleaved"] else 0)
        q, k, v = state["qkv"][:, :h * d], state["qkv"][:, h * d:(h + kv) * d], state["qkv"][:, (h + kv) * d:]
        turn = dict(q_weight=state["q_weight"], k_weight=state["k_weight"], eps=2.0**-20, cos_sin=state["table"],
                    table_rows=32768, rotary_dim=c["rotary"], positions=state["positions"], q_stride0=row,
                    k_stride0=row)
        if c["op"] == "rope":
            iree_amd.qk_norm_rope(q, k, state["q_out"], state["k_out"], t, h, kv, d, flags, **turn)
            return state["q_out"], state["k_out"]
        iree_amd.qk_norm_rope(q, k, state["q_out"], None, t, h, kv, d, flags, **turn, v=v, v_stride0=row,
                              cache=state["cache"], pages=state["pages"], page_size=c["page"], slots=state["slots"])
        iree_amd.kv4_read(state["cache"], state["pages"], c["page"], state["slots"], state["k_out"], state["v_out"], t,
                          kv, d, kind)
        return state["q_out"], state["k_out"], state["v_out"]
    if c["op"] == "pages":
        dev = state["pool"].device
        state["pool"][state["dst"].to(dev).long()] = state["pool"][state["src"].to(dev).long()]
        return state["pool"]
    return _plain_attention(state) if c["op"] == "attention" else _plain_rope(state)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_turn(x, weight, table, positions, interleaved):
    """Pairs of one head row as complex numbers, turned by cos + i sin."""
    x = x.double()
    x = x / ((x.square().sum(-1, keepdim=True) / x.shape[-1]) + 2.0**-20).sqrt() * weight.double()
    n = table.shape[1] // 2
    turn = torch.complex(*(table.double()[positions.long()][:, None, i * n:(i + 1) * n].contiguous() for i in (0, 1)))
    i = torch.arange(n, device=x.device)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    z = torch.complex(x[..., first], x[..., second]) * turn
    out = x.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_cached(x):
    """The nearest of a row's sixteen values to each of its elements, the even code where two are as near."""
    x = x.double()
    lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    s, m = ((hi - lo) / 15).half().double(), lo.half().double()
    best, far = m.expand_as(x).clone(), (x - m).abs()
    for code in range(1, 16):
        value = code * s + m
        gap = (x - value).abs()
        nearer = (gap < far) | ((gap == far) & (code % 2 == 0))
        best, far = torch.where(nearer, value, best), torch.where(nearer, gap, far)
    return best


def exact(case, seed):
    if case["op"] == "pages":
        return None
    s = prepare(case, seed)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] in ("rope", "append"):
        parts = s["qkv"].view(case["tokens"], h + 2 * kv, d).split((h, kv, kv), 1)
        q, k = (_exact_turn(x, w, s["table"], s["positions"], case["interleaved"])
                for x, w in ((parts[0], s["q_weight"]), (parts[1], s["k_weight"])))
        if case["op"] == "rope":
            return q, k
        # (the cache takes keys in the type of the rows)
        return q, _exact_cached(k.to(s["qkv"].dtype)), _exact_cached(parts[2])
    page, group = case["page"], h // kv
    token = torch.arange(s["most"] * page, device="cuda")
    pieces = []
    for b, (q_len, kv_len) in enumerate(zip(*_lengths(case))):
        t = token[:kv_len]
        block, inside = s["table"][b].long()[t // page], t % page
        pair, four = torch.arange(d // 2, device="cuda"), torch.arange(4, device="cuda")
        dword = (inside // 4)[:, None] * (d // 8) * 4 + (pair // 4)[None] * 4 + (inside % 4)[:, None]
        heads_out = []
        q = s["q"][int(s["starts"][b]):int(s["starts"][b + 1])].double()
        pos = torch.arange(kv_len - q_len, kv_len, device="cuda")
        seen = t[None] <= pos[:, None]
        if case["window"]:
            seen &= (t[None] >= pos[:, None] - (case["window"] - 1)) | (t[None] < case["sinks"])
        for n in range(kv):
            mine = s["cache"].view(s["pages"], kv, -1)[:, n]
            k_codes = mine[block[:, None], inside[:, None] * (d // 2) + pair]
            v_codes = mine[block[:, None], page * d // 2 + dword * 4 + pair % 4]
            k_par = mine[block[:, None], page * d + inside[:, None] * 4 + four]
            v_par = mine[block[:, None], page * (d + 4) + inside[:, None] * 4 + four]
            cols = []
            for codes, par in ((k_codes, k_par), (v_codes, v_par)):
                par = par.contiguous().view(torch.float16).double()
                wide = torch.empty(kv_len, d, dtype=torch.float64, device="cuda")
                wide[:, 0::2], wide[:, 1::2] = (codes % 16).double(), (codes // 16).double()
                cols.append(wide * par[:, :1] + par[:, 1:])
            rows = q[:, n * group:(n + 1) * group].transpose(0, 1)
            p = torch.softmax((rows @ cols[0].T.contiguous() / math.sqrt(d)).masked_fill(~seen[None], -math.inf), -1)
            heads_out.append((p @ cols[1]).transpose(0, 1))
        pieces.append(torch.cat(heads_out, 1))
    return torch.cat(pieces, 0)
