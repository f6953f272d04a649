"""The attention block on the 4-bit cache in 64 bits, from its formulas, and inputs for
its tests. Nothing here calls the library."""
import math

import torch

F16_HALF, BF16_HALF = 2.0**-11, 2.0**-8
HALF = {torch.float16: F16_HALF, torch.bfloat16: BF16_HALF}


def block_bytes(page, dim):
    return page * (dim + 8)


def quantise(x):
    """(codes, scale, offset) of rows of f16 / bf16 values [..., D]; scale NaN for a row that is not finite."""
    x = x.double()
    finite = torch.isfinite(x).all(-1)
    x = torch.where(finite[..., None], x, torch.zeros_like(x))
    lo, hi = x.min(-1).values, x.max(-1).values
    offset = lo.clamp(-65504, 65504).float().half()
    scale = ((hi - lo) / 15).float().clamp(max=65504).half()
    s = scale.double()[..., None]
    codes = torch.where(s > 0, torch.round((x - offset.double()[..., None]) / s), torch.zeros_like(x)).clamp(0, 15)
    scale = torch.where(finite, scale, torch.full_like(scale, math.nan))
    return codes.to(torch.uint8), scale, torch.where(finite, offset, torch.zeros_like(offset))


def pack(k, v, page):
    """Whole pages of K and V rows [pages][heads][page][D] as the bytes [pages][heads * block]."""
    pages, heads, _, dim = k.shape
    codes_of, params_of = [], []
    for which, rows in enumerate((k, v)):
        codes, scale, offset = quantise(rows)
        packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
        if which:
            packed = packed.view(pages, heads, page // 4, 4, dim // 8, 4).transpose(3, 4)
        codes_of.append(packed.reshape(pages, heads, -1))
        params_of.append(torch.stack((scale, offset), -1).contiguous().view(torch.uint8).reshape(pages, heads, -1))
    return torch.cat(codes_of + params_of, -1).reshape(pages, -1).contiguous()


def poison(cache, slots, page, heads, dim):
    """The rows at `slots` get NaN scales and offsets (of K and of V)."""
    view = cache.view(cache.shape[0], heads, block_bytes(page, dim))
    for slot in slots:
        for at in (page * dim, page * (dim + 4)):
            view[slot // page, :, at + slot % page * 4:at + slot % page * 4 + 4] = 0xFF


def load(cache, page, heads, dim, layer_offset=0):
    """(K codes, V codes, K params, V params) of every row of a cache [pages][bytes]: codes
    [pages][heads][page][D] and (scale, offset) [pages][heads][page][2], f64."""
    n = cache.shape[0]
    blocks = cache[:, layer_offset:layer_offset + heads * block_bytes(page, dim)].reshape(n, heads, -1)
    half = page * dim // 2

    def unpack(b):
        return torch.stack((b & 15, b >> 4), -1).reshape(n, heads, page, dim).double()

    def params(at):
        return blocks[..., at:at + 4 * page].contiguous().view(torch.float16).double().view(n, heads, page, 2)

    k = unpack(blocks[..., :half].reshape(n, heads, page, dim // 2))
    v = blocks[..., half:2 * half].reshape(n, heads, page // 4, dim // 8, 4, 4).transpose(3, 4)
    return k, unpack(v.reshape(n, heads, page, dim // 2)), params(page * dim), params(page * (dim + 4))


def norm_rope(x, weight, eps, table, positions, interleaved):
    """Head rows [tokens][heads][D], f64, before the rounding."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    if table is None:
        return x
    n = table.shape[1] // 2
    cos, sin = (table.double()[positions.long()][:, None, i * n:(i + 1) * n] for i in (0, 1))
    x = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * n:2].clone(), x[..., 1:2 * n:2].clone()
        x[..., 0:2 * n:2], x[..., 1:2 * n:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :n].clone(), x[..., n:2 * n].clone()
        x[..., :n], x[..., n:2 * n] = a * cos - b * sin, b * cos + a * sin
    return x


def attention(q, cache, page, table, starts, kv_lens, kv_heads, scale, window=0, sinks=0, layer_offset=0):
    """(out, bound): [tokens][heads][D] in f64, and how far a result whose scores, softmax
    and sums are f32 and whose weights are rounded to f16 once may be from it before the
    result's own rounding. Rows outside the sequences are NaN."""
    tokens, heads, dim = q.shape
    group = heads // kv_heads
    kc, vc, kp, vp = load(cache, page, kv_heads, dim, layer_offset)
    out = torch.full((tokens, heads, dim), math.nan, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b in range(len(kv_lens)):
        n, most = kv_lens[b], table.shape[1] * page
        count = starts[b + 1] - starts[b]
        if count == 0:
            continue
        j = torch.arange(min(max(n, 0), most), device=q.device)
        pages = table[b].long()[j // page]
        exists = (pages >= 0) & (pages < cache.shape[0])
        pages = torch.where(exists, pages, torch.zeros_like(pages))
        pos = torch.arange(n - count, n, device=q.device)
        seen = (j[None] <= pos[:, None]) & exists[None]
        if window:
            seen &= (j[None] > pos[:, None] - window) | (j[None] < sinks)
        for h in range(kv_heads):
            x = q[starts[b]:starts[b + 1], h * group:(h + 1) * group].double().transpose(0, 1)
            at = (pages, torch.full_like(pages, h), j % page)
            rows = slice(starts[b], starts[b + 1]), slice(h * group, (h + 1) * group)
            if not len(j):
                out[rows] = 0
                continue
            ks, km = kp[at].unbind(-1)
            vs, vm = vp[at].unbind(-1)
            ok = seen.any(0)
            zero = torch.zeros((), dtype=torch.float64, device=q.device)
            k = torch.where(ok[:, None], kc[at] * ks[:, None] + km[:, None], zero)
            v = torch.where(ok[:, None], vc[at] * vs[:, None] + vm[:, None], zero)
            size_k = torch.where(ok, 15 * ks.abs() + km.abs(), zero)
            size_v = torch.where(ok, 15 * vs.abs() + vm.abs(), zero)
            score = scale * (x @ k.T.contiguous())
            masked = torch.where(seen[None], score, torch.full_like(score, -math.inf))
            top = masked.max(-1, keepdim=True).values
            p = torch.exp(masked - torch.where(torch.isinf(top), zero, top))
            p = torch.where(seen[None], p, zero)
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, zero + 1, total)
            # (a value that is not finite reaches the rows that see it, and no others)
            broken = ~torch.isfinite(v).all(-1)
            got = p @ torch.where(broken[:, None], zero, v)
            got[:, (seen & broken[None]).any(-1)] = math.nan
            out[rows] = got.transpose(0, 1)
            size_v = torch.where(broken, zero, size_v)
            # scores: a sum of D products and the two terms of a key, each addition within 2^-24
            # of what the sum of all sizes can be
            score_off = (dim + 8) * 2.0**-24 * abs(scale) * x.abs().sum(-1, keepdim=True) * size_k[None]
            score_off = torch.where(seen[None], score_off + 4 * 2.0**-24 * score.abs() + 4 * 2.0**-24, zero).amax(-1)
            # weights: f16 once, and an exponential of such a score, above and below the line;
            # sums of len(j) terms in f32
            off = F16_HALF + 2 * score_off + (len(j) + 16) * 2.0**-24
            reach = p @ size_v
            bound[rows] = (off * reach)[..., None].expand(-1, -1, dim).transpose(0, 1)
    return out, bound


def assert_near(got, want, bound, rows=None):
    """got (f16 / bf16) is within its own rounding of something within `bound` of want; rows: those to look at."""
    half = HALF[got.dtype]
    got, nan = got.double(), torch.isnan(want)
    allowed = half * (want.abs() + bound) + bound + 2.0**-24
    if rows is not None:
        got, want, allowed, nan = got[rows], want[rows], allowed[rows], nan[rows]
    assert torch.equal(torch.isnan(got), nan), "NaN in other places"
    off = torch.where(nan, torch.zeros_like(got), (got - want).abs() - allowed)
    worst = off.flatten().argmax()
    assert off.flatten()[worst] <= 0, (
        f"element {worst}: {got.flatten()[worst]} for {want.flatten()[worst]}, allowed {allowed.flatten()[worst]}")


def angles(rows, rotary, device="cpu"):
    rate = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * rate
    return torch.cat((a.cos(), a.sin()), -1).float().to(device)
