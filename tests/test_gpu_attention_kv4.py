"""The attention block on the 4-bit cache (qk_norm_rope, kv4_read, attention_kv4,
copy_pages, Kv4Cache) against its formulas in 64 bits."""
import math

import pytest
import torch

import kv4ref
from iree_amd import flags as F

pytestmark = pytest.mark.gpu

TYPES = {torch.float16: F.ATTENTION_TYPE_F16, torch.bfloat16: F.ATTENTION_TYPE_BF16}
F16, BF16 = torch.float16, torch.bfloat16


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------------------
# qk_norm_rope, kv4_read
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,interleaved,norm", [
    (1, 32, 8, 128, 128, False, True),
    (3, 5, 1, 64, 64, True, True),
    (7, 3, 3, 256, 64, False, False),
    (33, 4, 2, 128, 8, False, True),
    (515, 9, 3, 64, 24, False, True),
    (601, 2, 1, 256, 256, True, True),
    (700, 3, 2, 128, 0, False, True),
])
def test_norm_and_rotation(uk, cuda, dtype, tokens, heads, kv_heads, dim, rotary, interleaved, norm):
    """Rows of a joint q/k/v buffer to rows with strides of their own; in place gives the
    same bits; padding tokens (a position outside the table) and the gaps keep what they held.
    In f32: the sum of squares within 12 roundings (8 in a lane, up to 5 over the row, less what
    the first terms have behind them), halved by the root; the root, its two products, a rotation's
    product and sum one each or two: below 12 x 2^-24 of either term of a pair, and the pair's two terms
    are together at most sqrt 2 times the larger value: 17 x 2^-24, with 2^-24 for the last rounding
    below 2^-19 of the largest value of the row."""
    gen = _gen(tokens + dim)
    row = (heads + 2 * kv_heads) * dim + 8
    qkv = (_normal(gen, tokens, row) * 3).to(dtype)
    weights = [(1 + 0.2 * _normal(gen, dim)).to(dtype) if norm else None for _ in range(2)]
    table = kv4ref.angles(1000, rotary, "cuda") if rotary else None
    positions = torch.randint(0, 1000, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    padding = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    if rotary and tokens > 2:
        positions[1], positions[tokens - 1] = -1, 1000
        padding[1] = padding[tokens - 1] = True
    q, k = qkv[:, :heads * dim], qkv[:, heads * dim:(heads + kv_heads) * dim]
    outs = [torch.full((tokens, n * dim + 16), 7.0, dtype=dtype, device="cuda") for n in (heads, kv_heads)]
    flags = TYPES[dtype] | (F.ATTENTION_ROPE_INTERLEAVED if interleaved else 0)
    args = dict(q_weight=weights[0], k_weight=weights[1], eps=2.0**-17, cos_sin=table, table_rows=1000,
                rotary_dim=rotary, positions=positions, q_stride0=row, k_stride0=row)
    uk.qk_norm_rope(q, k, outs[0], outs[1], tokens, heads, kv_heads, dim, flags,
                    q_out_stride0=heads * dim + 16, k_out_stride0=kv_heads * dim + 16, **args)
    for x, n, out, w in ((q, heads, outs[0], weights[0]), (k, kv_heads, outs[1], weights[1])):
        assert bool((out[:, n * dim:] == 7).all()) and bool((out[padding] == 7).all())
        want = kv4ref.norm_rope(x.reshape(tokens, n, dim), w, 2.0**-17, table, positions.clamp(0, 999), interleaved)
        got = out[:, :n * dim].reshape(tokens, n, dim)
        bound = 2.0**-19 * want.abs().amax(-1, keepdim=True).expand_as(want)
        kv4ref.assert_near(got, want, bound, rows=~padding)
    both = qkv.clone()
    uk.qk_norm_rope(both[:, :heads * dim], both[:, heads * dim:(heads + kv_heads) * dim], both[:, :heads * dim],
                    both[:, heads * dim:(heads + kv_heads) * dim], tokens, heads, kv_heads, dim, flags,
                    q_out_stride0=row, k_out_stride0=row, **args)
    at = ~padding
    assert torch.equal(both[at][:, :heads * dim], outs[0][at][:, :heads * dim])
    assert torch.equal(both[at][:, heads * dim:(heads + kv_heads) * dim], outs[1][at][:, :kv_heads * dim])
    assert torch.equal(both[padding], qkv[padding])
    assert torch.equal(both[:, (heads + kv_heads) * dim:], qkv[:, (heads + kv_heads) * dim:])


def _rows_in_cache(cache, slots, page, heads, dim):
    kc, vc, kp, vp = kv4ref.load(cache, page, heads, dim)
    return tuple(c[slots // page, :, slots % page] for c in (kc, vc, kp, vp))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,kv_heads,dim,page,turned", [
    (1, 8, 128, 16, True), (37, 3, 64, 32, True), (5, 1, 256, 256, False), (530, 2, 128, 16, True)])
def test_rows_go_into_the_cache_and_come_back(uk, cuda, dtype, tokens, kv_heads, dim, page, turned):
    """Codes, scales and offsets to the bit (64 bits on both sides up to the code), at slots in a
    mixed order; slots outside the cache are not stored; every other byte of the pool keeps its
    value, another layer's half of each page among them; kv4_read gives the values they stand for.
    Rows: constant ones, zeros, ones with large and tiny values, on ties, with an infinity and a NaN."""
    gen = _gen(dim + tokens)
    pages = -(-tokens // page) + 2
    k = (_normal(gen, tokens, kv_heads, dim) * 2).to(dtype)
    v = _normal(gen, tokens, kv_heads, dim).to(dtype)
    if tokens > 30:
        v[0] = 0
        v[1] = 0.37
        v[2] *= 2.0**-12
        v[3] = v[3] * (30000 if dtype == F16 else 1e30)
        v[4] = torch.arange(dim, device="cuda").to(dtype) % 31 / 2      # scale 1: every half is a tie
        v[5, 0, 3], v[6, 0, 9], v[7, -1, 0] = math.inf, math.nan, -math.inf
        v[8] = v[8] * 2.0**-20
    table = kv4ref.angles(64, dim, "cuda") if turned else None
    weight = (1 + 0.1 * _normal(gen, dim)).to(dtype) if turned else None
    positions = torch.randint(0, 64, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens].long()
    given = slots.clone()
    missing = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    if tokens > 30:
        given[9], given[10] = -1, pages * page
        missing[9] = missing[10] = True
    stride = 2 * uk.kv4_page_bytes(page, kv_heads, dim)
    pool = torch.randint(0, 256, (pages, stride), generator=gen, device="cuda", dtype=torch.uint8)
    before = pool.clone()
    layer = pool.view(-1)[stride // 2:]
    k_out = torch.empty_like(k)
    uk.qk_norm_rope(None, k, None, k_out, tokens, 0, kv_heads, dim, TYPES[dtype], k_weight=weight, eps=2.0**-17,
                    cos_sin=table, table_rows=64, rotary_dim=dim, positions=positions, v=v, cache=layer, pages=pages,
                    page_stride=stride, page_size=page, slots=given)
    kept = ~missing
    want_k = kv4ref.norm_rope(k, weight, 2.0**-17, table, positions, False).float().to(dtype)
    assert torch.equal(k_out, want_k)
    mine = pool[:, stride // 2:].contiguous()
    kc, vc, kp, vp = _rows_in_cache(mine, slots[kept], page, kv_heads, dim)
    for x, codes, params in ((want_k[kept], kc, kp), (v[kept], vc, vp)):
        c, s, m = kv4ref.quantise(x)
        assert torch.equal(codes, c.double())
        both = torch.stack((s, m), -1).double()
        assert torch.equal(torch.isnan(params), torch.isnan(both))
        assert torch.equal(torch.nan_to_num(params), torch.nan_to_num(both))
    # the rest of the pool
    expect = before.clone()
    marks = kv4ref.block_bytes(page, dim)
    view, old = pool.view(pages, 2, kv_heads, marks), expect.view(pages, 2, kv_heads, marks)
    for slot in slots[kept].tolist():
        p, r = slot // page, slot % page
        new = view[p, 1]
        for a, b in ((r * dim // 2, (r + 1) * dim // 2), (page * dim + r * 4, page * dim + r * 4 + 4),
                     (page * (dim + 4) + r * 4, page * (dim + 4) + r * 4 + 4)):
            old[p, 1, :, a:b] = new[:, a:b]
        four = old[p, 1, :, page * dim // 2:page * dim].view(kv_heads, page // 4, dim // 8, 4, 4)
        four[:, r // 4, :, r % 4] = new[:, page * dim // 2:page * dim].view(kv_heads, page // 4, dim // 8, 4, 4)[
            :, r // 4, :, r % 4]
    assert torch.equal(pool, expect)
    # and back: one rounding of c * scale + offset (a fused multiply-add in f32)
    outs = [torch.full((tokens, kv_heads * dim + 8), 5.0, dtype=dtype, device="cuda") for _ in range(2)]
    uk.kv4_read(layer, pages, page, given, outs[0], outs[1], tokens, kv_heads, dim, TYPES[dtype], page_stride=stride,
                k_out_stride0=kv_heads * dim + 8, v_out_stride0=kv_heads * dim + 8)
    for out, codes, params in ((outs[0], kc, kp), (outs[1], vc, vp)):
        assert bool((out[:, kv_heads * dim:] == 5).all()) and bool((out[missing] == 5).all())
        value = codes * params[..., :1] + params[..., 1:]
        kv4ref.assert_near(out[kept][:, :kv_heads * dim].view(-1, kv_heads, dim), value, 2.0**-24 * value.abs())
    only = torch.full_like(v, 5.0)
    uk.kv4_read(layer, pages, page, given, None, only, tokens, kv_heads, dim, TYPES[dtype], page_stride=stride)
    assert torch.equal(only.view(torch.int16), outs[1][:, :kv_heads * dim].reshape(only.shape).view(torch.int16))


# ---------------------------------------------------------------------------
# attention_kv4
# ---------------------------------------------------------------------------

class Case:
    """A batch: q rows with gaps between tokens and rows of no sequence at both ends, pages in a
    mixed order, NaN in every cached row that no sequence owns, a table wider than it needs."""

    def __init__(self, seed, dtype, heads, kv_heads, dim, page, q_lens, kv_lens, front=1, back=2, size=1.0, missing=()):
        self.dtype, self.heads, self.kv_heads, self.dim, self.page = dtype, heads, kv_heads, dim, page
        self.q_lens, self.kv_lens = q_lens, kv_lens
        gen = _gen(seed)
        need = [-(-max(n, 0) // page) for n in kv_lens]
        self.pages = sum(need) + 3
        self.wide = max(need) + 1
        perm = torch.randperm(self.pages, generator=gen, device="cuda").tolist()
        table = torch.full((len(kv_lens), self.wide + 2), self.pages + 5, dtype=torch.int32)
        owned, at = [], 0
        for b, n in enumerate(need):
            mine = perm[at:at + n]
            at += n
            table[b, :n] = torch.tensor(mine, dtype=torch.int32)
            owned += [mine[t // page] * page + t % page for t in range(max(kv_lens[b], 0))]
        for b, i, entry in missing:
            table[b, i] = entry
        self.table = table.cuda()
        shape = (self.pages, kv_heads, page, dim)
        channels = torch.where(torch.arange(dim, device="cuda") % 13 == 5, 3.0, 1.0)
        self.cache = kv4ref.pack((_normal(gen, *shape) * channels).half(), _normal(gen, *shape).half(), page)
        keep = torch.zeros(self.pages * page, dtype=torch.bool)
        keep[torch.tensor(owned, dtype=torch.long)] = True
        view = self.cache.view(self.pages, kv_heads, -1)
        behind = (~keep).cuda().view(self.pages, page)
        for at in (page * dim, page * (dim + 4)):
            params = view[:, :, at:at + 4 * page].reshape(self.pages, kv_heads, page, 4)
            params[behind[:, None].expand(-1, kv_heads, -1)] = 0xFF
            view[:, :, at:at + 4 * page] = params.reshape(self.pages, kv_heads, -1)
        self.starts = [front]
        for n in q_lens:
            self.starts.append(self.starts[-1] + n)
        self.tokens = self.starts[-1] + back
        self.row = heads * dim + 8
        self.q = (_normal(gen, self.tokens, self.row) * size).to(dtype)
        self.rows = torch.zeros(self.tokens, dtype=torch.bool, device="cuda")
        self.rows[front:self.starts[-1]] = True
        self.device_starts = torch.tensor(self.starts, dtype=torch.int32, device="cuda")
        self.device_lens = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")

    def run(self, uk, scale=None, window=0, sinks=0, q=None, out=None, **more):
        if out is None:
            out = torch.full((self.tokens, self.heads * self.dim + 16), 3.0, dtype=self.dtype, device="cuda")
        uk.attention_kv4(self.q if q is None else q, out, self.cache, self.pages, self.page, self.table,
                         self.device_starts, self.device_lens, self.tokens, len(self.kv_lens), self.heads,
                         self.kv_heads, self.dim, self.wide, TYPES[self.dtype],
                         scale=self.scale(scale), window=window, sinks=sinks, page_table_stride=self.table.shape[1],
                         q_stride0=self.row, out_stride0=self.heads * self.dim + 16, **more)
        return out

    def scale(self, scale):
        return 1 / math.sqrt(self.dim) if scale is None else scale

    def check(self, out, scale=None, window=0, sinks=0):
        assert bool((out[:, self.heads * self.dim:] == 3).all()), "gaps between rows were written"
        assert bool((out[~self.rows] == 3).all()), "rows of no sequence were written"
        q = self.q[:, :self.heads * self.dim].reshape(self.tokens, self.heads, self.dim)
        want, bound = kv4ref.attention(q, self.cache, self.page, self.table[:, :self.wide], self.starts, self.kv_lens,
                                       self.kv_heads, self.scale(scale), window, sinks)
        got = out[:, :self.heads * self.dim].reshape(self.tokens, self.heads, self.dim)
        kv4ref.assert_near(got, want, bound, rows=self.rows)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (32, 8, 128, 16), (3, 3, 64, 32), (10, 2, 64, 16), (16, 1, 256, 64), (34, 2, 128, 32), (5, 1, 128, 256),
    (33, 1, 64, 128)])
def test_single_tokens(uk, cuda, dtype, heads, kv_heads, dim, page):
    """Decode steps of sequences whose lengths end before, at and behind every tile and page."""
    case = Case(heads, dtype, heads, kv_heads, dim, page, [1] * 14,
                [1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 127, 129, 300, 1111])
    case.check(case.run(uk))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (16, 4), (31, 33), (40, 0), (100, 70), (999, 4),
                                          (1 << 50, 1 << 50)])
@pytest.mark.parametrize("heads,kv_heads,dim,page,q_lens,kv_lens", [
    (8, 2, 128, 16, [1] * 6, [1, 7, 33, 64, 257, 1000]),
    (4, 2, 64, 32, [40, 1, 130, 3], [40, 260, 131, 90])])
def test_windows_and_sinks(uk, cuda, heads, kv_heads, dim, page, q_lens, kv_lens, window, sinks):
    case = Case(window % 97 + sinks % 89, F16, heads, kv_heads, dim, page, q_lens, kv_lens)
    case.check(case.run(uk, window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,q_lens,kv_lens", [
    (8, 2, 128, 32, [1, 200, 5, 64, 33], [1, 200, 300, 64, 700]),
    (3, 3, 64, 16, [150, 0, 17], [150, 80, 400]),
    (6, 1, 256, 64, [70, 9], [70, 333]),
    (12, 2, 64, 256, [300], [811]),
    (16, 16, 128, 16, [129, 2], [129, 515])])
def test_prompts(uk, cuda, dtype, heads, kv_heads, dim, page, q_lens, kv_lens):
    """Whole prompts, continued ones, a few drafted tokens, an empty sequence between others."""
    case = Case(dim + heads, dtype, heads, kv_heads, dim, page, q_lens, kv_lens)
    case.check(case.run(uk))


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [0, 5, -3]), ([4, 70, 2], [2, 66, 0]), ([90], [1])])
def test_rows_that_see_nothing_are_zero(uk, cuda, q_lens, kv_lens):
    """No cached token, or fewer than queries: the first of them stand before position 0."""
    case = Case(5, F16, 8, 2, 128, 16, q_lens, kv_lens)
    out = case.run(uk)
    case.check(out)
    empty = out[case.starts[0]:case.starts[0] + max(0, q_lens[0] - max(kv_lens[0], 0))]
    assert bool((empty[:, :8 * 128] == 0).all())


@pytest.mark.parametrize("q_len", [1, 80])
def test_pages_that_do_not_exist(uk, cuda, q_len):
    """Entries of -1 and beyond the pool hide their tokens, a whole sequence's too."""
    missing = [(0, 1, -1), (0, 4, 1 << 30), (1, 0, -7)] + [(2, i, -1) for i in range(6)]
    case = Case(11, BF16, 6, 2, 128, 16, [q_len] * 3, [150, 90, 81], missing=missing)
    out = case.run(uk)
    case.check(out)
    assert bool((out[case.starts[2]:case.starts[3], :6 * 128] == 0).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_len,size,scale", [(1, 30.0, None), (1, 1e-4, 2.0), (60, 30.0, None), (1, 1.0, 0.0),
                                              (60, 1.0, -0.3), (1, 2000.0, 1e-3), (60, 2000.0, 1e-3)])
def test_sizes_of_scores(uk, cuda, dtype, q_len, size, scale):
    """Scores that leave one key, that are all but equal, negative scales."""
    case = Case(21, dtype, 4, 2, 128, 32, [q_len] * 2, [333, 64 + q_len], size=size)
    case.check(case.run(uk, scale=scale), scale=scale)


@pytest.mark.parametrize("q_len", [1, 70])
def test_sizes_of_values(uk, cuda, q_len):
    """V rows from 2^-20 to 2^14, zeros and constants among them, in one sequence; and a key
    of most of the weight whose value is small next to the others'."""
    case = Case(31, F16, 4, 1, 64, 16, [q_len], [400])
    gen = _gen(3)
    v = _normal(gen, case.pages, 1, 16, 64)
    v = v * 2.0 ** torch.randint(-20, 15, (case.pages, 1, 16, 1), generator=gen, device="cuda")
    v[:, :, 3] = 0
    v[:, :, 7] = 1.5
    k = _normal(gen, case.pages, 1, 16, 64)
    case.cache.copy_(kv4ref.pack(k.half(), v.half(), 16))
    case.check(case.run(uk))


@pytest.mark.parametrize("which", ["keys", "values"])
@pytest.mark.parametrize("q_len", [1, 90])
def test_rows_that_are_not_finite(uk, cuda, q_len, which):
    """A cached row that was not finite (scale NaN) makes NaN of every query that sees it and of no
    other: not of earlier ones in its tile, nor of those whose window has passed it."""
    case = Case(17, F16, 4, 2, 64, 16, [q_len, q_len], [200, 210])
    view = case.cache.view(case.pages, 2, -1)
    at = (16 * 64 if which == "keys" else 16 * 68)
    for token in (150, 197):
        page = int(case.table[0, token // 16])
        view[page, 1, at + token % 16 * 4:at + token % 16 * 4 + 4] = torch.tensor([0, 0x7E, 0, 0], dtype=torch.uint8)
    for window, sinks in ((0, 0), (30, 0), (30, 151)):
        out = case.run(uk, window=window, sinks=sinks)
        case.check(out, window=window, sinks=sinks)
        bad = torch.isnan(out[case.starts[0]:case.starts[1], :4 * 64]).view(q_len, 4, 64)
        assert bool(bad[-1, 2:].all()) and not bool(bad[:, :2].any())
    assert not bool(torch.isnan(out[case.starts[1]:case.starts[2]]).any())


@pytest.mark.parametrize("heads,kv_heads,dim,kv_lens", [(8, 2, 128, [70001, 5, 20000]), (5, 1, 64, [40003]),
                                                        (2, 2, 256, [9000, 33])])
def test_long_caches_are_split(uk, cuda, heads, kv_heads, dim, kv_lens):
    """The same call with the workspace it asks for, with too little, and with none: each right,
    the first the same bits twice; what max_kv_len says changes no result beyond its rounding."""
    case = Case(7, F16, heads, kv_heads, dim, 64, [1] * len(kv_lens), kv_lens)
    nbytes = uk.attention_kv4_workspace(case.tokens, len(kv_lens), heads, kv_heads, dim, max_kv_len=max(kv_lens))
    assert nbytes > 0
    workspace = torch.full((nbytes,), 0xFF, dtype=torch.uint8, device="cuda")
    first = case.run(uk, max_kv_len=max(kv_lens), workspace=workspace)
    case.check(first)
    workspace.fill_(0x7F)
    assert torch.equal(first, case.run(uk, max_kv_len=max(kv_lens), workspace=workspace))
    assert torch.equal(first, case.run(uk, max_kv_len=max(kv_lens)))
    case.check(case.run(uk, max_kv_len=max(kv_lens), workspace=workspace[:64]))
    case.check(case.run(uk, max_kv_len=1))
    case.check(case.run(uk, max_kv_len=1 << 40))
    case.check(case.run(uk, max_kv_len=max(kv_lens), window=3000, sinks=17), window=3000, sinks=17)


@pytest.mark.parametrize("heads,kv_heads,dim,q_lens,kv_lens", [
    (4, 1, 128, [130, 40], [20000, 333]), (8, 2, 64, [33, 0, 300], [9000, 5000, 30011]), (2, 1, 256, [90], [7001])])
def test_prompts_over_long_caches_are_split(uk, cuda, heads, kv_heads, dim, q_lens, kv_lens):
    """The next part of a prompt whose first parts are cached, as above."""
    case = Case(12, BF16, heads, kv_heads, dim, 32, q_lens, kv_lens)
    nbytes = uk.attention_kv4_workspace(case.tokens, len(kv_lens), heads, kv_heads, dim, max_kv_len=max(kv_lens))
    assert nbytes > 0
    workspace = torch.full((nbytes,), 0xFF, dtype=torch.uint8, device="cuda")
    first = case.run(uk, max_kv_len=max(kv_lens), workspace=workspace)
    case.check(first)
    workspace.fill_(0x7F)
    assert torch.equal(first, case.run(uk, max_kv_len=max(kv_lens), workspace=workspace))
    case.check(case.run(uk, max_kv_len=max(kv_lens), workspace=workspace[:64]))
    case.check(case.run(uk, max_kv_len=1))
    case.check(case.run(uk, max_kv_len=max(kv_lens), window=2500, sinks=40), window=2500, sinks=40)


@pytest.mark.parametrize("q_len,every,batch,heads", [(1, 1, 65, 2), (1, 41, 4200, 3), (120, 9, 130, 16)])
def test_many_sequences(uk, cuda, q_len, every, batch, heads):
    """More sequences than a wave looks at in one step, most without queries between those with."""
    q_lens = [q_len if b % every == every // 2 else 0 for b in range(batch)]
    case = Case(batch, F16, heads, 1, 64, 16, q_lens, [b % 50 + q_len for b in range(batch)])
    case.check(case.run(uk))


def test_no_pages(uk, cuda):
    """A page table without columns, or a pool without pages: nothing is visible."""
    case = Case(4, F16, 4, 2, 64, 16, [1, 100], [5, 100])
    case.wide = 0
    out = case.run(uk)
    case.wide, case.pages = case.table.shape[1] - 2, 0
    for out in (out, case.run(uk)):
        assert bool((out[case.rows][:, :4 * 64] == 0).all()) and bool((out[~case.rows] == 3).all())


def test_two_calls_at_once(uk, cuda):
    """Calls on two streams, each with the workspace that it takes for itself, do not disturb each other."""
    cases = [Case(50 + i, F16, 8, 2, 128, 64, [1, 1], [20000 - 999 * i, 7000]) for i in range(2)]
    want = [case.run(uk) for case in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[torch.full_like(w, 3.0) for _ in range(10)] for w in want]
    torch.cuda.synchronize()
    for turn in range(10):
        for case, stream, mine in zip(cases, streams, outs):
            case.run(uk, out=mine[turn], stream=stream)
    torch.cuda.synchronize()
    assert all(torch.equal(out, w) for w, mine in zip(want, outs) for out in mine)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(F16, 8, 2, 128), (BF16, 4, 4, 64), (F16, 2, 1, 256)])
def test_caches_too_large_to_stay_in_the_device_s_caches(uk, cuda, dtype, heads, kv_heads, dim):
    """Steps whose keys may come to more than the device's caches hold, by the longest length, which read
    them past these; each result is that of the step that is told of short ones, or nearly."""
    kv_lens = [30001] + [3 * i for i in range(40)]
    case = Case(8, dtype, heads, kv_heads, dim, 16, [1] * 41, kv_lens)
    case.check(case.run(uk, max_kv_len=30001))
    case.check(case.run(uk, max_kv_len=100))


def test_windows_past_every_position_are_none(uk, cuda):
    sizes = (2, 2, 8, 2, 128)
    for window in (2**31, 2**63 - 1):
        for sinks in (0, 2**63 - 1):
            assert uk.attention_kv4_workspace(*sizes, max_kv_len=1 << 17, window=window, sinks=sinks) == \
                uk.attention_kv4_workspace(*sizes, max_kv_len=1 << 17)


def test_a_pool_past_32_bits(uk, cuda):
    """Pages whose bytes begin beyond 4 GiB, stored, read back, attended and copied."""
    dim, page, heads, pages, stride = 128, 16, 1, 4200, 1 << 20
    pool = torch.empty(pages, stride, dtype=torch.uint8, device="cuda")
    gen = _gen(1)
    use = [4199, 3, 4150, 2100]
    n = 50
    k, v = _normal(gen, n, heads, dim).half(), _normal(gen, n, heads, dim).half()
    slots = torch.tensor([use[t // page] * page + t % page for t in range(n)], device="cuda")
    uk.qk_norm_rope(None, k, None, None, n, 0, heads, dim, F.ATTENTION_TYPE_F16, v=v, cache=pool, pages=pages,
                    page_stride=stride, page_size=page, slots=slots)
    q = _normal(gen, 1, 4, dim).half()
    small = torch.stack([pool[p, :kv4ref.block_bytes(page, dim)] for p in use])
    table = torch.tensor([use], dtype=torch.int32, device="cuda")
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")

    def attend(table):
        out = torch.empty_like(q)
        uk.attention_kv4(q, out, pool, pages, page, table, one, lens, 1, 1, 4, heads, dim, 4, F.ATTENTION_TYPE_F16,
                         scale=0.1, page_stride=stride)
        return out

    want, bound = kv4ref.attention(q, small, page, torch.arange(4, device="cuda")[None], [0, 1], [n], heads, 0.1)
    out = attend(table)
    kv4ref.assert_near(out, want, bound)
    uk.copy_pages(pool, pages, stride, [4199, 4150, 3], [4198, 10, 4000])
    moved = torch.tensor([[4198, 4000, 10, 2100]], dtype=torch.int32, device="cuda")
    assert torch.equal(out, attend(moved))


def test_on_another_stream(uk, cuda):
    """Work given a stream runs behind that stream's own work, given as an object, a handle or as the
    current stream."""
    case = Case(3, F16, 8, 2, 128, 64, [1, 1], [30000, 12345])
    want = case.run(uk)
    side = torch.cuda.Stream()
    right = case.q.clone()
    for form in range(3):
        q = torch.zeros_like(right)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(2000000)
            q.copy_(right)
            out = torch.full_like(want, 3.0)
            if form == 2:
                case.run(uk, q=q, out=out)
        if form < 2:
            case.run(uk, q=q, out=out, stream=side if form == 0 else side.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_captured_and_replayed(uk, cuda):
    """Two graphs of a long decode step, replayed in turns with eager steps between: each has the
    eager call's bits for the inputs and lengths that it finds at its replay."""
    cases = [Case(40 + i, F16, 8, 2, 128, 64, [1, 1], [20000, 7000 + i]) for i in range(2)]
    graphs, outs = [], []
    for case in cases:
        case.run(uk)
        out = torch.full((case.tokens, 8 * 128 + 16), 3.0, dtype=F16, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            case.run(uk, out=out)
        graphs.append(graph)
        outs.append(out)
    for turn in range(4):
        for case, graph, out in zip(cases, graphs, outs):
            case.q.mul_(-0.7)
            case.device_lens.sub_(311)
            case.kv_lens = [n - 311 for n in case.kv_lens]
            out.fill_(3.0)
            graph.replay()
        eager = [case.run(uk) for case in cases]
        torch.cuda.synchronize()
        for case, out, want in zip(cases, outs, eager):
            assert torch.equal(out, want)
            if turn == 3:
                case.check(out)


def test_block_of_a_decode_step_captured(uk, cuda):
    """Norm, rotation, append and attention of two steps in one graph give the eager bits."""
    gen = _gen(77)
    heads, kv_heads, dim, page, batch = 8, 2, 64, 16, 3
    pool = uk.Kv4Cache(40, page, 1, kv_heads, dim)
    seqs = [pool.new() for _ in range(batch)]
    qkv = _normal(gen, 60 * batch, (heads + 2 * kv_heads) * dim).half()
    table = kv4ref.angles(256, dim, "cuda")
    row = qkv.shape[1]

    def step(x, n, slots, positions, tables, starts, out):
        q, k, v = x[:, :heads * dim], x[:, heads * dim:(heads + kv_heads) * dim], x[:, (heads + kv_heads) * dim:]
        turned = torch.empty(n, heads * dim, dtype=F16, device="cuda")
        uk.qk_norm_rope(q, k, turned, None, n, heads, kv_heads, dim, F.ATTENTION_TYPE_F16, cos_sin=table,
                        table_rows=256, rotary_dim=dim, positions=positions, q_stride0=row, k_stride0=row, v=v,
                        v_stride0=row, cache=pool.layer(0), pages=pool.pages, page_size=page, slots=slots)
        uk.attention_kv4(turned, out, pool.layer(0), pool.pages, page, tables[0], starts, tables[1], n, batch, heads,
                         kv_heads, dim, tables[2], F.ATTENTION_TYPE_F16, scale=0.125)

    slots = pool.extend(seqs, [50, 7, 31])
    lens = [50, 7, 31]
    positions = torch.cat([torch.arange(n) for n in lens]).int().cuda()
    starts = torch.tensor([0, 50, 57, 88], dtype=torch.int32, device="cuda")
    prompt = torch.empty(88, heads * dim, dtype=F16, device="cuda")
    step(qkv[:88], 88, slots, positions, pool.tables(seqs), starts, prompt)
    one = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    slots = pool.extend(seqs, [1] * batch)
    tables = pool.tables(seqs)
    x, positions = qkv[88:88 + batch].clone(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.empty(batch, heads * dim, dtype=F16, device="cuda")
    before = pool.buffer.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(x, batch, slots, positions, tables, one, out)
    for turn in range(3):
        x.copy_(qkv[88 + batch * turn:88 + batch * (turn + 1)])
        pool.buffer.copy_(before)
        graph.replay()
        after = pool.buffer.clone()
        pool.buffer.copy_(before)
        eager = torch.empty_like(out)
        step(x, batch, slots, positions, tables, one, eager)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(after, pool.buffer)


def test_layer_of_a_decode_step(uk, cuda):
    """One layer of 32 sequences, as a program runs it: int4 projections of q, k and v, norms, rotation
    and append, attention, the int4 output projection, the fp8 gate/up/down block. Each stage of
    the block against 64 bits on the inputs that it got, and all of it in one graph, replayed over
    steps, against the eager bits; a sequence that has ended is padding (position and slot -1)."""
    gen = _gen(123)
    batch, heads, kv_heads, dim, page, ffn, gs = 32, 4, 2, 64, 16, 512, 128
    hidden, row = heads * dim, (heads + 2 * kv_heads) * dim
    pool = uk.Kv4Cache(200, page, 1, kv_heads, dim)
    seqs = [pool.new() for _ in range(batch)]
    table = kv4ref.angles(256, dim, "cuda")
    weights = [(1 + 0.1 * _normal(gen, dim)).half() for _ in range(2)]

    def int4(n, k):
        w = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        tiled = torch.empty_like(w)
        uk.pack_i4_weights(w, tiled, n, k)
        scale = (torch.rand(n, k // gs, generator=gen, device="cuda") * 0.01 + 0.005).half()
        zp = torch.full((n, k // gs), 7.5, dtype=F16, device="cuda")
        return w, tiled, scale, zp

    def project(x, weight, out, n, k):
        uk.dequant_matmul_i4(x, weight[1], weight[2], weight[3], out, batch, n, k, gs, F.DEQUANT_MATMUL_W_TILED)

    def dense(weight, n, k):
        codes = torch.stack((weight[0] & 15, weight[0] >> 4), -1).view(n, k // gs, gs).double()
        return ((codes - 7.5) * weight[2].double()[..., None]).view(n, k)

    w_qkv, w_o = int4(row, hidden), int4(hidden, hidden)
    codes = [torch.randint(0, 120, (n,), generator=gen, device="cuda", dtype=torch.uint8)
             for n in (ffn * hidden, ffn * hidden, hidden * ffn)]
    mlp = uk.Fp8Mlp(hidden, ffn, *codes, 2e-3, 2e-3, 2e-3, 0.05, 0.05, max_tokens=batch)
    ones = torch.arange(batch + 1, dtype=torch.int32, device="cuda")

    class Step:
        def __init__(self):
            self.qkv = torch.empty(batch, row, dtype=F16, device="cuda")
            self.turned, self.seen, self.added = (torch.empty(batch, hidden, dtype=F16, device="cuda") for _ in range(3))
            self.y = torch.empty(batch, hidden, dtype=torch.float32, device="cuda")

        def run(self, x, positions, slots, tables):
            project(x, w_qkv, self.qkv, row, hidden)
            q, k, v = self.qkv[:, :hidden], self.qkv[:, hidden:-kv_heads * dim], self.qkv[:, -kv_heads * dim:]
            uk.qk_norm_rope(q, k, self.turned, None, batch, heads, kv_heads, dim, F.ATTENTION_TYPE_F16,
                            q_weight=weights[0], k_weight=weights[1], eps=2.0**-17, cos_sin=table, table_rows=256,
                            rotary_dim=dim, positions=positions, q_stride0=row, k_stride0=row, v=v, v_stride0=row,
                            cache=pool.layer(0), pages=pool.pages, page_size=page, slots=slots)
            uk.attention_kv4(self.turned, self.seen, pool.layer(0), pool.pages, page, tables[0], ones, tables[1], batch,
                             batch, heads, kv_heads, dim, tables[2], F.ATTENTION_TYPE_F16, scale=dim**-0.5)
            project(self.seen, w_o, self.added, hidden, hidden)
            mlp(self.added, self.y, batch)

    # what is cached before the first step: rows of their own, nothing for the first sequence
    lens = [7 * i % 61 for i in range(batch)]
    slots = pool.extend(seqs, lens)
    k, v = (_normal(gen, sum(lens), kv_heads, dim).half() for _ in range(2))
    uk.qk_norm_rope(None, k, None, None, sum(lens), 0, kv_heads, dim, F.ATTENTION_TYPE_F16, v=v, cache=pool.layer(0),
                    pages=pool.pages, page_size=page, slots=slots)
    eager, replayed = Step(), Step()
    # (tables for all steps at once, as wide as they come to be; lengths and slots are a step's own)
    steps = 3
    new_slots = pool.extend(seqs, [steps] * batch).view(batch, steps)
    wide_table, _, wide = pool.tables(seqs)
    x, positions = torch.empty(batch, hidden, dtype=F16, device="cuda"), torch.empty_like(ones[:batch])
    slots, kv_lens = torch.empty(batch, dtype=torch.int64, device="cuda"), torch.empty_like(positions)
    tables = (wide_table, kv_lens, wide)
    ended = 9
    graph = None
    for step in range(steps):
        x.copy_(_normal(gen, batch, hidden))
        positions.copy_(torch.tensor(lens).int() + step)
        slots.copy_(new_slots[:, step])
        kv_lens.copy_(positions + 1)
        if step:
            positions[ended] = slots[ended] = -1
            kv_lens[ended] = 0
        before = pool.buffer.clone()
        eager.turned.zero_()
        eager.run(x, positions, slots, tables)
        after = pool.buffer.clone()
        if graph is None:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                replayed.run(x, positions, slots, tables)
        pool.buffer.copy_(before)
        replayed.turned.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool.buffer, after)
        for name in ("qkv", "turned", "seen", "added", "y"):
            assert torch.equal(getattr(eager, name), getattr(replayed, name)), name
        assert bool(torch.isfinite(eager.y).all())
        # projections: f32 sums of exact products, or of products with a weight rounded to f16, one
        # rounding at the end
        for got, weight, source in ((eager.qkv, w_qkv, x), (eager.added, w_o, eager.seen)):
            w = dense(weight, got.shape[1], hidden)
            size = source.double().abs() @ w.abs().T.contiguous()
            kv4ref.assert_near(got, source.double() @ w.T.contiguous(), size * (2.0**-11 + hidden * 2.0**-24))
        live = positions >= 0
        q = eager.qkv[:, :hidden].view(batch, heads, dim)
        want = kv4ref.norm_rope(q, weights[0], 2.0**-17, table, positions.clamp(min=0), False)
        # (f32: 64 products and a few steps more)
        kv4ref.assert_near(eager.turned.view(batch, heads, dim), want, 80 * 2.0**-24 * want.abs().amax(-1, keepdim=True), live)
        want, bound = kv4ref.attention(eager.turned.view(batch, heads, dim), pool.buffer, page, wide_table,
                                       list(range(batch + 1)), kv_lens.tolist(), kv_heads, dim**-0.5)
        kv4ref.assert_near(eager.seen.view(batch, heads, dim), want, bound)
        if step:
            assert bool((eager.seen[ended] == 0).all()) and bool((eager.turned[ended] == 0).all())


# ---------------------------------------------------------------------------
# copy_pages, Kv4Cache
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("pages,page_bytes,gap,count", [(5, 16, 0, 2), (9, 48, 16, 4), (2000, 4352, 0, 900),
                                                        (12, 1 << 20, 64, 5)])
def test_copy_pages(uk, cuda, pages, page_bytes, gap, count):
    gen = _gen(pages)
    stride = page_bytes + gap
    pool = torch.randint(0, 256, (pages, stride), generator=gen, device="cuda", dtype=torch.uint8)
    perm = torch.randperm(pages, generator=gen, device="cuda").int().cpu()
    src, dst = perm[:count].contiguous(), perm[count:2 * count].contiguous()
    src[count - 1] = src[0]                        # a page may be copied to several
    want = pool.clone()
    want[dst.long().cuda(), :page_bytes] = want[src.long().cuda(), :page_bytes]
    uk.copy_pages(pool, pages, page_bytes, src, dst, page_stride=stride)
    assert torch.equal(pool, want)
    uk.copy_pages(pool, pages, page_bytes, [], [])
    assert torch.equal(pool, want)


def test_copy_pages_captured(uk, cuda):
    """A captured call copies its pages as they are at each replay; what the program does with its
    lists of page numbers afterwards changes nothing. 800 pairs: more than one launch."""
    gen = _gen(6)
    pool = torch.empty(2000, 144, dtype=torch.uint8, device="cuda")
    perm = torch.randperm(2000, generator=gen, device="cuda").int().cpu()
    src, dst = perm[:800].clone(), perm[800:1600].clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        uk.copy_pages(pool, 2000, 144, src, dst)
    at = src.long().cuda(), dst.long().cuda()
    src.fill_(0)
    dst.fill_(1999)
    for _ in range(3):
        pool.copy_(torch.randint(0, 256, (2000, 144), generator=gen, device="cuda", dtype=torch.uint8))
        want = pool.clone()
        want[at[1]] = want[at[0]]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool, want)


def test_sequences_fork_drop_and_compact(uk, cuda):
    """What a sequence attends to survives forks, the ends of others, a compaction and pages dropped
    behind a window, over two layers; a fork's tokens are its own."""
    gen = _gen(9)
    heads, kv_heads, dim, page, layers = 4, 2, 64, 16, 2
    pool = uk.Kv4Cache(64, page, layers, kv_heads, dim)
    rows = {}

    def append(seq, n):
        slots = pool.extend([seq], [n])
        for layer in range(layers):
            k, v = (_normal(gen, n, kv_heads, dim).half() for _ in range(2))
            uk.qk_norm_rope(None, k, None, None, n, 0, kv_heads, dim, F.ATTENTION_TYPE_F16, v=v,
                            cache=pool.layer(layer), pages=pool.pages, page_stride=pool.page_bytes, page_size=page,
                            slots=slots)
            old = rows.get((seq, layer))
            both = torch.stack([kv4ref.pack(x[:, :, None].repeat(1, 1, 16, 1), x[:, :, None].repeat(1, 1, 16, 1), 16)
                                for x in (k, v)])
            rows[seq, layer] = both if old is None else torch.cat((old, both), 1)

    def check(seqs, window=0, sinks=0):
        table, lens, wide = pool.tables(seqs)
        starts = torch.arange(len(seqs) + 1, dtype=torch.int32, device="cuda")
        q = _normal(gen, len(seqs), heads, dim).half()
        for layer in range(layers):
            out = torch.empty_like(q)
            uk.attention_kv4(q, out, pool.layer(layer), pool.pages, page, table, starts, lens, len(seqs), len(seqs),
                             heads, kv_heads, dim, wide, F.ATTENTION_TYPE_F16, scale=0.2, window=window, sinks=sinks,
                             page_stride=pool.page_bytes)
            for i, seq in enumerate(seqs):
                n = pool.length(seq)
                # the rows themselves, in pages of a cache of their own: K from one half, V from the other
                kc, _, kp, _ = kv4ref.load(rows[seq, layer][0], 16, kv_heads, dim)
                _, vc, _, vp = kv4ref.load(rows[seq, layer][1], 16, kv_heads, dim)
                k = (kc[:, :, 0] * kp[:, :, 0, :1] + kp[:, :, 0, 1:])[:n]
                v = (vc[:, :, 0] * vp[:, :, 0, :1] + vp[:, :, 0, 1:])[:n]
                j = torch.arange(n, device="cuda")
                seen = (j > n - 1 - window) | (j < sinks) if window else j >= 0
                x = q[i].double().view(kv_heads, heads // kv_heads, dim)
                score = 0.2 * (x @ k.permute(1, 2, 0).contiguous())
                p = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
                want = (p @ v.transpose(0, 1).contiguous()).view(heads, dim)
                # (as kv4ref.attention: a weight's rounding, and twice a score's (64 + 8) 2^-24 0.2 sum |q| (below
                # 90) (15 scale + |offset|) (below 20), which is 2^-8; a V row's 15 scale + |offset| is at most
                # 3 times its largest value)
                bound = (2.0**-11 + 2.0**-8) * 3 * (p @ v.abs().amax(-1).T.contiguous()[..., None]).expand(
                    -1, -1, dim).reshape(heads, dim)
                kv4ref.assert_near(out[i], want, bound)

    a, b = pool.new(), pool.new()
    append(a, 53)
    append(b, 32)
    check([a, b])
    c, d = pool.fork(a), pool.fork(b)
    for new, old in ((c, a), (d, b)):
        for layer in range(layers):
            rows[new, layer] = rows[old, layer].clone()
    assert pool.free_pages() == 64 - (4 + 1 + 2)      # a's last page was copied, b's full pages are shared
    append(a, 5)
    append(c, 20)
    append(d, 1)
    check([a, b, c, d])
    pool.free(a)
    append(b, 40)
    assert pool.compact() == 64 - pool.free_pages()
    check([b, c, d])
    table = pool.tables([b, c, d])[0]
    assert int(table.max()) < 64 - pool.free_pages()
    before = pool.free_pages()
    pool.drop(b, 20, sinks=3)
    assert pool.free_pages() == before + 1 and pool.tables([b])[0][0].tolist().count(-1) == 2   # (one is d's too)
    check([b], window=20, sinks=3)
    append(b, 30)
    check([b, c, d], window=20, sinks=3)
    for seq in (b, c, d):
        pool.free(seq)
    assert pool.free_pages() == 64
