"""The layer in 8-bit integers and its experts on the device, against the 64-bit reference."""
import math

import pytest
import torch

import iree_amd
import w8a8ref as ref
from iree_amd import flags as F

pytestmark = pytest.mark.gpu
TYPES, FLAGS = ref.TYPES, ref.FLAGS


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(gen, kind, *shape):
    x = torch.randn(*shape, generator=gen) * 2
    x[..., ::29] *= 9
    return x.to(TYPES[kind])


def _norm(x, kind, residual=None, weight=None, factors=None, eps=2.0**-20, keep=True):
    """The call on tight copies; (sum, q, scale) on the CPU."""
    tokens, addends, dim = x.shape
    on = lambda t: None if t is None else t.cuda()  # noqa: E731
    q = torch.full((tokens, dim), 99, dtype=torch.int8, device="cuda")
    scale = torch.full((tokens,), -1.0, device="cuda")
    out = torch.zeros(tokens, dim, dtype=TYPES[kind], device="cuda") if keep else None
    iree_amd.rms_norm_quantize(on(x), q, scale, tokens, dim, FLAGS[kind], weight=on(weight), eps=eps, residual=on(residual),
                               sum_out=out, addends=addends, addend_weights=on(factors))
    return None if out is None else out.cpu(), q.cpu(), scale.cpu()


def _assert_norm(got, x, residual, weight, factors, eps=2.0**-20):
    h = ref.total(x, residual, factors)
    q, scale = ref.norm(h, weight, eps)
    assert torch.equal(got[0].nan_to_num(7), h.nan_to_num(7))
    assert torch.equal(got[1], q)
    assert torch.equal(torch.isnan(got[2]), torch.isnan(scale))
    # (64 bits, rounded once to 32)
    assert ((got[2].double() - scale).abs().nan_to_num(0) <= (1.001 * 2.0**-24) * scale.abs().nan_to_num(0)).all()


DIMS = [1, 7, 8, 9, 16, 64, 121, 128, 129, 333, 512, 513, 1024, 1025, 2048, 2049, 2050, 4096, 4099, 8192, 8200, 16384, 16390, 32768, 65529, 65536]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_norm(cuda, kind, dim):
    gen = _gen(dim)
    x, residual, weight = _rows(gen, kind, 5, 1, dim), _rows(gen, kind, 5, dim), _rows(gen, kind, dim)
    _assert_norm(_norm(x, kind, residual, weight), x, residual, weight, None)


@pytest.mark.parametrize("addends", [2, 5, 8, 33])
@pytest.mark.parametrize("dim", [40, 1500, 4096, 20000])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_norm_of_several_addends(cuda, kind, dim, addends):
    gen = _gen(dim + addends)
    x, residual = _rows(gen, kind, 3, addends, dim), _rows(gen, kind, 3, dim)
    factors = torch.softmax(torch.randn(3, addends, generator=gen), -1)
    factors[1, 0] = 0                        # what its row holds is not looked at
    x[1, 0] = math.nan
    _assert_norm(_norm(x, kind, residual, None, factors), x, residual, None, factors)
    x[1, 0] = 1
    _assert_norm(_norm(x, kind), x, None, None, None)


@pytest.mark.parametrize("dim", [64, 4096, 9000])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_norm_of_special_rows(cuda, kind, dim):
    gen = _gen(dim)
    x, weight = _rows(gen, kind, 8, 1, dim), (1 + torch.rand(dim, generator=gen)).to(TYPES[kind])
    x[0] = 0                                 # a row of nothing
    x[1, 0, 5] = math.inf
    x[2, 0, dim - 1] = math.nan
    x[3] = x[3] * 1e-7                       # (f16: subnormals)
    x[4] = 0
    x[4, 0, 3] = -1
    x[5] = torch.randint(-254, 255, (dim,), generator=gen).to(TYPES[kind])    # halves between two codes
    x[5, 0, 0] = 254
    x[6] = torch.finfo(TYPES[kind]).max / 8 if kind == "f16" else 1e30
    weight[7] = 0
    _assert_norm(_norm(x, kind, None, weight), x, None, weight, None)
    _assert_norm(_norm(x, kind, None, None), x, None, None, None)
    _assert_norm(_norm(x[3:6], kind, None, None, eps=0.0), x[3:6], None, None, None, eps=0.0)
    # a weight of 0 next to a value that is not finite
    x[7, 0, 7] = math.inf
    assert torch.isnan(_norm(x, kind, None, weight)[2][7])


def test_norm_takes_strides_and_runs_in_place(cuda):
    gen, dim, tokens = _gen(3), 257, 6
    x, residual = _rows(gen, "bf16", tokens, 2, dim), _rows(gen, "bf16", tokens, dim)
    big = torch.zeros(tokens, 2, 300, dtype=torch.bfloat16)
    big[:, :, 3:3 + dim] = x
    held = torch.zeros(tokens, 271, dtype=torch.bfloat16)
    held[:, 1:1 + dim] = residual
    held_gpu, big_gpu = held.cuda(), big.cuda()
    q = torch.full((tokens, 301), 55, dtype=torch.int8, device="cuda")
    scale = torch.zeros(tokens, device="cuda")
    at = held_gpu.view(-1)[1:]
    iree_amd.rms_norm_quantize(big_gpu.view(-1)[3:], q.view(-1)[5:], scale, tokens, dim, F.ROWS_TYPE_BF16, residual=at,
                               sum_out=at, addends=2, x_stride0=600, x_stride1=300, residual_stride0=271,
                               sum_out_stride0=271, q_stride0=301, eps=0.25)
    got = held_gpu.cpu()
    _assert_norm((got[:, 1:1 + dim], q.cpu()[:, 5:5 + dim], scale.cpu()), x, residual, None, None, 0.25)
    assert not got[:, 0].any() and not got[:, 1 + dim:].any()
    assert (q[:, :5] == 55).all() and (q[:, 5 + dim:] == 55).all()
    # one addend onto its own row, nothing kept, nothing of a second token touched
    y = _rows(gen, "f16", 4, 1, 72)
    y_gpu = y.cuda()
    q, scale = torch.full((4, 72), 9, dtype=torch.int8, device="cuda"), torch.full((4,), 3.0, device="cuda")
    iree_amd.rms_norm_quantize(y_gpu, q, scale, 3, 72, F.ROWS_TYPE_F16, sum_out=y_gpu, eps=0.25)
    _assert_norm((y_gpu.cpu()[:3, 0], q.cpu()[:3], scale.cpu()[:3]), y[:3], None, None, None, 0.25)
    assert (q[3] == 9).all() and scale[3] == 3
    assert torch.equal(_norm(y, "f16", keep=False)[1], _norm(y, "f16")[1])


def _quantize(x, up, kind):
    rows, cols = x.shape
    q = torch.full((rows, cols), 99, dtype=torch.int8, device="cuda")
    scale = torch.full((rows,), -1.0, device="cuda")
    iree_amd.quantize_rows(x.cuda(), q, scale, rows, cols, FLAGS[kind], up=None if up is None else up.cuda())
    return q.cpu(), scale.cpu()


def _assert_rows(got, x, up):
    q, scale = ref.codes(x.double() if up is None else ref.silu_mul(x, up))
    assert torch.equal(got[0], q), (got[0] != q).nonzero()[:5]
    assert torch.equal(torch.isnan(got[1]), torch.isnan(scale))
    assert ((got[1].double() - scale).abs().nan_to_num(0) <= (1.001 * 2.0**-24) * scale.nan_to_num(0) + 2.0**-150).all()


@pytest.mark.parametrize("cols", DIMS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_rows(cuda, kind, gated, cols):
    gen = _gen(cols)
    x, up = _rows(gen, kind, 6, cols), _rows(gen, kind, 6, cols) if gated else None
    _assert_rows(_quantize(x, up, kind), x, up)


@pytest.mark.parametrize("cols", [40, 5001, 30000])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_special_rows(cuda, kind, cols):
    gen = _gen(cols)
    most = torch.finfo(TYPES[kind]).max
    x, up = _rows(gen, kind, 12, cols), _rows(gen, kind, 12, cols)
    x[0] = 0
    x[1, 7] = math.inf
    x[2, cols - 1] = math.nan
    up[3, 4] = -math.inf
    x[4] = -300                              # all gates closed as far as f32 sees
    x[5] = x[5] * 1e-6
    up[5] = up[5] * 1e-6
    x[6] = torch.linspace(-95, 95, cols).to(TYPES[kind])
    x[7] = most
    up[7] = 0
    up[7, 3] = 1 if kind == "f16" else 1e-3
    x[8] = torch.linspace(-most / 2, most / 2, cols).to(TYPES[kind])
    up[8] = 1e-3
    x[9] = -80
    up[9] = most / 4
    x[10, ::2], up[10] = -120, 3
    up[11] = 0
    _assert_rows(_quantize(x, up, kind), x, up)
    x[6] = torch.randint(-254, 255, (cols,), generator=gen).to(TYPES[kind])
    x[6, 0] = 254
    _assert_rows(_quantize(x, None, kind), x, None)
    if kind == "bf16":                       # a product that f32 does not hold
        x[0], up[0] = most, most
        q, scale = _quantize(x[:1], up[:1], kind)
        assert math.isnan(scale[0]) and not q.any()


def test_rows_take_strides(cuda):
    gen, rows, cols = _gen(5), 7, 101
    both = _rows(gen, "f16", rows, 2 * cols + 3)
    on = both.cuda()
    q, scale = torch.full((rows, 112), 44, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    iree_amd.quantize_rows(on, q, scale, rows, cols, F.ROWS_TYPE_F16, up=on.view(-1)[cols:], x_stride0=2 * cols + 3,
                           up_stride0=2 * cols + 3, q_stride0=112)
    _assert_rows((q.cpu()[:, :cols], scale.cpu()), both[:, :cols], both[:, cols:2 * cols])
    assert (q[:, cols:] == 44).all()


def _product_case(gen, M, N, K):
    wide = -(-K // 16) * 16
    lhs = torch.full((M, wide), 77, dtype=torch.int8)        # (what lies past K does not count)
    lhs[:, :K] = ref.rows8(gen, M, K)
    return lhs, ref.scales(gen, M), ref.rows8(gen, N, K), ref.scales(gen, N)


def _assert_product(kind, M, N, K, bias=False, seed=1, **how):
    gen = _gen(seed + M + N + K)
    lhs, lhs_scale, w, w_scale = _product_case(gen, M, N, K)
    extra = torch.randn(N, generator=gen) if bias else None
    out = torch.full((M, N), 5.0, dtype=TYPES[kind], device="cuda")
    iree_amd.matmul_w8a8(lhs.cuda(), ref.pack(w).cuda(), out, lhs_scale.cuda(), w_scale.cuda(), M, N, K, FLAGS[kind],
                         bias=None if extra is None else extra.cuda(), **how)
    ref.assert_near(out.cpu(), *ref.product(lhs[:, :K], lhs_scale, w, w_scale, extra))


@pytest.mark.parametrize("M,N,K", [
    (1, 1, 1), (1, 64, 64), (3, 33, 17), (15, 31, 16), (16, 32, 15), (17, 100, 100), (2, 4, 1000), (31, 65, 513), (33, 130, 64),
    (64, 64, 128), (65, 96, 129), (100, 513, 320), (128, 256, 192), (129, 257, 448), (200, 70, 2049), (256, 512, 64),
    (300, 300, 300), (1, 2048, 4096), (5, 1000, 5000), (700, 640, 1024), (1, 40, 14336), (48, 48, 14336), (513, 1030, 700),
    (260, 129, 4100), (1000, 33, 96), (4, 5001, 333)])
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_product(cuda, kind, M, N, K):
    _assert_product(kind, M, N, K, bias=(M + N) % 2 == 0)


def test_every_tile_of_the_product(cuda):
    # (which one a call takes follows from estimates: the sizes differ enough to reach all)
    found = set()
    for M, N, K in [(12, 3847, 4430), (70, 64, 1600), (6, 8582, 4829), (3, 200, 333), (30, 7279, 4722), (64, 4096, 1024),
                    (119, 4221, 4564), (35, 8676, 2697), (2040, 779, 4870), (500, 4096, 1000), (2503, 3137, 4914),
                    (2459, 3251, 4988), (1869, 8463, 3748), (4100, 4100, 1100), (1439, 8757, 4623), (2048, 14336, 4096)]:
        gen = torch.Generator(device="cuda").manual_seed(M + N)
        wide = -(-K // 16) * 16
        lhs = torch.randint(-127, 128, (M, wide), generator=gen, device="cuda", dtype=torch.int8)
        w = torch.randint(-127, 128, (N, K), generator=gen, device="cuda", dtype=torch.int8)
        s, t = (torch.rand(n, generator=gen, device="cuda") + 0.5 for n in (M, N))
        out = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
        iree_amd.matmul_w8a8(lhs, ref.pack(w.cpu()).cuda(), out, s, t, M, N, K, F.ROWS_TYPE_BF16)
        found.add(iree_amd.last_macro_tile()[:2])
        assert iree_amd.last_kernel_path() in ("w8a8:few-rows", "w8a8:mfma")
        ref.assert_near(out, *ref.product(lhs[:, :K], s, w, t))
    assert len(found) == 9, found


def test_product_without_a_sum(cuda):
    # K = 0: the bias, or zeros
    s, bias = torch.ones(40, device="cuda"), torch.arange(40.0, device="cuda")
    out = torch.full((3, 40), 7.0, device="cuda")
    lhs, w = torch.zeros(3, 16, dtype=torch.int8, device="cuda"), torch.zeros(2, 1, 32, 16, dtype=torch.int8, device="cuda")
    iree_amd.matmul_w8a8(lhs, w, out, s, s, 3, 40, 0, F.ROWS_TYPE_F32, bias=bias)
    assert torch.equal(out.cpu(), bias.cpu().expand(3, 40))
    iree_amd.matmul_w8a8(lhs, w, out, s, s, 3, 40, 0, F.ROWS_TYPE_F32)
    assert not out.any()


@pytest.mark.parametrize("M", [2, 40, 300])
def test_product_of_largest_values(cuda, M):
    # (the longest sum there is, of the largest products: 2^31 - 2^14)
    K, N = 131071, 32
    lhs = torch.full((M, 131072), -128, dtype=torch.int8, device="cuda")
    w = torch.full((1, 8192, 32, 16), -128, dtype=torch.int8, device="cuda")
    w[0, 8191, :, 15] = 0
    out = torch.zeros(M, N, device="cuda")
    one = torch.ones(max(M, N), device="cuda")
    iree_amd.matmul_w8a8(lhs, w, out, one, one, M, N, K, F.ROWS_TYPE_F32)
    assert (out == float(torch.tensor(131071.0 * 16384))).all()


def test_product_takes_strides_and_keeps_what_is_beside(cuda):
    gen, M, N, K = _gen(8), 37, 75, 90
    lhs, lhs_scale, w, w_scale = _product_case(gen, M, N, K)
    big = torch.full((M, 160), 101, dtype=torch.int8)
    big[:, 16:112] = lhs
    packed = ref.pack(w)
    spread = torch.full((3, 6 * 512 + 64), 33, dtype=torch.int8)
    spread[:, :6 * 512] = packed.view(3, -1)
    out = torch.full((M, 81), 5.0, dtype=torch.float16, device="cuda")
    iree_amd.matmul_w8a8(big.cuda().view(-1)[16:], spread.cuda(), out.view(-1)[3:], lhs_scale.cuda(), w_scale.cuda(), M, N, K,
                         F.ROWS_TYPE_F16, lhs_stride0=160, rhs_stride0=6 * 512 + 64, out_stride0=81)
    ref.assert_near(out.cpu()[:, 3:3 + N], *ref.product(lhs[:, :K], lhs_scale, w, w_scale))
    assert (out[:, :3] == 5).all() and (out[:, 3 + N:] == 5).all()


@pytest.mark.parametrize("M", [4, 300])
def test_a_row_whose_scale_is_nan_reads_as_nan(cuda, M):
    gen = _gen(9)
    lhs, lhs_scale, w, w_scale = _product_case(gen, M, 64, 64)
    lhs_scale[2] = math.nan
    out = torch.zeros(M, 64, device="cuda")
    iree_amd.matmul_w8a8(lhs.cuda(), ref.pack(w).cuda(), out, lhs_scale.cuda(), w_scale.cuda(), M, 64, 64, F.ROWS_TYPE_F32)
    nan = torch.isnan(out.cpu())
    assert nan[2].all() and nan.sum() == 64


def _route(logits, kind, top_k, renormalize, **how):
    tokens, experts = logits.shape
    ids = torch.full((tokens, top_k), 77, dtype=torch.int32, device="cuda")
    weights = torch.full((tokens, top_k), 77.0, device="cuda")
    offsets = torch.full((experts + 1,), 77, dtype=torch.int32, device="cuda")
    rows = torch.full((tokens * top_k,), 77, dtype=torch.int32, device="cuda")
    iree_amd.moe_route(logits.cuda(), ids, weights, offsets, rows, tokens, experts, top_k,
                       FLAGS[kind] | (F.ROUTE_RENORMALIZE if renormalize else 0), **how)
    return [t.cpu() for t in (ids, weights, offsets, rows)]


def _assert_route(got, logits, top_k, renormalize):
    ids, weights, offsets, rows = ref.route(logits, top_k, renormalize)
    assert torch.equal(got[0], ids)
    assert torch.equal(got[2], offsets) and torch.equal(got[3], rows)
    # Logits lie within 16 of the largest, or their weight below 2^-20: a difference rounded by 2^-24 of itself moves an
    # exponential by 2^-20, expf by 2^-23; sums of up to 512 terms in 8 + 6 additions by 14 2^-24, the division by 2^-23.
    off = (got[1].double() - weights).abs()
    assert (off <= 2.0**-18 * weights + 2.0**-30).all(), off.max()


@pytest.mark.parametrize("tokens", [1, 2, 63, 128, 129, 1000, 20000])
@pytest.mark.parametrize("experts,top_k", [(1, 1), (8, 2), (60, 4), (64, 8), (100, 64), (128, 8), (256, 8), (512, 10)])
def test_route(cuda, tokens, experts, top_k):
    if tokens * experts > 3000000:
        tokens = 3000
    kind, renormalize = ("f16", "bf16", "f32")[(tokens + experts) % 3], (tokens + top_k) % 2 == 0
    gen = _gen(tokens + experts)
    logits = (torch.randn(tokens, experts, generator=gen) * 2 + torch.randn(experts, generator=gen)).to(TYPES[kind])
    _assert_route(_route(logits, kind, top_k, renormalize), logits, top_k, renormalize)


@pytest.mark.parametrize("tokens", [7, 300])
def test_route_of_special_logits(cuda, tokens):
    gen, experts, top_k = _gen(tokens), 64, 8
    for renormalize in (False, True):
        logits = torch.randint(-3, 4, (tokens, experts), generator=gen).float()     # many are equal
        logits[0] = 0
        logits[1] = torch.where(torch.arange(experts) % 2 == 0, 0.0, -0.0)              # equal
        logits[2] = -math.inf                                                         # padding
        logits[3] = math.nan
        logits[4] = -math.inf
        logits[4, 9], logits[4, 5] = -1e30, 3                                         # two experts only
        logits[5, 60] = math.inf
        logits[6, 0:64:3] = math.nan
        for kind in ("f32", "bf16"):
            _assert_route(_route(logits.to(TYPES[kind]), kind, top_k, renormalize), logits.to(TYPES[kind]), top_k, renormalize)
    allpad = torch.full((tokens, experts), -math.inf)
    got = _route(allpad, "f32", top_k, True)
    assert (got[0] == -1).all() and not got[1].any() and not got[2].any() and (got[3] == -1).all()


def test_route_without_its_workspace_and_with_strides(cuda):
    gen, tokens, experts, top_k = _gen(11), 1111, 40, 3
    wide = torch.randn(tokens, 47, generator=gen)
    logits = wide[:, 5:45]
    tiny = torch.zeros(16, dtype=torch.uint8, device="cuda")
    want = ref.route(logits, top_k, True)
    for workspace in (None, tiny):
        got = _route(logits.contiguous(), "f32", top_k, True, workspace=workspace)
        assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3]) and torch.equal(got[2], want[2])
    on = wide.cuda()
    ids, weights = torch.zeros(tokens, top_k, dtype=torch.int32, device="cuda"), torch.zeros(tokens, top_k, device="cuda")
    offsets, rows = torch.zeros(41, dtype=torch.int32, device="cuda"), torch.zeros(tokens * top_k, dtype=torch.int32, device="cuda")
    iree_amd.moe_route(on.view(-1)[5:], ids, weights, offsets, rows, tokens, experts, top_k, F.ROWS_TYPE_F32, logits_stride0=47)
    assert torch.equal(ids.cpu(), want[0]) and torch.equal(rows.cpu(), want[3])


def test_route_of_nothing(cuda):
    offsets = torch.full((9,), 5, dtype=torch.int32, device="cuda")
    e = torch.empty(0, device="cuda")
    i = torch.empty(0, dtype=torch.int32, device="cuda")
    iree_amd.moe_route(e, i, e, offsets, i, 0, 8, 2, F.ROWS_TYPE_F32)
    assert not offsets.any()


def _grouped(kind, counts, N, K, top_k, gather, scatter, seed=0, tail=3, lhs_rows=None, spoil=()):
    """Groups of counts[e] positions, `tail` more behind them."""
    gen, experts = _gen(seed + sum(counts)), len(counts)
    positions = sum(counts) + tail
    slots = torch.randperm(positions, generator=gen).int()
    for p, row in spoil:
        slots[p] = row
    if lhs_rows is None:
        lhs_rows = -(-positions // top_k) if gather else positions
    lhs, lhs_scale, w, _ = _product_case(gen, lhs_rows, 1, K)
    w, w_scale = ref.rows8(gen, experts, N, K), ref.scales(gen, experts, N)
    offsets = torch.tensor([0] + counts).cumsum(0).int()
    out = torch.full((positions, N), 5.0, dtype=TYPES[kind], device="cuda")
    flags = FLAGS[kind] | (F.GROUPED_GATHER if gather else 0) | (F.GROUPED_SCATTER if scatter else 0)
    iree_amd.grouped_matmul_w8a8(lhs.cuda(), ref.pack(w).cuda(), out, lhs_scale.cuda(), w_scale.cuda(), offsets.cuda(), positions,
                                 experts, N, K, flags, lhs_rows=lhs_rows, rows=slots.cuda() if gather or scatter else None,
                                 rows_per_token=top_k)
    got = out.cpu()
    found = ref.grouped(lhs[:, :K], lhs_scale, w, w_scale, offsets, slots, gather, scatter, top_k, positions)
    written = torch.zeros(positions, dtype=torch.bool)
    if found:
        at = torch.tensor([t for t, _ in found])
        written[at] = True
        p = torch.stack([p for _, p in found])
        ref.assert_near(got[at], p, p)
    assert (got[~written] == 5).all()


@pytest.mark.parametrize("counts,N,K", [
    ([1], 32, 16), ([0, 3, 0, 0, 17, 1], 70, 100), ([16, 15, 33, 0], 33, 64), ([0] * 100 + [5] + [0] * 60 + [2], 64, 130),
    ([100, 1, 0, 90], 100, 200), ([300, 0, 257], 257, 520), ([1] * 70, 48, 1000), ([40] * 9, 96, 192), ([600, 5, 7, 0, 1], 130, 256)])
@pytest.mark.parametrize("how", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_grouped_product(cuda, kind, how, counts, N, K):
    _grouped(kind, counts, N, K, 3 if how[0] else 1, *how)


def test_grouped_product_leaves_out_rows_outside(cuda):
    spoil = [(0, -1), (4, 1 << 30), (17, 20), (21, -(1 << 31))]
    for how in ((True, False), (False, True), (True, True)):
        _grouped("f32", [3, 16, 0, 9], 40, 48, 1, *how, spoil=spoil, lhs_rows=11)
    _grouped("f32", [3, 16, 0, 9], 40, 48, 1, False, False, lhs_rows=11)


def test_grouped_product_uses_no_place_outside_its_list(cuda):
    gen = _gen(4)
    lhs, lhs_scale, w, _ = _product_case(gen, 20, 1, 32)
    w, w_scale = ref.rows8(gen, 3, 32, 32), ref.scales(gen, 3, 32)
    offsets = torch.tensor([-5, 4, 4, 90], dtype=torch.int32)
    out = torch.full((20, 32), 5.0, device="cuda")
    iree_amd.grouped_matmul_w8a8(lhs.cuda(), ref.pack(w).cuda(), out, lhs_scale.cuda(), w_scale.cuda(), offsets.cuda(), 20, 3, 32,
                                 32, F.ROWS_TYPE_F32, lhs_rows=20)
    clipped = torch.tensor([0, 4, 4, 20])
    found = ref.grouped(lhs, lhs_scale, w, w_scale, clipped, torch.arange(20), False, False, 1, 20)
    p = torch.stack([p for _, p in found])
    ref.assert_near(out.cpu(), p, p)


class Layer:
    """Norm, experts and their sum, every step on what the one before it left on the device."""

    def __init__(self, tokens, seed=0, dim=192, inner=80, experts=12, top_k=3, kind="bf16"):
        gen = _gen(seed)
        self.sizes = tokens, dim, inner, experts, top_k
        self.kind, self.flag = kind, FLAGS[kind]
        dtype, wide = TYPES[kind], -(-inner // 16) * 16
        self.x, self.residual = _rows(gen, kind, tokens, 1, dim).cuda(), _rows(gen, kind, tokens, dim).cuda()
        self.weight = (1 + torch.randn(dim, generator=gen) / 8).to(dtype).cuda()
        self.logits = torch.randn(tokens, experts, generator=gen).to(dtype)
        self.logits[tokens - tokens // 5:] = -math.inf
        self.logits = self.logits.cuda()
        self.up, self.up_scale = ref.rows8(gen, experts, 2 * inner, dim), ref.scales(gen, experts, 2 * inner)
        self.down, self.down_scale = ref.rows8(gen, experts, dim, inner), ref.scales(gen, experts, dim)
        self.on = [ref.pack(self.up).cuda(), self.up_scale.cuda(), ref.pack(self.down).cuda(), self.down_scale.cuda()]
        e, n = (lambda *s, dtype=dtype: torch.zeros(s, dtype=dtype, device="cuda")), tokens * top_k
        self.h, self.q, self.s = e(tokens, dim), e(tokens, dim, dtype=torch.int8), e(tokens, dtype=torch.float32)
        self.ids, self.w = e(tokens, top_k, dtype=torch.int32), e(tokens, top_k, dtype=torch.float32)
        self.offsets, self.rows = e(experts + 1, dtype=torch.int32), e(n, dtype=torch.int32)
        self.gate_up, self.q2, self.s2 = e(n, 2 * inner), e(n, wide, dtype=torch.int8), e(n, dtype=torch.float32)
        self.slots = torch.full((n, dim), math.nan, dtype=dtype, device="cuda")
        self.h3, self.q3, self.s3 = e(tokens, dim), e(tokens, dim, dtype=torch.int8), e(tokens, dtype=torch.float32)
        nbytes = iree_amd.moe_route_workspace(tokens, experts)
        self.workspace = torch.zeros(max(nbytes, 16), dtype=torch.uint8, device="cuda")

    def run(self):
        tokens, dim, inner, experts, top_k = self.sizes
        n, up, up_scale, down, down_scale = tokens * top_k, *self.on
        iree_amd.rms_norm_quantize(self.x, self.q, self.s, tokens, dim, self.flag, weight=self.weight, residual=self.residual,
                                   sum_out=self.h)
        iree_amd.moe_route(self.logits, self.ids, self.w, self.offsets, self.rows, tokens, experts, top_k,
                           self.flag | F.ROUTE_RENORMALIZE, workspace=self.workspace)
        iree_amd.grouped_matmul_w8a8(self.q, up, self.gate_up, self.s, up_scale, self.offsets, n, experts, 2 * inner, dim,
                                     self.flag | F.GROUPED_GATHER, lhs_rows=tokens, rows=self.rows, rows_per_token=top_k)
        iree_amd.quantize_rows(self.gate_up, self.q2, self.s2, n, inner, self.flag, up=self.gate_up[:, inner:],
                               x_stride0=2 * inner, up_stride0=2 * inner, q_stride0=self.q2.shape[1])
        iree_amd.grouped_matmul_w8a8(self.q2, down, self.slots, self.s2, down_scale, self.offsets, n, experts, dim, inner,
                                     self.flag | F.GROUPED_SCATTER, lhs_rows=n, rows=self.rows)
        iree_amd.rms_norm_quantize(self.slots, self.q3, self.s3, tokens, dim, self.flag, weight=self.weight, residual=self.h,
                                   sum_out=self.h3, addends=top_k, addend_weights=self.w)

    def results(self):
        return [t.clone() for t in (self.h, self.q, self.ids, self.w, self.offsets, self.rows, self.h3, self.q3, self.s3)]


@pytest.mark.parametrize("tokens", [1, 9, 150, 700])
def test_a_layer_with_experts(cuda, tokens):
    layer = Layer(tokens, seed=tokens)
    layer.run()
    _, dim, inner, experts, top_k = layer.sizes
    h, q, s, ids, w, offsets, rows, gate_up, q2, s2, slots, h3, q3, s3 = (getattr(layer, n).cpu() for n in (
        "h q s ids w offsets rows gate_up q2 s2 slots h3 q3 s3").split())
    _assert_norm((h, q, s), layer.x.cpu(), layer.residual.cpu(), layer.weight.cpu(), None, 1e-6)
    _assert_route((ids, w, offsets, rows), layer.logits.cpu(), top_k, True)
    found = ref.grouped(q, s, layer.up, layer.up_scale, offsets, rows, True, False, top_k, tokens * top_k)
    used = len(found)
    assert used == (tokens - tokens // 5) * top_k
    p = torch.stack([v for _, v in found])
    ref.assert_near(gate_up[:used], p, p)
    _assert_rows((q2[:used, :inner], s2[:used]), gate_up[:used, :inner], gate_up[:used, inner:])
    found = ref.grouped(q2[:, :inner], s2, layer.down, layer.down_scale, offsets, rows, False, True, 1, tokens * top_k)
    at, p = torch.tensor([t for t, _ in found]), torch.stack([v for _, v in found])
    ref.assert_near(slots[at], p, p)
    _assert_norm((h3, q3, s3), slots.view(tokens, top_k, dim), h, layer.weight.cpu(), w, 1e-6)


def test_two_captured_layers_on_two_streams(cuda):
    layers = [Layer(40, seed=1), Layer(300, seed=2)]
    eager = []
    for layer in layers:
        layer.run()
        eager.append(layer.results())
    streams, graphs = [torch.cuda.Stream() for _ in layers], []
    torch.cuda.synchronize()
    for layer, stream in zip(layers, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer.run()
        graphs.append(graph)
    for _ in range(4):
        for layer in layers:
            for t in (layer.h, layer.q, layer.rows, layer.h3, layer.q3):
                t.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for layer, want in zip(layers, eager):
            assert all(torch.equal(a, b) for a, b in zip(layer.results(), want))
        layers[0].run()                      # the program's own work in between
        assert all(torch.equal(a, b) for a, b in zip(layers[0].results(), eager[0]))


def _far_rows(rows, stride, K, at):
    """An otherwise empty matrix of 8 bits with rows at `at`, and those rows."""
    lhs = torch.zeros(rows, stride, dtype=torch.int8, device="cuda")
    mine = ref.rows8(_gen(rows), len(at), K)
    lhs[torch.tensor(at, device="cuda"), :K] = mine.cuda()
    return lhs, mine


@pytest.mark.parametrize("tokens", [24, 500])
def test_rows_gathered_from_almost_4_gib(cuda, tokens):
    rows, stride, K, N = 1044000, 4112, 80, 48                 # 4.293e9 bytes
    at = [0, 522300, rows - 1, rows - 2, 5]
    lhs, mine = _far_rows(rows, stride, K, at)
    gen = _gen(1)
    w, w_scale = ref.rows8(gen, 2, N, K), ref.scales(gen, 2, N)
    scale = torch.ones(rows, device="cuda")
    which = torch.arange(tokens) % len(at)
    half = tokens // 3
    out = torch.zeros(tokens, N, device="cuda")
    iree_amd.grouped_matmul_w8a8(lhs, ref.pack(w).cuda(), out, scale, w_scale.cuda(),
                                 torch.tensor([0, half, tokens], dtype=torch.int32).cuda(), tokens, 2, N, K,
                                 F.ROWS_TYPE_F32 | F.GROUPED_GATHER, lhs_rows=rows,
                                 rows=torch.tensor(at, dtype=torch.int32)[which].cuda(), lhs_stride0=stride)
    for e, part in ((0, slice(0, half)), (1, slice(half, tokens))):
        p, _ = ref.product(mine[which[part]], torch.ones(len(which[part])), w[e], w_scale[e])
        ref.assert_near(out[part].cpu(), p, p)


def test_a_matrix_of_more_than_4_gib(cuda):
    rows, stride, K, N = 2200000, 2064, 40, 32                 # 4.5e9 bytes
    at = [0, 1, 1099999, rows - 1]
    lhs, mine = _far_rows(rows, stride, K, at)
    gen = _gen(2)
    w, w_scale = ref.rows8(gen, N, K), ref.scales(gen, N)
    out = torch.full((rows, N), 3.0, dtype=torch.float16, device="cuda")
    iree_amd.matmul_w8a8(lhs, ref.pack(w).cuda(), out, torch.ones(rows, device="cuda"), w_scale.cuda(), rows, N, K,
                         F.ROWS_TYPE_F16, lhs_stride0=stride)
    ref.assert_near(out[torch.tensor(at, device="cuda")].cpu(), *ref.product(mine, torch.ones(4), w, w_scale))
    out[torch.tensor(at, device="cuda")] = 0
    assert not out.any()


@pytest.mark.parametrize("tokens", [3, 400])
def test_weights_of_more_than_4_gib(cuda, tokens):
    experts, N, K = 512, 4096, 2304                            # 4.8e9 bytes
    packed = torch.zeros(experts, N // 32, K // 16, 32, 16, dtype=torch.int8, device="cuda")
    gen = _gen(3)
    w, w_scale = ref.rows8(gen, N, K), ref.scales(gen, N)
    packed[experts - 1] = ref.pack(w).cuda()
    scale = torch.zeros(experts, N, device="cuda")
    scale[experts - 1] = w_scale.cuda()
    lhs, lhs_scale = ref.rows8(gen, tokens, K), ref.scales(gen, tokens)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    offsets[experts] = tokens
    out = torch.zeros(tokens, N, device="cuda")
    iree_amd.grouped_matmul_w8a8(lhs.cuda(), packed, out, lhs_scale.cuda(), scale, offsets, tokens, experts, N, K,
                                 F.ROWS_TYPE_F32, lhs_rows=tokens)
    p, _ = ref.product(lhs, lhs_scale, w, w_scale)
    ref.assert_near(out.cpu(), p, p)


def test_a_call_on_another_stream(cuda):
    gen, M, N, K = _gen(6), 70, 96, 200
    lhs, lhs_scale, w, w_scale = _product_case(gen, M, N, K)
    args = [t.cuda() for t in (lhs, ref.pack(w), lhs_scale, w_scale)]
    out = torch.zeros(M, N, device="cuda")
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    iree_amd.matmul_w8a8(args[0], args[1], out, args[2], args[3], M, N, K, F.ROWS_TYPE_F32, stream=stream)
    logits = torch.randn(500, 64, generator=gen)
    on = logits.cuda()
    ids, weights = torch.zeros(500, 4, dtype=torch.int32, device="cuda"), torch.zeros(500, 4, device="cuda")
    offsets, rows = torch.zeros(65, dtype=torch.int32, device="cuda"), torch.zeros(2000, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    iree_amd.moe_route(on, ids, weights, offsets, rows, 500, 64, 4, F.ROWS_TYPE_F32, stream=stream)
    stream.synchronize()
    ref.assert_near(out.cpu(), *ref.product(lhs[:, :K], lhs_scale, w, w_scale))
    _assert_route([t.cpu() for t in (ids, weights, offsets, rows)], logits, 4, False)


@pytest.mark.parametrize("M,N,K", [(5, 70, 100), (300, 513, 640), (1, 1000, 2048)])
def test_product_on_what_pack_makes_and_beside_the_integer_one(cuda, M, N, K):
    gen = _gen(M)
    lhs, w = ref.rows8(gen, M, K) // 8, ref.rows8(gen, N, K)
    high, wide = -(-N // 32), -(-K // 16)
    packed = torch.full((high, wide, 32, 16), 7, dtype=torch.int8, device="cuda")
    iree_amd.pack(w.cuda(), packed, N, K, high, wide, 32, 16, 0, F.PACK_TYPE_I8I8)
    assert torch.equal(packed.cpu(), ref.pack(w))
    rows = torch.zeros(M, wide * 16, dtype=torch.int8)
    rows[:, :K] = lhs
    one = torch.ones(max(M, N), device="cuda")
    out = torch.zeros(M, N, device="cuda")
    iree_amd.matmul_w8a8(rows.cuda(), packed, out, one, one, M, N, K, F.ROWS_TYPE_F32)
    whole = torch.zeros(M, high * 32, dtype=torch.int32, device="cuda")
    iree_amd.matmul_data_tiled(lhs.cuda(), w.T.contiguous().cuda(), whole.view(-1)[:M * N], M, N, K, F.MMT4D_TYPE_S8S8S32)
    assert torch.equal(out, whole.view(-1)[:M * N].view(M, N).float())        # (sums below 2^24)


@pytest.mark.parametrize("counts", [[3, 0, 17], [200, 90, 0]])
def test_grouped_product_takes_strides(cuda, counts):
    gen, N, K, positions = _gen(12), 70, 100, sum(counts)
    lhs, lhs_scale, w, _ = _product_case(gen, positions, 1, K)
    w, w_scale = ref.rows8(gen, 3, N, K), ref.scales(gen, 3, N)
    big = torch.full((positions, 144), 99, dtype=torch.int8)
    big[:, 16:128] = lhs
    spread = torch.full((3, 4 * 3648), 55, dtype=torch.int8)               # outer columns 3648 bytes apart, four's room
    packed = ref.pack(w).view(3, 3, 3584)
    for c in range(3):
        spread[:, c * 3648:c * 3648 + 3584] = packed[:, c]
    offsets = torch.tensor([0] + counts).cumsum(0).int()
    out = torch.full((positions, 75), 5.0, dtype=torch.bfloat16, device="cuda")
    iree_amd.grouped_matmul_w8a8(big.cuda().view(-1)[16:], spread.cuda(), out.view(-1)[2:], lhs_scale.cuda(), w_scale.cuda(),
                                 offsets.cuda(), positions, 3, N, K, F.ROWS_TYPE_BF16, lhs_rows=positions, lhs_stride0=144,
                                 rhs_stride0=3648, rhs_expert_stride=4 * 3648, out_stride0=75)
    p = torch.stack([v for _, v in ref.grouped(lhs[:, :K], lhs_scale, w, w_scale, offsets, torch.arange(positions), False,
                                               False, 1, positions)])
    ref.assert_near(out.cpu()[:, 2:72], p, p)
    assert (out[:, :2] == 5).all() and (out[:, 72:] == 5).all()


@pytest.mark.parametrize("cols", [24, 100, 128, 600, 1030])
def test_many_short_rows(cuda, cols):
    # (more rows than there are workgroups: each takes several in turn)
    gen, rows = _gen(cols), 70001 if cols < 200 else 20001
    x, up = _rows(gen, "bf16", rows, cols), _rows(gen, "bf16", rows, cols)
    x[17] = 0
    x[rows - 1, 3] = math.nan
    x[rows - 3] = 1e35
    x[rows // 2] = -500
    _assert_rows(_quantize(x, None, "bf16"), x, None)
    _assert_rows(_quantize(x, up, "bf16"), x, up)
    _assert_norm(_norm(x[:, None], "bf16", up, up[0]), x[:, None], up, up[0], None)
    both = torch.stack((x, up), 1)
    _assert_norm(_norm(both, "bf16"), both, None, None, None)
