"""The layer in 8-bit integers on the device where its definitions are easily missed: roundings, sizes
of values at the ends of f32, sizes of tensors next to the limits."""
import math

import pytest
import torch

import iree_amd
import w8a8ref as ref

pytestmark = pytest.mark.gpu
TYPES, FLAGS = ref.TYPES, ref.FLAGS


@pytest.mark.parametrize("kind,half", [("f16", 2.0**-11), ("bf16", 2.0**-8)])
def test_a_sum_of_several_addends_is_rounded_to_f32_and_then_to_its_type(cuda, kind, half):
    # 1, half a step of the type, and what f32 does not hold next to them (even, so down), or does (up)
    weights = torch.tensor([[1, half, 2.0**-30], [1, half, 2.0**-23], [1, half, -(2.0**-30)], [1, 3 * half, -(2.0**-30)]])
    want = torch.tensor([1.0, 1 + 2 * half, 1.0, 1 + 4 * half]).to(TYPES[kind])
    tokens, dim = weights.shape[0], 72
    x = torch.ones(tokens, 3, dim, dtype=TYPES[kind], device="cuda")
    out = torch.zeros(tokens, dim, dtype=TYPES[kind], device="cuda")
    q, scale = torch.zeros(tokens, dim, dtype=torch.int8, device="cuda"), torch.zeros(tokens, device="cuda")
    iree_amd.rms_norm_quantize(x, q, scale, tokens, dim, FLAGS[kind], sum_out=out, addends=3, addend_weights=weights.cuda())
    assert torch.equal(out.cpu(), want[:, None].expand(tokens, dim))


def _normed(h, weight, eps):
    """(q, scale f64) of the normed rows: of their products with the weight in f32, which 64 bits hold from there on."""
    t = (h.float() if weight is None else h.float() * weight.float()).double()
    top = t.abs().amax(-1)
    fine = top <= torch.finfo(torch.float32).max
    q = torch.where((fine & (top > 0))[:, None], torch.round(t * 127 / torch.where(top > 0, top, 1.0)[:, None]), 0.0)
    scale = torch.where(top == 0, 0.0, top / torch.sqrt(h.double().square().mean(-1) + eps) / 127)
    return q.nan_to_num(0.0).to(torch.int8), torch.where(fine, scale, math.nan)


def _assert_normed(x, weight, eps, addends=1, keep=True):
    """Of rows x [tokens][dim], which are the sums."""
    tokens, dim = x.shape
    given = x if addends == 1 else torch.stack([x] + [torch.zeros_like(x)] * (addends - 1), 1)
    q, scale = torch.full((tokens, dim), 99, dtype=torch.int8, device="cuda"), torch.full((tokens,), -1.0, device="cuda")
    out = torch.zeros_like(x).cuda() if keep else None
    iree_amd.rms_norm_quantize(given.cuda(), q, scale, tokens, dim, FLAGS["bf16"], weight=weight.cuda(), eps=eps, sum_out=out,
                               addends=addends)
    want_q, want = _normed(x, weight, eps)
    if keep:
        assert torch.equal(out.cpu().nan_to_num(7), x.nan_to_num(7))
    q, scale = q.cpu(), scale.cpu()
    assert torch.equal(q, want_q), (q != want_q).any(-1).nonzero()
    assert torch.equal(torch.isnan(scale), torch.isnan(want)), scale
    # 64 bits, rounded once to 32: by 2^-24 of it, below 2^-126 by 2^-150, from 2^128 - 2^103 on to infinity
    beyond = want >= 2.0**128 - 2.0**103
    assert torch.isinf(scale[beyond]).all()
    off = torch.where(beyond, 0.0, scale.double() - want).abs().nan_to_num(0)
    assert (off <= 1.001 * 2.0**-24 * want.nan_to_num(0) + 1.001 * 2.0**-150).all()


@pytest.mark.parametrize("dim", [40, 600, 1000, 4096, 8000, 16384, 30000, 65536])
def test_norms_of_products_at_the_ends_of_f32(cuda, dim):
    gen = torch.Generator().manual_seed(dim)
    x = torch.randn(11, dim, generator=gen)
    x[0] *= 1e30
    x[1] *= 1e-25
    x[2] = 0
    x[2, 7] = 1e-4                            # one value: the norm makes it sqrt(dim)
    x[3, 5] = math.inf
    x[4] *= 1e37
    x[5] = 0
    x[6] *= 1e-38                             # (subnormal ones among them)
    x[7, dim - 1] = math.nan
    x[8] = torch.randint(-127, 128, (dim,), generator=gen) * 2.0**90      # halves between two codes
    x[8, 0] = 127 * 2.0**91
    x = x.bfloat16()
    for size in (1.0, 1e10, 1e-20, 2e38, 1e-30):
        weight = (size * (1 + torch.rand(dim, generator=gen) / 2)).bfloat16()
        if size == 1e10:
            weight = (2.0**31 * torch.ones(dim)).bfloat16()               # (keeps the halves of row 8)
        _assert_normed(x, weight, 0.0)
        _assert_normed(x, weight, 1e-6, keep=False)
        _assert_normed(x, weight, 0.0, addends=2, keep=False)
    _assert_normed(x, torch.zeros(dim).bfloat16(), 1e-6)
    weight = torch.ones(dim).bfloat16()
    weight[3] = math.inf
    _assert_normed(x, weight, 1e-6)


def test_a_list_whose_small_tiles_no_grid_holds(cuda):
    # (few channels and a long sum: the estimate alone takes 16 x 16, of which there can be 2^23 and more)
    positions, N, K, experts = 143191276, 1, 8646, 8
    gen = torch.Generator().manual_seed(1)
    lhs, wide = ref.rows8(gen, 5, K), -(-K // 16) * 16
    rows8 = torch.zeros(5, wide, dtype=torch.int8)
    rows8[:, :K] = lhs
    w, w_scale, lhs_scale = ref.rows8(gen, experts, N, K), ref.scales(gen, experts, N), ref.scales(gen, 5)
    offsets = torch.tensor([0, 3, 3, 40, 41, 41, 90, 100, 150], dtype=torch.int32)
    rows = torch.zeros(positions, dtype=torch.int32, device="cuda")
    mine = torch.randint(-1, 6, (150,), generator=gen).int()                 # (some outside)
    rows[:150] = mine.cuda()
    out = torch.full((positions, N), 5.0, dtype=torch.float16, device="cuda")
    iree_amd.grouped_matmul_w8a8(rows8.cuda(), ref.pack(w).cuda(), out, lhs_scale.cuda(), w_scale.cuda(), offsets.cuda(),
                                 positions, experts, N, K, FLAGS["f16"] | iree_amd.flags.GROUPED_GATHER, lhs_rows=5, rows=rows)
    found = ref.grouped(lhs, lhs_scale, w, w_scale, offsets, mine, True, False, 1, 150)
    at, p = torch.tensor([t for t, _ in found]), torch.stack([p for _, p in found])
    got = out[:200].cpu()
    ref.assert_near(got[at], p, p)
    got[at] = 5
    assert (got == 5).all() and (out[200:] == 5).all()


@pytest.mark.parametrize("used", [30, 900])
@pytest.mark.parametrize("how", [0, iree_amd.flags.GROUPED_GATHER, iree_amd.flags.GROUPED_SCATTER])
def test_grouped_products_without_a_sum_are_zeros(cuda, how, used):
    positions, N, experts = used + 20, 70, 3
    offsets = torch.tensor([0, used // 3, used // 3, used], dtype=torch.int32, device="cuda")
    rows = torch.arange(positions, dtype=torch.int32, device="cuda")
    lhs = torch.full((positions, 16), 3, dtype=torch.int8, device="cuda")
    w = torch.full((experts, 3, 1, 32, 16), 3, dtype=torch.int8, device="cuda")
    one, out = torch.ones(positions, device="cuda"), torch.full((positions, N), 5.0, device="cuda")
    iree_amd.grouped_matmul_w8a8(lhs, w, out, one, torch.ones(experts, N, device="cuda"), offsets, positions, experts, N, 0,
                                 FLAGS["f32"] | how, lhs_rows=positions, rows=rows if how else None)
    assert not out[:used].any() and (out[used:] == 5).all()


def test_routing_of_many_tokens_with_no_workspace_at_all(cuda):
    # (the Python function takes one by itself)
    gen, tokens, experts, top_k = torch.Generator().manual_seed(7), 900, 24, 3
    logits = torch.randn(tokens, experts, generator=gen)
    want = ref.route(logits, top_k, True)
    on = logits.cuda()
    ids, weights = torch.zeros(tokens, top_k, dtype=torch.int32, device="cuda"), torch.zeros(tokens, top_k, device="cuda")
    offsets, rows = torch.zeros(experts + 1, dtype=torch.int32, device="cuda"), torch.zeros(tokens * top_k, dtype=torch.int32, device="cuda")
    lib, flags = iree_amd.load_library(), FLAGS["f32"] | iree_amd.flags.ROUTE_RENORMALIZE
    call = lambda workspace, nbytes: lib.iree_amd_uk_moe_route(  # noqa: E731
        on.data_ptr(), experts, ids.data_ptr(), weights.data_ptr(), offsets.data_ptr(), rows.data_ptr(), tokens, experts, top_k,
        workspace, nbytes, flags, torch.cuda.current_stream().cuda_stream)
    assert call(None, iree_amd.moe_route_workspace(tokens, experts)) == 3
    assert not ids.any() and not rows.any()
    assert call(None, 0) == 0
    assert torch.equal(ids.cpu(), want[0]) and torch.equal(offsets.cpu(), want[2]) and torch.equal(rows.cpu(), want[3])


def test_rows_gathered_from_the_last_bytes_below_4_gib(cuda):
    # 2113665 x 2032 bytes are 2^32 - 16
    rows, K, N, tokens = 2113665, 2030, 40, 700
    gen = torch.Generator().manual_seed(3)
    at = torch.tensor([0, rows - 1, 1056832, rows - 2])
    mine = ref.rows8(gen, 4, K)
    lhs = torch.zeros(rows, 2032, dtype=torch.int8, device="cuda")
    lhs[at.cuda(), :K] = mine.cuda()
    w, w_scale, scale = ref.rows8(gen, 2, N, K), ref.scales(gen, 2, N), torch.ones(rows, device="cuda")
    for count in (8, tokens):
        which = torch.arange(count) % 4
        out = torch.zeros(count, N, device="cuda")
        iree_amd.grouped_matmul_w8a8(lhs, ref.pack(w).cuda(), out, scale, w_scale.cuda(),
                                     torch.tensor([0, count // 2, count], dtype=torch.int32).cuda(), count, 2, N, K,
                                     FLAGS["f32"] | iree_amd.flags.GROUPED_GATHER, lhs_rows=rows, rows=at[which].int().cuda())
        for e, part in ((0, slice(0, count // 2)), (1, slice(count // 2, count))):
            p, _ = ref.product(mine[which[part]], torch.ones(len(which[part])), w[e], w_scale[e])
            ref.assert_near(out[part].cpu(), p, p)


@pytest.mark.parametrize("M,N,K,path", [(3, 70, 100, "w8a8:few-rows"), (5534, 71, 36, "w8a8:mfma")])
def test_products_round_the_sum_times_the_row_scale_to_f32(cuda, M, N, K, path):
    gen = torch.Generator().manual_seed(M)
    lhs, wide = ref.rows8(gen, M, K), -(-K // 16) * 16
    rows8 = torch.zeros(M, wide, dtype=torch.int8)
    rows8[:, :K] = lhs
    w = ref.rows8(gen, N, K)
    w[3] = 0                                  # (sums of 0)
    lhs_scale, w_scale = ref.scales(gen, M) * 1e38, ref.scales(gen, N) * 1e-30
    lhs_scale[1::3] = 2.0**-140               # (subnormal: the products with whole numbers are exact)
    w_scale[::7], w_scale[2] = 1e5, 0
    out = torch.zeros(M, N, device="cuda")
    iree_amd.matmul_w8a8(rows8.cuda(), ref.pack(w).cuda(), out, lhs_scale.cuda(), w_scale.cuda(), M, N, K, FLAGS["f32"])
    assert iree_amd.last_kernel_path() == path
    first = ((lhs.double() @ w.double().T).float() * lhs_scale[:, None]).double()
    want = (first * w_scale.double()).float()              # (64 bits hold the product: rounded once)
    assert torch.isinf(want).any() and torch.isnan(want).any() and (want == 0).any()
    assert torch.equal(out.cpu().nan_to_num(7), want.nan_to_num(7)) and torch.equal(torch.isnan(out.cpu()), torch.isnan(want))


@pytest.mark.parametrize("tokens,experts,top_k,whole", [(6001, 40, 4, False), (600001, 16, 4, True), (150000, 300, 64, True)])
def test_routing_of_more_slots_than_a_workgroup_holds(cuda, tokens, experts, top_k, whole):
    # (above 8192 slots a workgroup reads its choices back from memory: with a workspace from 4 or more such blocks, or in one)
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    logits = torch.randn(tokens, experts, generator=gen, device="cuda") + torch.randn(experts, generator=gen, device="cuda")
    logits[5] = -math.inf
    logits[tokens - 3, 3:] = math.nan
    ids, weights = torch.zeros(tokens, top_k, dtype=torch.int32, device="cuda"), torch.zeros(tokens, top_k, device="cuda")
    offsets, rows = torch.zeros(experts + 1, dtype=torch.int32, device="cuda"), torch.zeros(tokens * top_k, dtype=torch.int32, device="cuda")
    iree_amd.moe_route(logits, ids, weights, offsets, rows, tokens, experts, top_k, FLAGS["f32"] | iree_amd.flags.ROUTE_RENORMALIZE,
                       workspace=None if whole else torch.zeros(16, dtype=torch.uint8, device="cuda"))
    values, want = torch.sort(logits.nan_to_num(nan=-math.inf, neginf=-math.inf), dim=-1, descending=True, stable=True)
    want = torch.where(values[:, :top_k] > -math.inf, want[:, :top_k], -1)
    assert torch.equal(ids.long(), want)
    slots = torch.where(want < 0, experts, want).flatten()
    counts = torch.bincount(slots, minlength=experts + 1)
    assert torch.equal(offsets[1:].long(), counts[:experts].cumsum(0)) and offsets[0] == 0
    order = torch.sort(slots, stable=True).indices
    order[int(offsets[-1]):] = -1
    assert torch.equal(rows.long(), order)
    p = torch.exp(values[:, :top_k].double() - values[:, :1].double().clamp(min=-1e300)) * (want >= 0)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    # (differences of logits of at most 16 rounded by 2^-24 of themselves, expf and the division by 2^-23 each, six additions)
    assert ((weights.double() - p).abs() <= 2.0**-18 * p + 2.0**-30).all()


def test_products_captured_before_they_ever_ran(cuda):
    gen = torch.Generator(device="cuda").manual_seed(4)
    sizes = [(21, 65, 2055), (33, 1625, 3009), (30, 1473, 33), (8172, 71, 523), (6717, 67, 460), (6694, 989, 451), (8521, 262, 1186),
             (8925, 444, 1487), (1681, 8719, 5452)]                          # (a tile each)
    cases, tiles = [], set()
    for M, N, K in sizes:
        wide, high = -(-K // 16), -(-N // 32)
        lhs = torch.randint(-127, 128, (M, wide * 16), generator=gen, device="cuda", dtype=torch.int8)
        w = torch.randint(-127, 128, (high, wide, 32, 16), generator=gen, device="cuda", dtype=torch.int8)
        s, t = (torch.rand(n, generator=gen, device="cuda") + 0.5 for n in (M, N))
        cases.append((lhs, w, torch.zeros(M, N, dtype=torch.bfloat16, device="cuda"), s, t, M, N, K, FLAGS["bf16"]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for case in cases:
            iree_amd.matmul_w8a8(*case)
            tiles.add(iree_amd.last_macro_tile()[:2])
    assert len(tiles) == 9
    want = None
    for _ in range(4):
        for case in cases:
            case[2].zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [case[2].clone() for case in cases]
        for case in cases:                    # the program's own work in between
            case[2].zero_()
            iree_amd.matmul_w8a8(*case)
        want = [case[2].clone() for case in cases] if want is None else want
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(case[2], b) and b.abs().sum() > 0 for case, b in zip(cases, want))


def test_rows_of_more_than_4_gib(cuda):
    rows, cols = 70001, 32760
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")        # 4.59e9 bytes
    at = torch.tensor([0, 1, 35000, rows - 2, rows - 1], device="cuda")
    mine = (torch.randn(5, cols, generator=torch.Generator().manual_seed(1)) * 2).bfloat16()
    x[at] = mine.cuda()
    q, scale = torch.full((rows, cols), 9, dtype=torch.int8, device="cuda"), torch.full((rows,), -1.0, device="cuda")
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[at] = False

    def check(want, want_scale):
        assert torch.equal(q[at].cpu(), want)
        assert ((scale[at].cpu().double() - want_scale).abs() <= 1.001 * 2.0**-24 * want_scale).all()
        assert not scale[rest].any()
        q[at] = 0
        assert not q.any()
        q.fill_(9)

    iree_amd.quantize_rows(x, q, scale, rows, cols, FLAGS["bf16"])
    check(*ref.codes(mine.double()))
    iree_amd.quantize_rows(x, q, scale, rows, cols, FLAGS["bf16"], up=x)
    check(*ref.codes(ref.silu_mul(mine, mine)))
    iree_amd.rms_norm_quantize(x, q, scale, rows, cols, FLAGS["bf16"], eps=2.0**-20, sum_out=x)
    check(*ref.norm(mine, None, 2.0**-20))
    assert torch.equal(x[at].cpu(), mine)
