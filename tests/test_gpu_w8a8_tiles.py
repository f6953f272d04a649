"""The products in 8-bit integers on every tile, for one matrix and by expert, with remainders in all sizes, against
the exact product in 64 bits on the device. Which tile a call takes follows from estimates: every case says which one it
is for and checks that."""
import functools

import pytest
import torch

import iree_amd
import w8a8ref as ref
from iree_amd import flags as F

pytestmark = pytest.mark.gpu
TYPES, FLAGS = ref.TYPES, ref.FLAGS
FEW = ((16, 16), (16, 32), (32, 32), (64, 64))


def _pack(w):
    """[..., N, K] on the device in tiles [..., N / 32][K / 16][32][16], zeros past N and K."""
    n, k = w.shape[-2:]
    high, wide = -(-n // 32) * 32, -(-k // 16) * 16
    full = torch.zeros(*w.shape[:-2], high, wide, dtype=torch.int8, device="cuda")
    full[..., :n, :k] = w
    return full.view(*w.shape[:-2], high // 32, 32, wide // 16, 16).transpose(-3, -2).contiguous()


def _rows(gen, rows, K):
    """Rows of 8 bits, whole 16s long: what lies past K does not count."""
    return torch.randint(-127, 128, (rows, -(-K // 16) * 16), generator=gen, device="cuda", dtype=torch.int8)


def _scales(gen, *shape):
    return (torch.rand(shape, generator=gen, device="cuda") + 0.5) / 64


def _assert_tile(tile):
    assert iree_amd.last_macro_tile()[:2] == tile
    assert iree_amd.last_kernel_path() == ("w8a8:few-rows" if tile in FEW else "w8a8:mfma")


# Macro tiles once with fewer steps of K than their rings have slots, once with more.
DENSE = [((16, 16), 21, 65, 2055), ((16, 32), 33, 1625, 3009), ((32, 32), 30, 1473, 33), ((64, 64), 8172, 71, 523),
         ((64, 128), 5735, 65, 35), ((64, 128), 6717, 67, 460), ((64, 256), 6923, 740, 34), ((64, 256), 6694, 989, 451),
         ((128, 128), 11101, 521, 81), ((128, 128), 8521, 262, 1186), ((128, 256), 8925, 444, 1487),
         ((256, 256), 1681, 8719, 5452)]


@functools.lru_cache(maxsize=1)
def _dense(M, N, K):
    gen = torch.Generator(device="cuda").manual_seed(M)
    lhs, w = _rows(gen, M, K), torch.randint(-127, 128, (N, K), generator=gen, device="cuda", dtype=torch.int8)
    lhs_scale, w_scale = _scales(gen, M), _scales(gen, N)
    exact = (lhs[:, :K].double() @ w.double().T.contiguous()) * lhs_scale.double()[:, None] * w_scale.double()
    return lhs, _pack(w), lhs_scale, w_scale, torch.randn(N, generator=gen, device="cuda"), exact


@pytest.mark.parametrize("tile,M,N,K", DENSE)
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_the_product_on_every_tile(cuda, kind, tile, M, N, K):
    lhs, packed, lhs_scale, w_scale, bias, exact = _dense(M, N, K)
    for add in (None, bias):
        out = torch.full((M, N + 3), 5.0, dtype=TYPES[kind], device="cuda")
        iree_amd.matmul_w8a8(lhs, packed, out, lhs_scale, w_scale, M, N, K, FLAGS[kind], bias=add, out_stride0=N + 3)
        _assert_tile(tile)
        ref.assert_near(out[:, :N], exact, exact if add is None else exact + add.double())
        assert (out[:, N:] == 5).all()


@pytest.mark.parametrize("tile,M,N,K", [c for c in DENSE if c[3] > 100])
def test_a_row_whose_scale_is_nan_reads_as_nan_on_every_tile(cuda, tile, M, N, K):
    lhs, packed, lhs_scale, w_scale, _, _ = _dense(M, N, K)
    spoiled = lhs_scale.clone()
    spoiled[M // 2] = float("nan")
    out = torch.zeros(M, N, device="cuda")
    iree_amd.matmul_w8a8(lhs, packed, out, spoiled, w_scale, M, N, K, F.ROWS_TYPE_F32)
    _assert_tile(tile)
    nan = torch.isnan(out)
    assert nan[M // 2].all() and nan.sum() == N


@pytest.mark.parametrize("tile,M,N", [((16, 16), 2, 32), ((64, 64), 200, 2000), ((64, 128), 600, 3000), ((128, 128), 600, 6000),
                                      ((128, 256), 1500, 4000), ((256, 256), 1500, 6000)])
def test_the_largest_sums(cuda, tile, M, N):
    # (131071 products of -128 and -128: 2^31 - 2^14)
    K = 131071
    lhs = torch.full((M, 131072), -128, dtype=torch.int8, device="cuda")
    w = torch.full((-(-N // 32), 8192, 32, 16), -128, dtype=torch.int8, device="cuda")
    w[:, 8191, :, 15] = 0
    out = torch.zeros(M, N, device="cuda")
    one = torch.ones(max(M, N), device="cuda")
    iree_amd.matmul_w8a8(lhs, w, out, one, one, M, N, K, F.ROWS_TYPE_F32)
    _assert_tile(tile)
    assert (out == float(torch.tensor(131071.0 * 16384))).all()


GROUPED = [((16, 16), 20, 67, 1602, 3), ((16, 32), 20, 337, 711, 16), ((32, 32), 144, 72, 34, 3), ((64, 64), 2012, 101, 2328, 5),
           ((64, 128), 850, 241, 37, 16), ((64, 128), 4058, 67, 455, 16), ((64, 256), 1365, 2181, 39, 16),
           ((64, 256), 722, 4151, 513, 16), ((128, 128), 11131, 523, 141, 11), ((128, 128), 752, 1800, 968, 16),
           ((128, 256), 13340, 769, 333, 3), ((128, 256), 8487, 401, 1300, 7), ((256, 256), 1788, 3689, 2929, 16)]


@functools.lru_cache(maxsize=1)
def _grouped(positions, N, K, experts):
    gen = torch.Generator(device="cuda").manual_seed(positions)
    lhs = _rows(gen, positions, K)
    w = torch.randint(-127, 128, (experts, N, K), generator=gen, device="cuda", dtype=torch.int8)
    lhs_scale, w_scale = _scales(gen, positions), _scales(gen, experts, N)
    # One expert has most of the rows (several panels of tiles), one none, one a single row; some rows are behind the last.
    tail = 5
    counts = [0] * experts
    counts[1] = 1
    left = positions - tail - 1
    counts[experts - 1] = left * 7 // 10
    left -= counts[experts - 1]
    for e in range(2, experts - 1):
        counts[e] = left if e == experts - 2 else left // 3
        left -= counts[e]
    counts[experts - 1] += left
    assert sum(counts) == positions - tail and counts[0] == 0
    ends = torch.tensor([0] + counts).cumsum(0)
    rows = torch.randperm(positions, generator=gen, device="cuda").int()
    expert = torch.repeat_interleave(torch.arange(experts), torch.tensor(counts)).cuda()
    return lhs, w, _pack(w), lhs_scale, w_scale, ends.int().cuda(), expert, rows


@pytest.mark.parametrize("tile,positions,N,K,experts", GROUPED)
@pytest.mark.parametrize("how", [0, F.GROUPED_GATHER, F.GROUPED_SCATTER, F.GROUPED_GATHER | F.GROUPED_SCATTER])
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_grouped_products_on_every_tile(cuda, kind, how, tile, positions, N, K, experts):
    lhs, w, packed, lhs_scale, w_scale, offsets, expert, rows = _grouped(positions, N, K, experts)
    gather, scatter = how & F.GROUPED_GATHER, how & F.GROUPED_SCATTER
    used = expert.numel()
    # Places outside: of the list, of the left-hand side, of the result.
    rows = rows.clone()
    spoiled = torch.tensor([0, used // 3, used // 2, used - 1], device="cuda")
    rows[spoiled] = torch.tensor([-1, 1 << 30, positions + 7, -(1 << 31)], dtype=torch.int32, device="cuda")
    per_token = 3 if gather else 1
    lhs_rows = -(-positions // per_token) - 2 if gather else positions - 9
    out_rows = positions - 2
    out = torch.full((positions, N + 1), 5.0, dtype=TYPES[kind], device="cuda")
    iree_amd.grouped_matmul_w8a8(lhs, packed, out, lhs_scale, w_scale, offsets, positions, experts, N, K, FLAGS[kind] | how,
                                 lhs_rows=lhs_rows, out_rows=out_rows, rows=rows if how else None, rows_per_token=per_token,
                                 out_stride0=N + 1)
    _assert_tile(tile)
    place = torch.arange(used, device="cuda")
    listed = rows[:used].long()
    source = torch.where(listed < 0, -1, listed // per_token) if gather else place
    target = listed if scatter else place
    there = (source >= 0) & (source < lhs_rows) & (target >= 0) & (target < out_rows)
    written = torch.zeros(positions, dtype=torch.bool, device="cuda")
    for e in range(experts):
        mine = there & (expert == e)
        if not mine.any():
            continue
        s, t = source[mine], target[mine]
        exact = lhs[s, :K].double() @ w[e].double().T.contiguous()
        exact = exact * lhs_scale[s].double()[:, None] * w_scale[e].double()
        ref.assert_near(out[t, :N], exact, exact)
        written[t] = True
    assert written.sum() == there.sum()                        # (nothing is scattered to twice)
    assert (out[~written] == 5).all() and (out[:, N] == 5).all()


@pytest.mark.parametrize("tile,positions,N,K,experts", GROUPED)
def test_offsets_outside_the_list_on_every_tile(cuda, tile, positions, N, K, experts):
    """The first expert's rows begin before the list and the last one's end behind it."""
    lhs, w, packed, lhs_scale, w_scale, offsets, _, _ = _grouped(positions, N, K, experts)
    wild = offsets.clone()
    wild[0], wild[-1] = -7, positions + 900
    out = torch.full((positions + 1, N), 5.0, device="cuda")
    iree_amd.grouped_matmul_w8a8(lhs, packed, out, lhs_scale, w_scale, wild, positions, experts, N, K, F.ROWS_TYPE_F32,
                                 lhs_rows=positions)
    _assert_tile(tile)
    ends = wild.clamp(0, positions).tolist()
    for e in range(experts):
        part = slice(ends[e], ends[e + 1])
        exact = lhs[part, :K].double() @ w[e].double().T.contiguous()
        exact = exact * lhs_scale[part].double()[:, None] * w_scale[e].double()
        ref.assert_near(out[part], exact, exact)
    assert (out[positions:] == 5).all()
