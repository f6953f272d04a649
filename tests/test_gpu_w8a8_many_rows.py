"""Rows in 8 bits where a workgroup takes several rows in turn, for every shape that rows of more than 1024 elements have:
the loop over rows, the next row on its way, what the rows share in LDS. Rows of all kinds follow one another in each
workgroup. Against 64 bits on the device."""
import math

import pytest
import torch

import iree_amd
import w8a8ref as ref

pytestmark = pytest.mark.gpu
TYPES, FLAGS = ref.TYPES, ref.FLAGS


def _codes(y):
    """(q, scale f64) of rows y (f64)."""
    top = y.abs().amax(-1)
    fine = top <= torch.finfo(torch.float32).max
    q = torch.where((fine & (top > 0))[:, None], torch.round(y * 127 / torch.where(top > 0, top, 1.0)[:, None]), 0.0)
    return q.nan_to_num(0.0).to(torch.int8), torch.where(fine, top / 127, math.nan)


def _assert_rows(got, scale, want, want_scale):
    wrong = (got != want).any(-1)
    assert not wrong.any(), wrong.nonzero()[:8]
    assert torch.equal(torch.isnan(scale), torch.isnan(want_scale))
    off = (scale.double() - want_scale).abs().nan_to_num(0)
    assert (off <= 1.001 * 2.0**-24 * want_scale.nan_to_num(0) + 2.0**-150).all()


KINDS = 9


def _rows(gen, kind, rows, cols, blocks):
    """Rows of `KINDS` kinds, of which those `blocks` apart are of different ones, and which is which."""
    x = torch.randn(rows, cols, generator=gen, device="cuda") * 2
    x[:, ::29] *= 9
    n = torch.arange(rows, device="cuda")
    which = (n + n // blocks * (2 if (blocks + 2) % KINDS else 3)) % KINDS
    assert (which[blocks:] != which[:-blocks]).all()
    small = 1e-35 if kind == "bf16" else 2e-7
    for row_kind, change in (
            (1, lambda r: r.index_fill_(1, torch.tensor([cols // 3], device="cuda"), math.nan)),
            (2, lambda r: r.zero_()),
            (3, lambda r: r.mul_(small)),
            (4, lambda r: r.index_fill_(1, torch.tensor([cols - 1], device="cuda"), math.inf)),
            (5, lambda r: r.mul_(1e30 if kind == "bf16" else 500)),
            (6, lambda r: r.copy_(torch.randint(-254, 255, r.shape, generator=gen, device="cuda").index_fill_(
                1, torch.tensor([0], device="cuda"), 254))),                         # (halves between two codes)
            (7, lambda r: r.fill_(1.5)),                                                # (every value the largest)
            (8, lambda r: r.copy_(-300 - r.abs()))):                                    # (closed gates)
        at = which == row_kind
        x[at] = change(x[at])
    return x.to(TYPES[kind]), which


# Columns of one row shape each, and as many rows as its grid has workgroups, more than twice.
SHAPES = [(2048, 2048), (2045, 2048), (4096, 2048), (4091, 2048), (5000, 1024), (8192, 1024), (12000, 512), (16384, 512),
          (32768, 512), (32005, 512), (65536, 512), (40001, 512)]


@pytest.mark.parametrize("cols,blocks", SHAPES)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_many_rows(cuda, kind, cols, blocks):
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x, _ = _rows(gen, kind, 2 * blocks + 77, cols, blocks)
    q = torch.full((x.shape[0] + 1, cols), 99, dtype=torch.int8, device="cuda")
    scale = torch.full((x.shape[0] + 1,), -1.0, device="cuda")
    iree_amd.quantize_rows(x, q, scale, x.shape[0], cols, FLAGS[kind])
    _assert_rows(q[:-1], scale[:-1], *_codes(x.double()))
    assert (q[-1] == 99).all() and scale[-1] == -1


@pytest.mark.parametrize("cols,blocks", [(1024, 4096), (1500, 2048), (2048, 2048), (4096, 1024), (4091, 1024), (8192, 512),
                                         (14336, 256), (16384, 256), (16383, 256), (28672, 256), (32768, 256), (65536, 256),
                                         (50001, 256)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_many_gated_rows(cuda, kind, cols, blocks):
    gen = torch.Generator(device="cuda").manual_seed(cols)
    rows = 3 * blocks + 41
    gate, which = _rows(gen, kind, rows, cols, blocks)
    up = (torch.randn(rows, cols, generator=gen, device="cuda") * 2).to(TYPES[kind])
    up[which == 7] = 0.75
    q, scale = torch.full((rows, cols), 99, dtype=torch.int8, device="cuda"), torch.full((rows,), -1.0, device="cuda")
    iree_amd.quantize_rows(gate, q, scale, rows, cols, FLAGS[kind], up=up)
    g = gate.double()
    _assert_rows(q, scale, *_codes(g / (1 + torch.exp(-g)) * up.double()))


def _assert_norms(x, residual, weight, factors, in_place):
    tokens, addends, dim = x.shape
    kind = "bf16" if x.dtype is torch.bfloat16 else "f16"
    total = None if residual is None else residual.double()
    for j in range(addends):
        one = x[:, j].double()
        if factors is not None:
            one = torch.where(factors[:, j, None] == 0, 0.0, one) * factors[:, j, None].double()
        total = one if total is None else total + one
    h = total.float().to(x.dtype)
    q, scale = torch.full((tokens, dim), 99, dtype=torch.int8, device="cuda"), torch.full((tokens,), -1.0, device="cuda")
    out = (residual if residual is not None else x) if in_place else torch.zeros(tokens, dim, dtype=x.dtype, device="cuda")
    iree_amd.rms_norm_quantize(x, q, scale, tokens, dim, FLAGS[kind], weight=weight, eps=2.0**-20, residual=residual, sum_out=out,
                               addends=addends, addend_weights=factors)
    assert torch.equal(out.view(tokens, dim).nan_to_num(7), h.nan_to_num(7))
    want, want_scale = _codes((h.float() if weight is None else h.float() * weight.float()).double())
    rate = torch.sqrt(h.double().square().mean(-1) + 2.0**-20)
    _assert_rows(q, scale, want, want_scale / rate)


@pytest.mark.parametrize("dim,blocks", SHAPES)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_many_norms(cuda, kind, dim, blocks):
    gen = torch.Generator(device="cuda").manual_seed(dim)
    tokens = 2 * blocks + 77
    x, which = _rows(gen, kind, tokens, dim, blocks)
    residual = torch.randn(tokens, dim, generator=gen, device="cuda").to(TYPES[kind])
    residual[which == 2] = 0
    weight = (1 + torch.rand(dim, generator=gen, device="cuda")).to(TYPES[kind])
    _assert_norms(x[:, None], residual, weight, None, False)
    _assert_norms(x[:, None], residual, weight, None, True)
    _assert_norms(x[:, None].clone(), None, None, None, True)


@pytest.mark.parametrize("dim,blocks", [(1500, 2048), (4096, 2048), (4100, 512), (5000, 512), (8192, 512), (12000, 512), (16384, 512),
                                        (20000, 512), (40000, 512), (65536, 512)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_many_norms_of_several_addends(cuda, kind, dim, blocks):
    gen = torch.Generator(device="cuda").manual_seed(dim)
    tokens, addends = 2 * blocks + 77, 3
    first, which = _rows(gen, kind, tokens, dim, blocks)
    x = torch.randn(tokens, addends, dim, generator=gen, device="cuda").to(TYPES[kind])
    x[:, 1] = first
    x[which == 2] = 0
    residual = torch.randn(tokens, dim, generator=gen, device="cuda").to(TYPES[kind])
    residual[which == 2] = 0
    factors = torch.softmax(torch.randn(tokens, addends, generator=gen, device="cuda"), -1)
    factors[::5, 1] = 0                       # (what the slot holds is not looked at)
    _assert_norms(x, residual, None, factors, True)
    _assert_norms(x, None, None, None, False)
