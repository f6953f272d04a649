"""The layer in 8-bit integers without a device: what its entry points refuse, its workspaces, and
the 64-bit reference of the GPU tests against a few values worked out by hand."""
import ctypes as C
import math

import pytest
import torch

import iree_amd
import w8a8ref as ref
from iree_amd import flags as F

ONE = C.c_void_p(4096)
ODD = C.c_void_p(4097)
EIGHT = C.c_void_p(4096 + 8)
T = F.ROWS_TYPE_BF16


def _call(name, defaults, **changes):
    assert set(changes) <= set(defaults)
    lib = iree_amd.load_library()
    return getattr(lib, "iree_amd_uk_" + name)(*{**defaults, **changes}.values())


NORM = dict(x=ONE, x_stride0=64, x_stride1=64, addends=1, factors=None, factors_stride=1, residual=ONE, residual_stride=64,
            sum_out=C.c_void_p(8192), sum_stride=64, weight=ONE, eps=1e-6, q=ONE, q_stride=64, scale=ONE, tokens=3, dim=64,
            flags=T, stream=None)


@pytest.mark.parametrize("status,changes", [
    (3, dict(flags=0)), (3, dict(flags=3)), (3, dict(flags=T | 0x100)), (3, dict(tokens=-1)), (3, dict(tokens=1 << 31)),
    (3, dict(dim=-1)), (12, dict(dim=65537)), (3, dict(addends=0)), (3, dict(addends=-1)), (3, dict(addends=1025)),
    (3, dict(eps=-1.0)), (3, dict(eps=math.nan)), (3, dict(x=None)), (3, dict(x=ODD)), (3, dict(x_stride0=63)),
    (3, dict(x_stride0=-64)), (3, dict(x_stride0=1 << 62)), (3, dict(addends=2, x_stride1=63)),
    (3, dict(addends=2, x_stride1=1 << 60)), (3, dict(addends=2, x_stride0=127)), (3, dict(residual_stride=63)),
    (3, dict(residual=ODD)), (3, dict(sum_stride=60)), (3, dict(sum_out=ODD)), (3, dict(q=None)), (3, dict(q_stride=63)),
    (3, dict(scale=None)), (3, dict(scale=C.c_void_p(4098))), (3, dict(weight=ODD)), (3, dict(factors=C.c_void_p(4098))),
    (3, dict(addends=2, x_stride0=128, factors=ONE)),                                # weights closer than the addends
    (3, dict(sum_out=ONE, sum_stride=128, residual_stride=64)),                      # in place with another stride
    (3, dict(residual=None, sum_out=ONE, addends=2, x_stride0=128, sum_stride=128)),   # in place of several
])
def test_norm_refuses(status, changes):
    assert _call("rms_norm_quantize", NORM, **changes) == status
    assert iree_amd.load_library().iree_amd_uk_last_error()


QUANTIZE = dict(x=ONE, x_stride=64, up=ONE, up_stride=64, q=ONE, q_stride=64, scale=ONE, rows=3, cols=64, flags=T, stream=None)


@pytest.mark.parametrize("status,changes", [
    (3, dict(flags=0)), (3, dict(flags=3)), (3, dict(flags=T | 0x200)), (3, dict(rows=-1)), (3, dict(rows=1 << 31)),
    (3, dict(cols=-1)), (12, dict(cols=65537)), (3, dict(x=None)), (3, dict(x=ODD)), (3, dict(x_stride=63)),
    (3, dict(up=ODD)), (3, dict(up_stride=63)), (3, dict(q=None)), (3, dict(q_stride=63)), (3, dict(scale=None)),
    (3, dict(scale=C.c_void_p(4097))),
])
def test_rows_refuse(status, changes):
    assert _call("quantize_rows", QUANTIZE, **changes) == status


MATMUL = dict(lhs=ONE, lhs_stride=112, lhs_scale=ONE, rhs=ONE, rhs_stride=112 * 32, rhs_scale=ONE, bias=ONE, out=ONE,
              out_stride=70, M=5, N=70, K=100, flags=T, stream=None)


@pytest.mark.parametrize("status,changes", [
    (3, dict(flags=0)), (3, dict(flags=4)), (3, dict(flags=T | 0x100)), (3, dict(M=-1)), (3, dict(M=1 << 31)), (3, dict(N=-1)),
    (3, dict(N=(1 << 24) + 1)), (3, dict(K=-1)), (12, dict(K=131072)), (3, dict(lhs=None)), (3, dict(lhs=EIGHT)),
    (3, dict(lhs_stride=100)), (3, dict(lhs_stride=120)), (3, dict(lhs_stride=96)), (12, dict(lhs_stride=(1 << 22) + 16)),
    (3, dict(rhs=None)), (3, dict(rhs=EIGHT)), (3, dict(rhs_stride=112 * 32 - 16)), (3, dict(rhs_stride=112 * 32 + 8)),
    (3, dict(rhs_stride=(1 << 24) + 16)), (3, dict(lhs_scale=None)), (3, dict(rhs_scale=None)),
    (3, dict(rhs_scale=C.c_void_p(4098))), (3, dict(bias=ODD)), (3, dict(out=None)), (3, dict(out=ODD)),
    (3, dict(out_stride=69)), (3, dict(flags=F.ROWS_TYPE_F32, out=C.c_void_p(4098))),
])
def test_product_refuses(status, changes):
    assert _call("matmul_w8a8", MATMUL, **changes) == status


ROUTE = dict(logits=ONE, stride=64, ids=ONE, weights=ONE, offsets=ONE, rows=ONE, tokens=5, experts=64, top_k=8, workspace=None,
             nbytes=0, flags=T, stream=None)


@pytest.mark.parametrize("status,changes", [
    (3, dict(flags=0)), (3, dict(flags=4)), (3, dict(flags=T | 0x200)), (3, dict(tokens=-1)), (3, dict(tokens=1 << 28)),
    (3, dict(experts=0)), (3, dict(top_k=0)), (3, dict(top_k=65)), (12, dict(experts=513, stride=513)),
    (12, dict(experts=128, stride=128, top_k=65)), (3, dict(logits=None)), (3, dict(logits=ODD)), (3, dict(stride=63)),
    (3, dict(ids=None)), (3, dict(weights=None)), (3, dict(offsets=None)), (3, dict(rows=None)), (3, dict(rows=C.c_void_p(4098))),
    (3, dict(nbytes=64)), (3, dict(workspace=EIGHT, nbytes=64)), (3, dict(flags=F.ROWS_TYPE_F32, logits=C.c_void_p(4098))),
])
def test_route_refuses(status, changes):
    assert _call("moe_route", ROUTE, **changes) == status


GATHER, SCATTER = F.GROUPED_GATHER, F.GROUPED_SCATTER
GROUPED = dict(lhs=ONE, lhs_stride=112, lhs_rows=9, lhs_scale=ONE, rhs=ONE, rhs_stride=112 * 32, rhs_expert=3 * 112 * 32,
               rhs_scale=ONE, out=ONE, out_stride=70, out_rows=9, offsets=ONE, rows=ONE, rows_per_token=2, positions=9,
               experts=4, N=70, K=100, flags=T | GATHER, stream=None)


@pytest.mark.parametrize("status,changes", [
    (3, dict(flags=0)), (3, dict(flags=T | 0x400)), (3, dict(lhs_rows=-1)), (3, dict(out_rows=-1)), (3, dict(positions=-1)),
    (3, dict(positions=1 << 31)), (3, dict(experts=-1)), (12, dict(experts=513)), (3, dict(rows_per_token=0)),
    (3, dict(rows=None)), (3, dict(rows=None, flags=T | SCATTER)), (3, dict(rows=ODD, flags=T)), (3, dict(offsets=None)),
    (3, dict(rhs_expert=3 * 112 * 32 - 16)), (3, dict(rhs_expert=3 * 112 * 32 + 8)), (3, dict(lhs_stride=100)),
    (12, dict(lhs_rows=1 << 30)), (3, dict(N=-1)), (12, dict(K=131072)), (3, dict(out_stride=69)), (3, dict(lhs_scale=None)),
])
def test_grouped_product_refuses(status, changes):
    assert _call("grouped_matmul_w8a8", GROUPED, **changes) == status


def test_nothing_to_do():
    assert _call("rms_norm_quantize", NORM, tokens=0) == 0
    assert _call("rms_norm_quantize", NORM, dim=0) == 0
    assert _call("quantize_rows", QUANTIZE, rows=0) == 0
    assert _call("quantize_rows", QUANTIZE, cols=0) == 0
    assert _call("matmul_w8a8", MATMUL, M=0) == 0
    assert _call("matmul_w8a8", MATMUL, N=0) == 0
    for size in ("lhs_rows", "out_rows", "positions", "experts", "N"):
        assert _call("grouped_matmul_w8a8", GROUPED, **{size: 0}) == 0


def test_workspaces():
    assert iree_amd.moe_route_workspace(1, 8) == 0
    assert iree_amd.moe_route_workspace(0, 8) == 0
    n = iree_amd.moe_route_workspace(100000, 64)
    assert 0 < n <= 256 * 64 * 4
    for tokens, experts in ((-1, 8), (1 << 31, 8), (5, 0), (5, 513)):
        with pytest.raises(iree_amd.ukernel.UkError):
            iree_amd.moe_route_workspace(tokens, experts)
    lib = iree_amd.load_library()
    assert lib.iree_amd_uk_moe_route_workspace(5, 8, None) == 3


def test_tensors_are_checked():
    x = torch.zeros(4, 64, dtype=torch.float16)
    q, s = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)
    with pytest.raises(ValueError, match="current CUDA"):
        iree_amd.rms_norm_quantize(x, q, s, 4, 64, F.ROWS_TYPE_F16)
    with pytest.raises(ValueError, match="current CUDA"):
        iree_amd.quantize_rows(x, q, s, 4, 64, F.ROWS_TYPE_F16)
    with pytest.raises(ValueError, match="current CUDA"):
        iree_amd.matmul_w8a8(q, q, x, s, s, 4, 64, 64, F.ROWS_TYPE_F16)
    i = torch.zeros(64, dtype=torch.int32)
    with pytest.raises(ValueError, match="current CUDA"):
        iree_amd.moe_route(x, i, s, i, i, 4, 64, 2, F.ROWS_TYPE_F16)
    with pytest.raises(ValueError, match="current CUDA"):
        iree_amd.grouped_matmul_w8a8(q, q, x, s, s, i, 4, 2, 64, 64, F.ROWS_TYPE_F16, lhs_rows=4)


def test_the_reference():
    q, scale = ref.codes(torch.tensor([[254.0, 1.0, 3.0, -5.0], [0.0, 0, 0, 0], [math.inf, 1, 0, 0]], dtype=torch.float64))
    assert q.tolist() == [[127, 0, 2, -2], [0] * 4, [0] * 4]      # halves go to the even code
    assert scale[0] == 2 and scale[1] == 0 and math.isnan(scale[2])
    q, scale = ref.norm(torch.tensor([[3.0, -4.0]]), torch.tensor([1.0, 2.0]), 0.0)
    assert q.tolist() == [[48, -127]] and abs(scale[0] - 8 / math.sqrt(12.5) / 127) < 1e-15
    w = torch.arange(33 * 17, dtype=torch.int64).to(torch.int8).view(33, 17)
    p = ref.pack(w)
    assert p.shape == (2, 2, 32, 16) and p[1, 1, 0, 0] == w[32, 16] and p[0, 1, 5, 0] == w[5, 16] and p[1, 0, 1].sum() == 0
    ids, weights, offsets, rows = ref.route(torch.tensor([[1.0, 2, 2, -math.inf], [-math.inf] * 4, [0, 0, 0, 5]]), 2, True)
    assert ids.tolist() == [[1, 2], [-1, -1], [3, 0]] and weights[0].tolist() == [0.5, 0.5] and weights[1].tolist() == [0, 0]
    assert offsets.tolist() == [0, 1, 2, 3, 4] and rows.tolist() == [5, 0, 1, 4, -1, -1]
