"""A layer in 8-bit integers and its experts.

Thin wrappers of the entry points that include/iree_amd_uk.h describes under that heading
(formulas, layouts, what is refused). As in ``attention``, tensors own the device memory,
sizes are given, strides (in elements) default to tight, and work is enqueued on torch's
current stream; every tensor lies on the current device.

A layer: ``rms_norm_quantize`` adds what the layer before gave to the residual and makes rows
of 8 bits, ``matmul_w8a8`` multiplies them with packed weights, ``quantize_rows`` takes
attention's rows, or gate and up, back to 8 bits. With experts, ``moe_route`` chooses them and
sorts the tokens' slots, ``grouped_matmul_w8a8`` multiplies by expert (gathering tokens, then
scattering to slots), and the next ``rms_norm_quantize`` adds a token's slots up with their
weights.
"""
import ctypes as C
import functools

import torch

from . import flags as F
from ._lib import load_library
from .attention import _device, _stream_on, _tensor, _workspace
from .ukernel import _check

_TYPES = {F.ROWS_TYPE_F16: torch.float16, F.ROWS_TYPE_BF16: torch.bfloat16, F.ROWS_TYPE_F32: torch.float32}
_F32, _I32, _I8 = torch.float32, torch.int32, torch.int8


def rms_norm_quantize(x, q, scale, tokens, dim, flags, *, weight=None, eps=1e-6, residual=None, sum_out=None, addends=1,
                      addend_weights=None, x_stride0=None, x_stride1=None, addend_weights_stride0=None,
                      residual_stride0=None, sum_out_stride0=None, q_stride0=None, stream=None):
    """The residual's addition (of ``addends`` rows of ``x`` for every token, with weights if given), RMS
    norm, and rows of 8 bits in ``q`` with their ``scale``; the sum goes to ``sum_out``."""
    rows, device = _TYPES.get(flags & F.ROWS_TYPE_MASK), _device()
    if x_stride1 is None:
        x_stride1 = dim
    _check(load_library().iree_amd_uk_rms_norm_quantize(
        _tensor(x, rows, "x", device), addends * x_stride1 if x_stride0 is None else x_stride0, x_stride1, addends,
        _tensor(addend_weights, _F32, "addend_weights", device),
        addends if addend_weights_stride0 is None else addend_weights_stride0,
        _tensor(residual, rows, "residual", device), dim if residual_stride0 is None else residual_stride0,
        _tensor(sum_out, rows, "sum_out", device), dim if sum_out_stride0 is None else sum_out_stride0,
        _tensor(weight, rows, "weight", device), eps, _tensor(q, _I8, "q", device), dim if q_stride0 is None else q_stride0,
        _tensor(scale, _F32, "scale", device), tokens, dim, flags, _stream_on(stream, device)))


def quantize_rows(x, q, scale, rows, cols, flags, *, up=None, x_stride0=None, up_stride0=None, q_stride0=None, stream=None):
    """Rows of 8 bits of ``x``, or with ``up`` of silu(x) * up."""
    kind, device = _TYPES.get(flags & F.ROWS_TYPE_MASK), _device()
    _check(load_library().iree_amd_uk_quantize_rows(
        _tensor(x, kind, "x", device), cols if x_stride0 is None else x_stride0,
        _tensor(up, kind, "up", device), cols if up_stride0 is None else up_stride0,
        _tensor(q, _I8, "q", device), cols if q_stride0 is None else q_stride0, _tensor(scale, _F32, "scale", device), rows,
        cols, flags, _stream_on(stream, device)))


def matmul_w8a8(lhs, rhs_packed, out, lhs_scale, rhs_scale, M, N, K, flags, *, bias=None, lhs_stride0=None,
                rhs_stride0=None, out_stride0=None, stream=None):
    """``out[m][n] = sum_k lhs[m][k] rhs[n][k] * lhs_scale[m] * rhs_scale[n] + bias[n]``. Rows of ``lhs`` lie
    ``K`` rounded up to 16 apart unless told otherwise."""
    device, wide = _device(), -(-K // 16) * 16
    _check(load_library().iree_amd_uk_matmul_w8a8(
        _tensor(lhs, _I8, "lhs", device), wide if lhs_stride0 is None else lhs_stride0,
        _tensor(lhs_scale, _F32, "lhs_scale", device), _tensor(rhs_packed, _I8, "rhs_packed", device), 32 * wide if rhs_stride0 is None else rhs_stride0,
        _tensor(rhs_scale, _F32, "rhs_scale", device), _tensor(bias, _F32, "bias", device),
        _tensor(out, _TYPES.get(flags & F.ROWS_TYPE_MASK), "out", device), N if out_stride0 is None else out_stride0, M, N, K,
        flags, _stream_on(stream, device)))


def moe_route_workspace(tokens, experts):
    """Bytes of workspace that ``moe_route`` of these sizes uses (0: none)."""
    out = C.c_uint64(0)
    _check(load_library().iree_amd_uk_moe_route_workspace(tokens, experts, C.byref(out)))
    return out.value


_route_workspace = functools.lru_cache(maxsize=4096)(moe_route_workspace)


def moe_route(logits, expert_ids, expert_weights, offsets, rows, tokens, experts, top_k, flags, *, logits_stride0=None,
              workspace=None, stream=None):
    """The ``top_k`` experts of each token and their weights, and the slots in the order of their
    experts: ``rows``, those of expert ``e`` at ``offsets[e]`` to ``offsets[e + 1]``. Without a ``workspace``
    the call takes one from torch's allocator for its own duration where it uses one."""
    device = _device()
    at = _tensor(logits, _TYPES.get(flags & F.ROWS_TYPE_MASK), "logits", device)
    if workspace is None and 0 < tokens < 1 << 31 and 0 < experts <= 512:
        nbytes = _route_workspace(tokens, experts)
        if nbytes:
            workspace = _workspace(nbytes, stream)
    _check(load_library().iree_amd_uk_moe_route(
        at, experts if logits_stride0 is None else logits_stride0, _tensor(expert_ids, _I32, "expert_ids", device),
        _tensor(expert_weights, _F32, "expert_weights", device), _tensor(offsets, _I32, "offsets", device),
        _tensor(rows, _I32, "rows", device), tokens, experts, top_k, _tensor(workspace, None, "workspace", device),
        0 if workspace is None else workspace.nbytes, flags, _stream_on(stream, device)))


def grouped_matmul_w8a8(lhs, rhs_packed, out, lhs_scale, rhs_scale, offsets, positions, experts, N, K, flags, *, lhs_rows,
                        out_rows=None, rows=None, rows_per_token=1, lhs_stride0=None, rhs_stride0=None,
                        rhs_expert_stride=None, out_stride0=None, stream=None):
    """The product of ``matmul_w8a8`` by expert: the positions ``offsets[e]`` to ``offsets[e + 1]`` of a list
    with the weights of expert ``e``; by ``rows``, with GROUPED_GATHER from the rows ``rows[p] // rows_per_token``
    of ``lhs``, with GROUPED_SCATTER to the rows ``rows[p]`` of ``out`` (``out_rows`` of them, ``positions`` unless
    told otherwise)."""
    device, wide = _device(), -(-K // 16) * 16
    if rhs_stride0 is None:
        rhs_stride0 = 32 * wide
    _check(load_library().iree_amd_uk_grouped_matmul_w8a8(
        _tensor(lhs, _I8, "lhs", device), wide if lhs_stride0 is None else lhs_stride0, lhs_rows,
        _tensor(lhs_scale, _F32, "lhs_scale", device), _tensor(rhs_packed, _I8, "rhs_packed", device), rhs_stride0,
        -(-N // 32) * rhs_stride0 if rhs_expert_stride is None else rhs_expert_stride,
        _tensor(rhs_scale, _F32, "rhs_scale", device), _tensor(out, _TYPES.get(flags & F.ROWS_TYPE_MASK), "out", device),
        N if out_stride0 is None else out_stride0, positions if out_rows is None else out_rows,
        _tensor(offsets, _I32, "offsets", device), _tensor(rows, _I32, "rows", device), rows_per_token, positions, experts,
        N, K, flags, _stream_on(stream, device)))
