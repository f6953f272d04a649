"""The layer in 8-bit integers and its experts in 64 bits on the CPU, from the formulas of the
header, and inputs for its tests."""
import math

import torch

from iree_amd import flags as F

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
FLAGS = {"f16": F.ROWS_TYPE_F16, "bf16": F.ROWS_TYPE_BF16, "f32": F.ROWS_TYPE_F32}


def codes(y):
    """(q int8, scale f64) of rows y (f64)."""
    top = y.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(y).all(-1, keepdim=True) & (top <= torch.finfo(torch.float32).max)
    q = torch.where(fine & (top > 0), torch.round(y * 127 / torch.where(top > 0, top, 1.0)), 0.0)
    return q.nan_to_num(0.0).to(torch.int8), torch.where(fine, top / 127, math.nan)[..., 0]


def total(x, residual=None, factors=None):
    """The sum of [tokens][addends][dim], rounded to its type."""
    wide = x.double()
    if factors is not None:
        wide = torch.where(factors[..., None] == 0, 0.0, wide) * factors.double()[..., None]
    out = wide[:, 0].clone() if residual is None else residual.double() + wide[:, 0]
    for j in range(1, x.shape[1]):
        out = out + wide[:, j]
    return out.to(x.dtype)


def norm(h, weight, eps):
    """(q, scale f64) of the normed rows of h, the kept sum."""
    wide = h.double()
    y = wide if weight is None else wide * weight.double()
    q, scale = codes(y)
    return q, scale / torch.sqrt(wide.square().mean(-1) + eps)


def silu_mul(gate, up):
    gate = gate.double()
    return gate / (1 + torch.exp(-gate)) * up.double()


def pack(w):
    """[..., N, K] int8 as tiles [..., N / 32][K / 16][32][16], zeros past N and K."""
    n, k = w.shape[-2:]
    high, wide = -(-n // 32) * 32, -(-k // 16) * 16
    full = torch.zeros(*w.shape[:-2], high, wide, dtype=torch.int8)
    full[..., :n, :k] = w
    return full.view(*w.shape[:-2], high // 32, 32, wide // 16, 16).transpose(-3, -2).contiguous()


def product(lhs, lhs_scale, w, w_scale, bias=None):
    """The exact product without the bias, and the result, f64."""
    p = (lhs.double() @ w.double().T) * lhs_scale.double()[:, None] * w_scale.double()
    return p, p if bias is None else p + bias.double()


def assert_near(got, p, want):
    """The sum becomes f32 (2^-24 of the product), is multiplied by the row's scale (2^-24), then by the channel's and
    added to the bias (2^-24 of the result), and is rounded to its type (half a step; f16 below 2^-14: 2^-25)."""
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    tolerance = 2.01 * 2.0**-24 * p.abs() + (1.01 * 2.0**-24 + 1.01 * half) * want.abs()
    if got.dtype == torch.float16:
        tolerance = tolerance + 2.0**-25
    off = (got.double() - want).abs()
    bad = ~(off <= tolerance) & ~(torch.isnan(got) & torch.isnan(want))
    assert not bad.any(), (bad.sum().item(), off[bad][:4], want[bad][:4], bad.nonzero()[:4])


def route(logits, top_k, renormalize):
    """(ids, weights f64, offsets, rows) of [tokens][experts]."""
    tokens, experts = logits.shape
    lowest = torch.finfo(torch.float32).max
    wide = logits.double().nan_to_num(nan=-math.inf, posinf=lowest, neginf=-math.inf)
    values, ids = torch.sort(wide, dim=-1, descending=True, stable=True)
    ids, there = ids[:, :top_k], values[:, :top_k] > -math.inf
    top = values[:, :1].clamp(min=-lowest)
    p = torch.where(values > -math.inf, torch.exp(values - top), 0.0)
    mine = p[:, :top_k] * there
    weights = mine / (mine if renormalize else p).sum(-1, keepdim=True).clamp(min=1e-300)
    ids = torch.where(there, ids, -1)
    slots = ids.flatten()
    offsets, rows = [0], []
    for e in range(experts):
        rows += (slots == e).nonzero()[:, 0].tolist()
        offsets.append(len(rows))
    rows += [-1] * (slots.numel() - len(rows))
    return ids.int(), weights, torch.tensor(offsets, dtype=torch.int32), torch.tensor(rows, dtype=torch.int32)


def grouped(lhs, lhs_scale, w, w_scale, offsets, rows, gather, scatter, rows_per_token, out):
    """The rows of the result that are written: (row, exact product) pairs, f64."""
    found = []
    for e in range(w.shape[0]):
        for p in range(int(offsets[e]), int(offsets[e + 1])):
            source = int(rows[p]) // rows_per_token if gather else p
            target = int(rows[p]) if scatter else p
            if (gather and int(rows[p]) < 0) or not 0 <= source < lhs.shape[0] or not 0 <= target < out:
                continue
            found.append((target, (lhs[source].double() @ w[e].double().T) * float(lhs_scale[source]) * w_scale[e].double()))
    return found


def rows8(gen, *shape):
    return torch.randn(*shape, generator=gen).mul_(32).round_().clamp_(-127, 127).to(torch.int8)


def scales(gen, *shape):
    return (torch.rand(*shape, generator=gen) + 0.5) / 64
