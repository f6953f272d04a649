"""attention_kv4 on prompts that fill the device, against its formula in 64 bits."""
import math

import pytest
import torch

import kv4ref
from test_gpu_attention_kv4 import BF16, F16, Case, _gen, _normal

pytestmark = pytest.mark.gpu


def _replace(case, k, v):
    """Rows [pages][kv heads][page][D] in place of the case's own, what no sequence owns still NaN."""
    old = case.cache.view(case.pages, case.kv_heads, -1)
    new = kv4ref.pack(k, v, case.page).view(old.shape)
    at = case.page * case.dim
    unowned = (old[..., at:] == 0xFF)
    new[..., at:][unowned] = 0xFF
    old.copy_(new)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,q_lens", [(4, 2, [3, 40]), (64, 16, [130, 128, 200, 150])])
def test_values_past_the_range_of_f16(uk, cuda, heads, kv_heads, q_lens, dim, window, sinks):
    """V rows of bf16 whose offset + 8 scales pass 65504, as far as both saturate: finite in the
    result of the queries that see them, without a trace in that of all others, before them and behind
    their window."""
    case = Case(61, BF16, heads, kv_heads, dim, 16, q_lens, [n + 70 for n in q_lens])
    gen = _gen(62)
    k, v = (_normal(gen, case.pages, kv_heads, 16, dim) for _ in range(2))
    k, v = k.to(BF16), v.to(BF16)
    ramp = torch.linspace(0, 1, dim, device="cuda")
    for token, row in ((33, ramp * 150000), (75, ramp * 1e30), (76, (ramp - 1) * 1e30), (90, 60000 + ramp * 9e4),
                       (101, (ramp - 0.5) * 3e38)):
        for b, n in enumerate(case.kv_lens):
            if token < n:
                v[int(case.table[b, token // 16]), :, token % 16] = row.to(BF16)
    _replace(case, k, v)
    out = case.run(uk, window=window, sinks=sinks)
    assert bool(torch.isfinite(out).all())
    case.check(out, window=window, sinks=sinks)
