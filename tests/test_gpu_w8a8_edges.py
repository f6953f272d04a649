"""The layer in 8-bit integers on the device where its definitions are easily missed: roundings, sizes
of values at the ends of f32, sizes of tensors next to the limits."""
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
