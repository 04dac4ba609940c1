"""The 4-bit projection beside tests/test_q4_gpu.py."""
import pytest
import torch

import pesti_head as ph

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("back", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_held_again(back, group):
    """A weight that is read back and held again is the same, bit for bit, and so are its logits: the group's largest
    value is -8 of its scale, which every type here holds, so that the scale comes back; the other values are whole
    multiples of it, of at most 7, that reading back moves by at most 2^-8 of themselves: 7/256 of the scale."""
    g = torch.Generator(device="cuda").manual_seed(group)
    V, D = 300, 1000
    w = torch.randn(V, D, generator=g, device="cuda") * torch.logspace(-2, 1, V, device="cuda")[:, None]
    one = ph.quantize_head(w.bfloat16(), group)
    two = ph.quantize_head(one.dequantize(back), group)
    assert torch.equal(one.packed, two.packed) and torch.equal(one.tile_scale, two.tile_scale)
    for rows in (3, 20):
        x = torch.randn(rows, D, generator=g, device="cuda").bfloat16()
        assert torch.equal(ph.head_logits(x, one, dtype=torch.float32), ph.head_logits(x, two, dtype=torch.float32))
