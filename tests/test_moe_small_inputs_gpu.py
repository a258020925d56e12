"""16-bit inputs and inner activations near the end of their range: digits down to 2^-103, as for f32."""

import pytest
import torch

import moe_reference as ref
from test_moe_gpu import check, tokens_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [2.0 ** -80, 2.0 ** -88, 2.0 ** -92, 2.0 ** -96])
def test_blocks_far_below_their_neighbours(qx, fmt, dtype, size):
    """The gate sees the first block of columns and the up projection the second, whose elements are tiny: so are their
    products, the inner activations."""
    m = ref.layer(fmt, 3, 64, 64, 1, seed=51)
    for name, at, hidden in (("gate", 0, 1), ("up", 1, 0)):
        blocks = m.raw[at].reshape(-1, 2, (34, 18)[fmt])
        blocks[:, hidden, :2] = 0  # (the block's scale)
        getattr(m, name)[..., 32 * hidden:32 * hidden + 32] = 0
    x = tokens_of(m, 5, torch.float32)
    x[:, 32:] *= size
    # (of the formula's outputs: so that zeros are no answer)
    want, limit = ref.apply(m, x.to(dtype), 2, out_type=torch.float32)
    assert float((want.abs() - limit).max()) > 0
    check(qx, m, x.to(dtype), 2, torch.float32)
