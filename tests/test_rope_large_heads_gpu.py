"""Rotary positions on heads of any size that the calls accept, on both sides of what a row of threads holds."""

import pytest
import torch

from kv_reference import rotated
from test_rope_gpu import close, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [4080, 4096, 4112, 8192, 65536, 1 << 20])
@pytest.mark.parametrize("in_place", [False, True])
def test_large_heads(qx, dtype, dim, in_place):
    rope, (x, at) = qx.Rope(128), inputs(3, 2, dim, dtype)
    x_dev = x.cuda()
    y = x_dev if in_place else torch.full_like(x_dev, float("nan"))
    qx.check(rope.apply_dev(x_dev, y, at.cuda()), "rope")
    close(y[..., :128], rotated(x[..., :128].double(), at.tolist(), rope.view.frequency[:64]), x)
    assert torch.equal(y[..., 128:].cpu(), x[..., 128:])


def test_a_large_head_on_the_host(qx):
    rope, (x, at) = qx.Rope(256, qx.ROPE_INTERLEAVED), inputs(2, 1, 8192, torch.float32)
    y = torch.zeros_like(x)
    assert rope.apply(x.numpy(), y.numpy(), at.numpy()) == qx.OK, qx.last_error()
    close(y[..., :256], rotated(x[..., :256].double(), at.tolist(), rope.view.frequency[:128], interleaved=True), x)
    assert torch.equal(y[..., 256:], x[..., 256:])
