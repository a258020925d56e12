"""A workspace's first call may come at once, on a stream that does not wait for the default one: its arrival counters are
zero by then, whatever its memory held before."""

import ctypes as C

import pytest
import torch

from test_kv_attention_gpu import filled
from test_kv_cache_gpu import batch_of, on_device, table_of, typed

pytestmark = pytest.mark.gpu


def test_the_first_call_on_another_stream(qx):
    """Attention whose chunks are joined by the last thread block to arrive."""
    cache, table = filled(40, 8, 64, 128), table_of(1, 32, 40)
    dev, q = on_device(qx, cache), typed((1, 8, 128), torch.bfloat16, 1).cuda()
    batch, _, _ = batch_of(qx, table, [1000], [1], 0)
    want, out = torch.empty_like(q), torch.empty_like(q)
    qx.check(dev.attention_dev(batch, q, want), "attention")
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    for _ in range(20):
        # (memory that was not zero, for the workspace to get)
        held, size = C.c_void_p(), 64 << 20
        junk = torch.full((size // 4,), 7, dtype=torch.int32, device="cuda")
        del junk
        torch.cuda.empty_cache()
        out.zero_()
        torch.cuda.synchronize()
        qx.check(qx.lib.qx_workspace_create(size, C.byref(held)), "workspace")
        with torch.cuda.stream(stream):
            qx.check(dev.attention_dev(batch, q, out, workspace=held), "attention")
        stream.synchronize()
        assert torch.equal(out, want)
        qx.lib.qx_workspace_destroy(held)
    qx.check(qx.lib.qx_check_device_errors(), "attention")
