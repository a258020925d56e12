"""A batch that contradicts itself is reported without touching what other calls are at: no kernel was stopped, so the
arrival counters that calls share with their workspace stay as they are."""

import ctypes as C

import numpy as np
import pytest
import torch

from test_kv_attention_gpu import BF16, filled
from test_kv_cache_gpu import batch_of, on_device, table_of, typed

pytestmark = pytest.mark.gpu


def bad_append(qx, dev, stream):
    """A function that enqueues an append into a block that the cache does not have."""
    batch, _, _ = batch_of(qx, np.array([[99]], np.int32), [1], [1])
    k = torch.zeros(1, *dev.arrays[0].shape[1::2], device="cuda")

    def call():
        with torch.cuda.stream(stream):
            assert dev.append_dev(batch, k, k) == qx.OK
    return call


def test_a_report_during_a_capture(qx):
    """The report reads a word of the host's and waits for nothing: a capture on another stream goes on."""
    cache, table = filled(60, 2, 64, 128), table_of(1, 60, 60)
    dev, batch = on_device(qx, cache), batch_of(qx, table, [3800], [1])[0]
    q = typed((1, 8, 128), BF16, 1).cuda()
    want, out = torch.zeros_like(q), torch.zeros_like(q)
    assert dev.attention_dev(batch, q, want) == qx.OK
    bad_append(qx, dev, torch.cuda.current_stream())()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert dev.attention_dev(batch, q, out) == qx.OK
        assert qx.lib.qx_check_device_errors() == qx.DEVICE_ERROR and "block" in qx.last_error()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and qx.lib.qx_check_device_errors() == qx.OK


@pytest.mark.parametrize("lengths", [[3800], [4000] * 30])
def test_reports_beside_attention_on_another_stream(qx, lengths):
    """One session in parts, and many cut evenly, in the library's own workspace, while another stream's batches are
    reported: every call's output is whole, and so is the next one's."""
    cache, table = filled(64, 2, 64, 128), table_of(1, 64, 64).repeat(len(lengths), 0)
    dev, batch = on_device(qx, cache), batch_of(qx, table, lengths, [1] * len(lengths))[0]
    q = typed((len(lengths), 8, 128), BF16, 1).cuda()
    want = torch.zeros_like(q)
    assert dev.attention_dev(batch, q, want) == qx.OK
    torch.cuda.synchronize()
    work, other = torch.cuda.Stream(), torch.cuda.Stream()
    bad, outs, reports = bad_append(qx, dev, other), [torch.zeros_like(q) for _ in range(300)], 0
    for i, out in enumerate(outs):
        with torch.cuda.stream(work):
            assert dev.attention_dev(batch, q, out) == qx.OK
        if i % 4 == 0:
            bad()
        reports += qx.lib.qx_check_device_errors() == qx.DEVICE_ERROR
    torch.cuda.synchronize()
    assert reports + (qx.lib.qx_check_device_errors() == qx.DEVICE_ERROR) > 1
    assert all(torch.equal(out, want) for out in outs)
    after = torch.zeros_like(q)
    assert dev.attention_dev(batch, q, after) == qx.OK
    torch.cuda.synchronize()
    assert torch.equal(after, want) and qx.lib.qx_check_device_errors() == qx.OK


def test_a_workspace_of_another_device_is_refused(qx):
    """Its memory lies where the kernels of this device must not follow it. (There is one device here: the workspace says
    that it belongs to another.)"""
    cache, table = filled(60, 2, 64, 128), table_of(1, 60, 60)
    dev, batch = on_device(qx, cache), batch_of(qx, table, [3800], [1])[0]
    q, out = typed((1, 8, 128), BF16, 1).cuda(), torch.full((1, 8, 128), 5.0, dtype=BF16, device="cuda")
    workspace = C.c_void_p()
    assert qx.lib.qx_workspace_create(64 << 20, C.byref(workspace)) == qx.OK
    device = C.c_int.from_address(workspace.value)
    assert device.value == torch.cuda.current_device()
    device.value += 1
    assert dev.attention_dev(batch, q, out, workspace=workspace) == qx.INVALID_ARGUMENT
    torch.cuda.synchronize()
    assert bool((out == 5).all())
    device.value -= 1
    assert dev.attention_dev(batch, q, out, workspace=workspace) == qx.OK
    qx.lib.qx_workspace_destroy(workspace)
