"""What host calls of a mixture-of-experts layer give back besides the output; threads that each call with a stream and a
workspace of their own, of which every call is counted."""

import threading

import numpy as np
import pytest
import torch

import moe_reference as ref
from test_moe_gpu import prepared, router, tokens_of, workspace

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("normalise", [False, True])
def test_experts_and_weights_of_host_calls(qx, dtype, sigmoid, normalise):
    m = ref.layer(1, 9, 128, 64, 1, seed=13)
    x = tokens_of(m, 8, dtype)
    chosen, weights = np.full((8, 3), -1, np.int32), np.full((8, 3), np.nan, np.float32)
    r = qx.Router(m.router.numpy(), 3, qx.SCORE_SIGMOID if sigmoid else qx.SCORE_SOFTMAX, m.bias.numpy(), normalise, 1.5)
    out = np.empty_like(x.numpy())
    qx.check(prepared(qx, m, host=True).apply(r, x.numpy(), out, chosen=chosen, weights=weights), "apply")
    kind = dict(sigmoid=sigmoid, biased=True, normalise=normalise, scale=1.5)
    _, want, limit = ref.route(m, x, 3, chosen=torch.from_numpy(chosen).long(), **kind)
    assert bool(((torch.from_numpy(weights).double() - want).abs() <= limit).all())
    # the device's are the same
    picks, shares = torch.empty(8, 3, dtype=torch.int32, device="cuda"), torch.empty(8, 3, device="cuda")
    qx.check(prepared(qx, m).apply_dev(router(qx, m, 3, **kind), x.cuda(), torch.empty_like(x, device="cuda"), chosen=picks,
                                       weights=shares), "apply")
    assert np.array_equal(picks.cpu().numpy(), chosen) and np.array_equal(shares.cpu().numpy(), weights)


def test_every_call_of_every_thread(qx):
    m = ref.layer(1, 16, 512, 256, 1, seed=35)
    experts, r = prepared(qx, m), router(qx, m, 4)
    x = tokens_of(m, 9, torch.bfloat16).cuda()
    want = torch.empty_like(x)
    qx.check(experts.apply_dev(r, x, want), "apply")
    torch.cuda.synchronize()
    right, failures = [0] * 3, []

    def work(number):
        try:
            space, stream = workspace(qx), torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(50):
                    out = torch.full_like(x, float("nan"))
                    qx.check(experts.apply_dev(r, x, out, workspace=space), "apply")
                    stream.synchronize()
                    assert torch.equal(out, want), "other bits"
                    right[number] += 1
            qx.lib.qx_workspace_destroy(space)
        except BaseException as e:  # (a thread's end would go unnoticed)
            failures.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    qx.check(qx.lib.qx_check_device_errors(), "apply")
    assert not failures, failures
    assert right == [50] * 3
