"""The device status word, whatever the mode of the first call on a device."""

import pytest
import torch

from tests.test_few_tokens_gpu import make, make_module

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture
def first_call(device):
    """As in a process that has made no call yet."""
    from moe_b200.kernels import _ops

    torch.cuda.synchronize()
    kept = dict(_ops._status_bufs), dict(_ops._dep_buffers)
    _ops._status_bufs.clear()
    _ops._dep_buffers.clear()
    yield
    torch.cuda.synchronize()
    _ops._status_bufs.update(kept[0])
    _ops._dep_buffers.update(kept[1])


def test_first_call_in_inference_mode(first_call, device):
    from moe_b200._lib import MoEKernelError
    from moe_b200.kernels import check_device_status, moe_few_tokens

    p = make(3, 64, [(4, 32)], BF)
    off = torch.tensor([0, 32, 60, 96, 128], dtype=torch.int32, device=device)
    m = make_module([(4, 64)], 128, 2, BF)
    with torch.inference_mode():
        m(torch.randn(1, 3, 128, device=device, dtype=BF))
        check_device_status(device)
        moe_few_tokens(p["x"], p["router"], p["w1"], p["w2"], off, 32, 2)
    with pytest.raises(MoEKernelError):
        check_device_status(device)
    check_device_status(device)
    with torch.inference_mode():
        moe_few_tokens(p["x"], p["router"], p["w1"], p["w2"], off, 32, 2)
        with pytest.raises(MoEKernelError):
            check_device_status(device)
        check_device_status(device)


def test_first_call_in_a_capture(first_call, device):
    """The word is zero before the graph runs, and a replay does not clear what another
    call has set."""
    from moe_b200._lib import MoEKernelError
    from moe_b200.kernels import check_device_status, moe_few_tokens

    p = make(3, 64, [(4, 32)], BF)
    good = torch.tensor(p["off"], dtype=torch.int32, device=device)
    bad = torch.tensor([0, 32, 60, 96, 128], dtype=torch.int32, device=device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = moe_few_tokens(p["x"], p["router"], p["w1"], p["w2"], good, 32, 2)
    check_device_status(device)
    moe_few_tokens(p["x"], p["router"], p["w1"], p["w2"], bad, 32, 2)
    graph.replay()
    torch.cuda.synchronize()
    with pytest.raises(MoEKernelError):
        check_device_status(device)
    check_device_status(device)
    assert torch.equal(out, moe_few_tokens(p["x"], p["router"], p["w1"], p["w2"], good, 32, 2))
