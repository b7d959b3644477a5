"""A wait for copied weights that runs out, in the few-token layer and the 4-bit products.

With a limit of 1 ns (moe_set_wait_timeout_ns) a warp gives up on weights that are still
on their way: the copies themselves are sound and land, as every warp waits for its own
before its block ends.  The launch ends with MOE_ERR_TIMEOUT in the status word, its
output means nothing, and the next call is right.  The weights (64 MB and more) are
evicted from L2 first, so that a copy takes a microsecond or more."""

import pytest
import torch

from tests.test_few_tokens_gpu import make

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def evict(device):
    buf = torch.empty(1 << 28, dtype=torch.uint8, device=device)
    return lambda: buf.fill_(1)


def runs_out(run, evict, device):
    """Three launches whose waits run out, of at most 20: not every launch has a warp that
    looks for weights before they are there (4 bits: 9 in 10; it loads its tokens first)."""
    from moe_b200._lib import MoEKernelError, lib
    from moe_b200.kernels import check_device_status

    want = run()
    check_device_status(device)
    out_of_time = 0
    for _ in range(20):
        evict()
        torch.cuda.synchronize()
        lib.moe_set_wait_timeout_ns(1)
        try:
            got = run()
            torch.cuda.synchronize()  # the launch returned on its own
        finally:
            lib.moe_set_wait_timeout_ns(0)
        try:
            check_device_status(device)
            assert torch.equal(got, want)
        except MoEKernelError as e:
            assert "timed out" in str(e)
            out_of_time += 1
        evict()
        assert torch.equal(run(), want)
        check_device_status(device)
        if out_of_time == 3:
            return
    raise AssertionError(f"{out_of_time} of 20 launches ran out of time")


@pytest.mark.parametrize("T,dtype,packed", [(4, BF, False), (20, BF, False), (3, F32, False),
                                            (4, BF, True), (20, BF, True)])
def test_layer(T, dtype, packed, evict, device):
    from moe_b200.kernels import moe_few_tokens, quantize_int4

    p = make(T, 2048, [(64, 512 if not packed else 1024)], dtype, seed=2)
    off = torch.tensor(p["off"], dtype=torch.int32, device=device)
    w1, w2 = p["w1"], p["w2"]
    if packed:
        w1, w2 = quantize_int4(w1, 64), quantize_int4(w2, 64, row_offsets=p["off"])
    runs_out(lambda: moe_few_tokens(p["x"], p["router"], w1, w2, off, p["max_width"], 8), evict,
             device)


@pytest.mark.parametrize("down", [False, True])
def test_products(down, evict, device):
    from moe_b200.kernels import grouped_gemv_down_int4, grouped_gemv_up_int4, quantize_int4

    p = make(1, 2048, [(64, 1024)], BF, seed=3)
    i32 = dict(dtype=torch.int32, device=device)
    off, tok = torch.tensor(p["off"], **i32), torch.arange(65, **i32)
    wid = torch.full((64,), 1024, **i32)
    x = torch.randn(64, 1024 if down else 2048, device=device).to(BF)
    if down:
        q = quantize_int4(p["w2"], 64, row_offsets=p["off"])
        runs_out(lambda: grouped_gemv_down_int4(x, q, tok, off, wid, None, 2048), evict, device)
    else:
        q = quantize_int4(p["w1"], 64)
        runs_out(lambda: grouped_gemv_up_int4(x, q, tok, off, wid, None, 1024), evict, device)
