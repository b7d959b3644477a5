"""4-bit experts beside an fp32 router: sizes at the edges, strides, graphs and streams."""

import pytest
import torch

from tests import few_reference as ref
from tests.test_few_tokens_gpu import make
from tests.test_int4_gpu import quantized

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def problem(T, H, sizes, k, act, dtype, group, seed=40):
    """make()'s problem with an fp32 router that 16 bits cannot hold, of the first seed
    without a near tie."""
    while True:
        p = make(T, H, sizes, dtype, act, seed=seed)
        g = torch.Generator().manual_seed(seed)
        p["router"] = (torch.randn(p["router"].shape, generator=g) * H**-0.5).cuda()
        if ref.clear_choice(p["x"], p["router"], k):
            return p, quantized(p, act, group)
        seed += 100


def call(p, q, k, norm, act, x=None):
    from moe_b200.kernels import moe_few_tokens

    off = torch.tensor(p["off"], dtype=torch.int32, device="cuda")
    return moe_few_tokens(p["x"] if x is None else x, p["router"], q[0], q[1], off, p["max_width"], k,
                          norm, act)


CASES = [
    (1, 16, [(1, 16)], 1, True, "relu_squared", BF, 32),
    (8, 272, [(33, 16)], 5, True, "relu_squared", HF, 64),
    (9, 1104, [(3, 336), (5, 176), (3, 16)], 3, False, "swiglu", HF, 32),
    (64, 64, [(256, 16)], 32, True, "none", BF, 128),
    (5, 4096, [(64, 32)], 8, True, "relu_squared", BF, 128),
    (31, 2064, [(7, 80), (2, 0), (3, 48)], 4, True, "relu_squared", BF, 64),
]


@pytest.mark.parametrize("T,H,sizes,k,norm,act,dtype,group", CASES)
def test_matches_definition(T, H, sizes, k, norm, act, dtype, group, device):
    from moe_b200.kernels import check_device_status

    p, (q1, q2, v1, v2, m1, m2) = problem(T, H, sizes, k, act, dtype, group)
    out = call(p, (q1, q2), k, norm, act)
    r, b = ref.layer(p["x"], p["router"], v1, v2, p["off"], k, norm, act, m1, m2)
    ref.assert_within(out, r, b, "out")
    check_device_status(device)
    # rows apart, and on no 16 bytes
    wide = torch.full((T, H + 24), float("nan"), dtype=dtype, device=device)
    wide[:, 8:8 + H] = p["x"]
    assert torch.equal(call(p, (q1, q2), k, norm, act, wide[:, 8:8 + H]), out)
    wide[:, 3:3 + H] = p["x"]
    assert torch.equal(call(p, (q1, q2), k, norm, act, wide[:, 3:3 + H]), out)


@pytest.mark.parametrize("T", [3, 20])
def test_captured_and_on_two_streams(T, device):
    p, q = problem(T, 256, [(8, 128)], 2, "relu_squared", BF, 64)
    o, u = problem(T, 256, [(8, 128)], 2, "relu_squared", BF, 64, seed=41)
    want = [call(a, b, 2, True, "relu_squared") for a, b in ((p, q), (o, u))]
    off = torch.tensor(p["off"], dtype=torch.int32, device=device)
    from moe_b200.kernels import moe_few_tokens

    graphs = []
    for a, b in ((p, q), (o, u)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = moe_few_tokens(a["x"], a["router"], b[0], b[1], off, 128, 2)
        graphs.append((g, y, torch.cuda.Stream()))
    for _ in range(10):
        for g, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for (_, y, _), w in zip(graphs, want))


def test_down_product_captured_with_empty_experts(device):
    from moe_b200.kernels import check_device_status, grouped_gemv_down_int4

    p = make(1, 272, [(2, 80), (2, 0), (3, 48)], BF, seed=42)
    _, q2, _, v2, _, m2 = quantized(p, "none", 32)
    i32 = dict(dtype=torch.int32, device=device)
    counts = [3, 0, 2, 1, 0, 9, 4]
    start = [0]
    for c in counts:
        start.append(start[-1] + c)
    tok, off = torch.tensor(start, **i32), torch.tensor(p["off"], **i32)
    x = torch.randn(start[-1], 80, generator=torch.Generator().manual_seed(1)).to(device, BF)

    def run():
        return grouped_gemv_down_int4(x, q2, tok, off, off[1:] - off[:-1], None, 272)

    run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = run()
    x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(2)).to(device, BF))
    g.replay()
    r, b = ref.grouped(x, v2, list(zip(start, counts)), p["off"], 80, "none", True, m2)
    ref.assert_within(y, r, b, "out")
    check_device_status(device)
