"""4-bit w2 and the offsets that a call names: an expert that is refused adds nothing
and changes nothing for the others."""

import pytest
import torch

from tests import few_reference as ref
from tests.test_few_tokens_gpu import make
from tests.test_int4_gpu import quantized

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
WIDTH = 32
GOOD = [0, 32, 64, 96, 128]


def i32(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def refused_status(device):
    from moe_b200._lib import MoEKernelError
    from moe_b200.kernels import check_device_status

    with pytest.raises(MoEKernelError, match="invalid argument"):
        check_device_status(device)
    check_device_status(device)


# device offsets, token offsets, counts, experts that stay
DOWN = [
    ([0, 32, 60, 96, 128], [0, 2, 3, 5, 7], [2, 1, 2, 2], [0, 3]),
    ([0, -16, 64, 96, 128], [0, 2, 3, 5, 7], [2, 1, 2, 2], [2, 3]),
    (GOOD, [0, 2, 3, 5, 7], [2, -1, 2, 2], [0, 2, 3]),
    (GOOD, [0, 2, 9, 5, 7], [2, 1, 2, 2], [0, 3]),
    (GOOD, [-1, 2, 3, 5, 7], [2, 1, 2, 2], [1, 2, 3]),
]


@pytest.mark.parametrize("off,tok,cnt,stay", DOWN)
@pytest.mark.parametrize("dtype,group", [(BF, 32), (HF, 64)])
def test_refused_expert_leaves_the_others_of_a_down_product(off, tok, cnt, stay, dtype, group,
                                                            device):
    from moe_b200.kernels import grouped_gemv_down_int4

    p = make(1, 80, [(4, WIDTH)], dtype, seed=6)
    _, q2, _, v2, _, m2 = quantized(p, "none", group)
    x = torch.randn(7, WIDTH, generator=torch.Generator().manual_seed(3)).to(device, dtype)
    out = grouped_gemv_down_int4(x, q2, i32(tok, device), i32(off, device),
                                 i32([WIDTH] * 4, device), i32(cnt, device), 80)
    refused_status(device)
    rows = [(tok[e], cnt[e]) if e in stay else (0, 0) for e in range(4)]
    r, b = ref.grouped(x, v2, rows, GOOD, WIDTH, "none", True, m2)
    ref.assert_within(out, r, b, "out")


def layer_without(p, k, v1, v2, m1, m2, gone):
    """The layer's definition with the experts in `gone` adding nothing."""
    v2, m2 = v2.clone(), m2.clone()
    for e in gone:
        v2[GOOD[e]:GOOD[e + 1]] = 0
        m2[GOOD[e]:GOOD[e + 1]] = 0
    return ref.layer(p["x"], p["router"], v1, v2, GOOD, k, True, "relu_squared", m1, m2)


@pytest.mark.parametrize("T", [5, 12])
@pytest.mark.parametrize("off,gone", [([0, 32, 60, 96, 128], [1, 2]), ([16, 32, 64, 96, 128], [0]),
                                      ([0, 32, 64, 160, 128], [2, 3])])
def test_refused_expert_leaves_the_others_of_a_layer(off, gone, T, device):
    from moe_b200.kernels import moe_few_tokens

    p = make(T, 64, [(4, WIDTH)], BF, seed=7)
    q1, q2, v1, v2, m1, m2 = quantized(p, "relu_squared", 32)
    out = moe_few_tokens(p["x"], p["router"], q1, q2, i32(off, device), WIDTH, 4)
    refused_status(device)
    r, b = layer_without(p, 4, v1, v2, m1, m2, gone)
    ref.assert_within(out, r, b, "out")


def test_expert_wider_than_the_limit_leaves_the_others(device):
    from moe_b200.kernels import moe_few_tokens

    p = make(3, 64, [(1, 32), (1, 64), (2, 32)], BF, seed=8)
    q1, q2, v1, v2, m1, m2 = quantized(p, "relu_squared", 32)
    out = moe_few_tokens(p["x"], p["router"], q1, q2, i32(p["off"], device), 32, 4)
    refused_status(device)
    v2[32:96] = m2[32:96] = 0
    r, b = ref.layer(p["x"], p["router"], v1, v2, p["off"], 4, True, "relu_squared", m1, m2)
    ref.assert_within(out, r, b, "out")


def c_layer(p, q1, q2, off, k):
    """moe_few_tokens of the C ABI on 4-bit weights, which does not know w2's row offsets."""
    from moe_b200._lib import ACT_CODE, DTYPE_CODE, lib
    from moe_b200.kernels._ops import status_buffer

    x = p["x"]
    (T, H), E = x.shape, p["router"].shape[0]
    act = ACT_CODE["relu_squared"]
    n = lib.moe_few_tokens_workspace_bytes(T, H, E, k, WIDTH, act)
    ws = torch.empty(n, dtype=torch.uint8, device=x.device)
    out = torch.empty_like(x)
    rc = lib.moe_few_tokens(
        x.data_ptr(), T, H, H, p["router"].data_ptr(), E, q1.packed.data_ptr(),
        q1.scales.data_ptr(), q2.packed.data_ptr(), q2.scales.data_ptr(), q1.group_size,
        q2.packed.shape[0], q2.scales.shape[0], q1.cols, off.data_ptr(), WIDTH, k, 1, act,
        out.data_ptr(), H, ws.data_ptr(), n, DTYPE_CODE[x.dtype],
        status_buffer(x.device).data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    return out


def test_unknown_rows_refuse_every_expert_after_a_bad_offset(device):
    """Without w2's row offsets nothing says where the experts after a bad one start."""
    from moe_b200.kernels import check_device_status, moe_few_tokens

    p = make(5, 64, [(4, WIDTH)], BF, seed=9)
    q1, q2, v1, v2, m1, m2 = quantized(p, "relu_squared", 32)
    good = i32(GOOD, device)
    assert torch.equal(c_layer(p, q1, q2, good, 4),
                       moe_few_tokens(p["x"], p["router"], q1, q2, good, WIDTH, 4))
    check_device_status(device)
    out = c_layer(p, q1, q2, i32([0, 32, 60, 96, 128], device), 4)
    refused_status(device)
    r, b = layer_without(p, 4, v1, v2, m1, m2, [1, 2, 3])
    ref.assert_within(out, r, b, "out")
