"""A 4-bit w2 that was quantised for other experts than the call's offsets name."""

import pytest
import torch

from tests import few_reference as ref
from tests.test_few_tokens_gpu import make, make_module
from tests.test_int4_gpu import quantized
from tests.test_packed_rows_gpu import BF, GOOD, WIDTH, i32, layer_without, refused_status

pytestmark = pytest.mark.gpu

# as many block rows, and groups of 64, as the offsets need
OTHER = [0, 16, 64, 96, 128]


@pytest.mark.parametrize("T", [4, 11])
def test_layer_refuses_experts_of_other_rows(T, device):
    from moe_b200.kernels import moe_few_tokens, quantize_int4

    p = make(T, 64, [(4, WIDTH)], BF, seed=11)
    q1, _, v1, v2, m1, m2 = quantized(p, "relu_squared", 64)
    other = quantize_int4(p["w2"], 64, row_offsets=OTHER)
    out = moe_few_tokens(p["x"], p["router"], q1, other, i32(GOOD, device), WIDTH, 4)
    refused_status(device)
    # experts 2 and 3 have the same rows in both
    r, b = layer_without(p, 4, v1, v2, m1, m2, [0, 1])
    ref.assert_within(out, r, b, "out")


def test_down_product_refuses_experts_of_other_rows(device):
    from moe_b200.kernels import grouped_gemv_down_int4, quantize_int4

    p = make(1, 64, [(4, WIDTH)], BF, seed=12)
    _, _, _, v2, _, m2 = quantized(p, "none", 64)
    other = quantize_int4(p["w2"], 64, row_offsets=OTHER)
    x = torch.randn(8, WIDTH, generator=torch.Generator().manual_seed(4)).to(device, BF)
    out = grouped_gemv_down_int4(x, other, i32([0, 2, 4, 6, 8], device), i32(GOOD, device),
                                 i32([WIDTH] * 4, device), None, 64)
    refused_status(device)
    r, b = ref.grouped(x, v2, [(0, 0), (0, 0), (4, 2), (6, 2)], GOOD, WIDTH, "none", True, m2)
    ref.assert_within(out, r, b, "out")


def test_decode_refuses_experts_of_another_layer(device):
    m = make_module([(4, 32)], 64, 2, BF)
    n = make_module([(1, 16), (1, 48), (2, 32)], 64, 2, BF)
    x = torch.randn(3, 64, device=device, dtype=BF)
    with torch.no_grad():
        m.decode(x, experts=m.quantize_experts())
        with pytest.raises(ValueError, match="offsets"):
            m.decode(x, experts=n.quantize_experts())


def test_decode_takes_experts_that_were_pickled(device):
    import copy

    m = make_module([(1, 16), (1, 48), (2, 32)], 64, 2, BF)
    x = torch.randn(3, 64, device=device, dtype=BF)
    with torch.no_grad():
        q = m.quantize_experts()
        assert torch.equal(m.decode(x, experts=copy.deepcopy(q)), m.decode(x, experts=q))
        assert torch.equal(m.decode(x, experts=(m.w1, m.w2)), m.decode(x))
        one = make_module([(1, 32)], 64, 1, BF)
        from moe_b200.kernels import quantize_int4

        whole = (quantize_int4(one.w1), quantize_int4(one.w2))  # one segment: no row offsets
        assert torch.equal(one.decode(x, experts=whole), one.decode(x, experts=one.quantize_experts()))
