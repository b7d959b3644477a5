"""The inference operators refuse forward-mode derivatives instead of dropping them."""

import pytest
import torch

from tests.test_few_tokens_gpu import make

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def test_tangents_are_refused(device):
    from torch.autograd import forward_ad

    from moe_b200.kernels import (Int4Weight, dequantize_int4, grouped_gemv_up_int4,
                                  moe_few_tokens, pack_int4, quantize_int4)

    p = make(2, 64, [(4, 32)], BF)
    i32 = dict(dtype=torch.int32, device=device)
    off, tok = torch.tensor(p["off"], **i32), torch.tensor([0, 1, 1, 2, 2], **i32)
    with torch.no_grad(), forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        q1 = quantize_int4(p["w1"], 32)
        plain = moe_few_tokens(p["x"], p["router"], p["w1"], p["w2"], off, 32, 2)
        for name in ("x", "router", "w1", "w2"):
            d = {**p, name: dual(p[name])}
            with pytest.raises(RuntimeError, match="tangent"):
                moe_few_tokens(d["x"], d["router"], d["w1"], d["w2"], off, 32, 2)
        with pytest.raises(RuntimeError, match="tangent"):
            grouped_gemv_up_int4(dual(p["x"]), q1, tok, off, torch.tensor([32] * 4, **i32), None, 32)
        with pytest.raises(RuntimeError, match="tangent"):
            quantize_int4(dual(p["w1"]), 32)
        with pytest.raises(RuntimeError, match="tangent"):
            pack_int4(torch.full((64, 128), 8, dtype=torch.uint8, device=device), dual(q1.scales), 32)
        scales = Int4Weight(q1.packed, dual(q1.scales), 64, 128, 32)
        q2 = quantize_int4(p["w2"], 32, row_offsets=p["off"])
        with pytest.raises(RuntimeError, match="tangent"):
            moe_few_tokens(p["x"], p["router"], scales, q2, off, 32, 2)
        with pytest.raises(RuntimeError, match="tangent"):
            dequantize_int4(scales)
        x = forward_ad.unpack_dual(dual(p["x"])).primal
        assert torch.equal(moe_few_tokens(x, p["router"], p["w1"], p["w2"], off, 32, 2), plain)
    assert torch.equal(moe_few_tokens(p["x"], p["router"], p["w1"], p["w2"], off, 32, 2), plain)
