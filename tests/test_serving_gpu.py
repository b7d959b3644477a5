"""decode as a server runs it: layers of other types and widths."""

import pytest
import torch

from tests import few_reference as ref
from tests.test_few_tokens_gpu import make_module
from tests.test_int4_gpu import spread, values

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("T", [1, 7, 30])
@pytest.mark.parametrize("sdtype", [None, BF, HF])
def test_decode_of_an_fp32_layer_on_int4_experts(sdtype, T, device):
    m = make_module([(4, 64), (3, 48)], 128, 2, F32)
    with torch.no_grad():
        q = m.quantize_experts(group_size=32, dtype=sdtype)
        dt = sdtype or BF
        assert q[0].dtype == q[1].dtype == dt
        x = torch.randn(T, 128, generator=torch.Generator().manual_seed(2)).to(device, dt)
        out = m.decode(x, experts=q)
        assert out.dtype == dt
        seg = [64] * 4 + [48] * 3
        c1, s1 = ref.quantize(m.w1, 32, [128], dt)
        c2, s2 = ref.quantize(m.w2, 32, seg, dt)
        assert ref.clear_choice(x, m.router.weight, 2)
        r, b = ref.layer(x, m.router.weight, values(c1, s1, 32, [128]), values(c2, s2, 32, seg),
                         m.expert_offsets, 2, True, "relu_squared",
                         ref.int4_terms(spread(s1, 32, [128]), dt),
                         ref.int4_terms(spread(s2, 32, seg), dt))
        ref.assert_within(out, r, b, "decode")
        with pytest.raises(TypeError, match="dtype"):
            m.decode(x.float(), experts=q)


@pytest.mark.parametrize("T", [1, 12])
def test_fp32_router_is_not_rounded(T, device):
    """Two router weights that 16 bits would make equal: the larger one wins."""
    m = make_module([(4, 32)], 64, 1, F32)
    with torch.no_grad():
        q = m.quantize_experts(group_size=32, dtype=HF)
        m.router.weight.zero_()
        m.router.weight[:, 0] = torch.tensor([0.25, 1.0, 1.0 + 2.0**-13, 0.5], device=device)
        x = torch.randn(T, 64, generator=torch.Generator().manual_seed(3)).to(device, HF)
        x[:, 0] = 1.0
        out = m.decode(x, experts=q)
        m.router.weight[[0, 1, 3]] = -4.0 * m.router.weight[2]  # expert 2 without a doubt
        assert torch.equal(out, m.decode(x, experts=q))


@pytest.mark.parametrize("sizes", [[(3, 64), (2, 24)], [(2, 8), (2, 16)]])
def test_decode_refuses_widths_that_it_cannot_compute(sizes, device):
    m = make_module(sizes, 64, 2, BF, block=8)
    x = torch.randn(2, 64, device=device, dtype=BF)
    with torch.no_grad(), pytest.raises(ValueError, match="multiples of 16"):
        m.decode(x)


def test_decode_of_blocks_of_8_that_make_widths_of_16(device):
    m, n = (make_module([(2, 16), (3, 48)], 64, 2, BF, block=b) for b in (8, 16))
    x = torch.randn(5, 64, device=device, dtype=BF)
    with torch.no_grad():
        assert torch.equal(m.decode(x), n.decode(x))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("logits,k,by_logit,by_sigmoid", [
    ([30.0, 20.0, 40.0, 0.0], 1, [2], [0]),  # sigmoids 1, 1, 1
    ([1.0, 25.0, 18.0, 32.0], 2, [3, 1], [1, 2]),
    ([-200.0, -100.0, -300.0, -90.0], 2, [3, 1], [0, 1]),  # all 0
    ([3.0, 5.0, 4.0, 1.0], 2, [1, 2], [1, 2]),  # the same choice between them
])
def test_ranking_where_sigmoids_saturate(logits, k, by_logit, by_sigmoid, dtype, device):
    """decode takes the larger logits; forward, among equal sigmoids, the lower index."""
    m = make_module([(4, 32)], 64, k, dtype)
    with torch.no_grad():
        m.router.weight.zero_()
        m.router.weight[:, 0] = torch.tensor(logits, device=device)
        x = torch.randn(3, 64, generator=torch.Generator().manual_seed(4)).to(device, dtype)
        x[:, 0] = 1.0
        inter = m.forward_with_intermediates(x[None])
        assert inter["selected_experts"].sort(1).values.tolist() == [sorted(by_sigmoid)] * 3
        sel, _ = ref.choose(x, m.router.weight, k)
        assert sel.tolist() == [by_logit] * 3
        out = m.decode(x)
        r, b = ref.layer(x, m.router.weight, m.w1, m.w2, m.expert_offsets, k, True, "relu_squared")
        # Below -88.7 expf(-logit) is infinite in fp32 and the sigmoid 0: it is off by all of
        # its value, at most exp(-88.7) < 2^-127, and its weight by 2^-127 / 1e-20 (the sum of
        # the chosen sigmoids is at least 0), times the expert's output.
        y = torch.stack([(x.double() @ m.w1[:, a:c].double()).clamp(min=0).square() @ m.w2[a:c].double()
                         for a, c in zip(m.expert_offsets, m.expert_offsets[1:])])
        b = b + k * (2.0**-127 / 1e-20) * y.abs().amax(0)
        ref.assert_within(out, r, b, "decode")
