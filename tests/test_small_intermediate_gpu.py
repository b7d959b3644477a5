"""Intermediates near the bottom of the storage type: what is kept of them is what the
documentation says, and no less than the layer's forward keeps."""

import pytest
import torch

from tests import few_reference as ref
from tests.test_few_tokens_gpu import call, make

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
H, W, T = 256, 128, 6


def small(dtype, u, device):
    """One expert that every token reaches with weight 1; pre-activations of about u; down
    weights near 1, so that the intermediate's error is not below the output's rounding."""
    p = make(T, H, [(1, W)], dtype, seed=21)
    p["w1"] = (p["w1"].float() * u).to(dtype)
    g = torch.Generator().manual_seed(22)
    p["w2"] = torch.randn(W, H, generator=g).to(device, dtype)
    h = (p["x"].double() @ p["w1"].double()).clamp(min=0).square()
    return p, h


@pytest.mark.parametrize("T_", [3, 6])  # remainders in spare columns, and not
@pytest.mark.parametrize("u", [0.25, 2.0**-5, 2.0**-9])
def test_fp16_keeps_2_to_the_minus_25(u, T_, device):
    p, h = small(HF, u, device)
    p["x"], h = p["x"][:T_], h[:T_]
    out = call(p, 1).double()
    w2 = p["w2"].double()
    want = h @ w2
    # first order: the up sums' rounding, the intermediate's, the down sums', the output's
    du = (p["x"].double().abs() @ p["w1"].double().abs()) * ref.adds(H, HF)
    kept = torch.maximum(h * 2.0**-22, torch.full_like(h, 2.0**-25)) * (h > 0)
    dh = 2 * h.sqrt() * du + du * du + h * 2.0**-22 + kept
    bound = dh @ w2.abs() + (h @ w2.abs()) * (ref.adds(W, HF) + 2.0**-20)
    bound += torch.maximum(want.abs() * 2.0**-11, torch.full_like(want, 2.0**-25)) * (1 + 2.0**-10)
    assert bool(((out - want).abs() <= bound).all())
    # and on the whole: roundings are independent, so their squares add up
    rms = (kept.square() @ w2.square() + (want.abs() * 2.0**-11).clamp(min=2.0**-25).square()).sum()
    assert float((out - want).square().sum()) <= float(rms)


@pytest.mark.parametrize("u", [2.0**-9, 2.0**-20])
def test_bf16_keeps_its_digits(u, device):
    """bf16 has fp32's range: 2^-16 of the value however small."""
    p, h = small(BF, u, device)
    out = call(p, 1).double()
    w2 = p["w2"].double()
    want = h @ w2
    du = (p["x"].double().abs() @ p["w1"].double().abs()) * ref.adds(H, BF)
    dh = 2 * h.sqrt() * du + du * du + h * 2.0**-16
    bound = dh @ w2.abs() + (h @ w2.abs()) * (ref.adds(W, BF) + 2.0**-20)
    bound += want.abs() * 2.0**-8 * (1 + 2.0**-10)
    assert bool(((out - want).abs() <= bound).all())
