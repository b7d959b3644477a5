"""How near 4-bit products come: errors of the whole beside the element bounds, weights
that are mostly zero, values near the end of the range."""

import pytest
import torch

from tests import few_reference as ref
from tests.test_int4_gpu import spread, values

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def problem(dtype, H, widths, group, seed, zero=False):
    """Codes, scales and a packed weight [H, sum of widths] of one segment."""
    from moe_b200.kernels import pack_int4

    g = torch.Generator().manual_seed(seed)
    N = sum(widths)
    codes = torch.randint(0, 16, (H, N), dtype=torch.uint8, generator=g)
    if zero:  # one code a group and column is not 8
        keep = torch.zeros(H, N, dtype=torch.bool)
        at = torch.randint(0, group, (-(-H // group), N), generator=g)
        rows = (torch.arange(-(-H // group))[:, None] * group + at).clamp(max=H - 1)
        keep.scatter_(0, rows, True)
        codes = torch.where(keep, codes, torch.full_like(codes, 8))
    scales = ((torch.rand(-(-H // group), N, generator=g) * 0.5 + 0.75) * 0.01).to(dtype)
    codes, scales = codes.cuda(), scales.cuda()
    return (pack_int4(codes, scales, group), values(codes, scales, group, [H]),
            ref.int4_terms(spread(scales, group, [H]), dtype))


def up(x, q, widths, act):
    from moe_b200.kernels import grouped_gemv_up_int4

    i32 = dict(dtype=torch.int32, device=x.device)
    off = torch.tensor([0, *torch.tensor(widths).cumsum(0).tolist()], **i32)
    E, n = len(widths), x.shape[0] // len(widths)
    tok = torch.arange(E + 1, **i32) * n
    out = grouped_gemv_up_int4(x, q, tok, off, torch.tensor(widths, **i32), None, max(widths), act)
    return out, [(e * n, n) for e in range(E)], off.tolist()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("act", ["none", "relu_squared"])
@pytest.mark.parametrize("widths", [[336, 176], [6400, 6400]])  # tiles of 64 and of 128 columns
def test_error_of_the_whole(dtype, group, act, widths, device):
    """Relative Frobenius error.  The output's rounding is at most half a step; the sums'
    error, some 2^-22 of a running sum of (B + 64) sum x over 32 rows, at most 16 K against
    products of 8 x 4.6 sqrt(32) = 210, is 2^-15.6 a group and less on the whole: below a
    quarter of fp16's half step (twice that when squared)."""
    H = 1104
    q, v, _ = problem(dtype, H, widths, group, 31)
    x = torch.randn(10, H, generator=torch.Generator().manual_seed(5)).to(device, dtype)
    out, rows, off = up(x, q, widths, act)
    want = torch.zeros_like(out, dtype=torch.float64)
    for e, (r, n) in enumerate(rows):
        u = x[r:r + n].double() @ v[:, off[e]:off[e + 1]]
        want[r:r + n, :widths[e]] = u.clamp(min=0).square() if act == "relu_squared" else u
    err = float((out.double() - want).norm() / want.norm())
    assert err <= 1.5 * ref.HALF_STEP[dtype], err


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("group", [32, 128])
def test_weights_that_are_mostly_zero(dtype, group, device):
    """The error follows the scales and x, not the weights."""
    H, widths = 592, [208, 64]
    q, v, m = problem(dtype, H, widths, group, 32, zero=True)
    x = (torch.randn(6, H, generator=torch.Generator().manual_seed(6)) + 2).to(device, dtype)
    out, rows, off = up(x, q, widths, "none")
    r, b = ref.grouped(x, v, rows, off, max(widths), "none", False, m)
    ref.assert_within(out, r, b, "out")


@pytest.mark.parametrize("dtype", [BF, HF])
def test_quantised_columns_of_zeros_are_zero(dtype, device):
    from moe_b200.kernels import quantize_int4

    w = (torch.randn(208, 96, generator=torch.Generator().manual_seed(7)) * 0.1).to(device, dtype)
    w[:, 5:70:3] = 0
    x = torch.randn(4, 208, generator=torch.Generator().manual_seed(8)).to(device, dtype)
    out, _, _ = up(x, quantize_int4(w, 64), [96], "none")
    assert not bool(out[:, 5:70:3].any()) and bool(out[:, 4].all())


def test_bf16_values_below_2_to_the_115(device):
    """The largest documented values, all of one sign, stay finite and right."""
    H, widths = 256, [64, 128]
    q, v, m = problem(BF, H, widths, 64, 33)
    g = torch.Generator().manual_seed(9)
    x = torch.rand(4, H, generator=g) * 0.5 + 0.5
    x = (x.to(BF).float().clamp(max=1 - 2.0**-8) * 2.0**115).to(device, BF)
    x[2:] = -x[2:]
    out, rows, off = up(x, q, widths, "none")
    assert bool(torch.isfinite(out).all())
    r, b = ref.grouped(x, v, rows, off, max(widths), "none", False, m)
    ref.assert_within(out, r, b, "out")


def test_scales_above_the_range_read_back_as_nan(device):
    from moe_b200.kernels import dequantize_int4, quantize_int4

    w = torch.randn(64, 16, device=device)
    w[40, 3] = 7.0 * 65536  # a scale of 65536: above fp16, fine in bf16
    back = dequantize_int4(quantize_int4(w, 32, dtype=HF))
    bad = torch.zeros(64, 16, dtype=torch.bool, device=device)
    bad[32:, 3] = True
    assert torch.equal(torch.isnan(back), bad)
    assert not bool(torch.isnan(dequantize_int4(quantize_int4(w, 32, dtype=BF))).any())
