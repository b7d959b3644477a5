"""4-bit weights: quantising, packing and back against the definition, and the
products that read them against 64 bits."""

import pytest
import torch

from tests import few_reference as ref
from tests.test_few_tokens_gpu import make, make_module, widths_of

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def weight(K, N, dtype, seed=0, std=0.05):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(K, N, generator=g) * std).to("cuda", dtype)


def spread(scales, group, segments):
    """The scale of every weight, in fp64."""
    gid, base = [], 0
    for n in segments:
        gid += [base + i // group for i in range(n)]
        base += -(-n // group)
    return scales.double()[torch.tensor(gid, device=scales.device)]


def values(codes, scales, group, segments):
    """(q - 8) * scale in fp64."""
    return (codes.double() - 8) * spread(scales, group, segments)


def offsets(segments):
    out = [0]
    for n in segments:
        out.append(out[-1] + n)
    return out


SHAPES = [
    # rows by segment (None: one), columns, group
    ([16], 16, 32), ([64], 64, 64), ([272], 48, 32), ([272], 80, 64), ([272], 144, 128),
    ([48, 16, 144, 128], 208, 32), ([48, 16, 144, 128], 64, 64), ([336, 176, 16, 0, 32], 112, 128),
    ([16] * 256, 32, 64), ([1104], 1008, 128),
]


@pytest.mark.parametrize("segments,N,group", SHAPES)
@pytest.mark.parametrize("dtype,sdtype", [(BF, BF), (HF, HF), (F32, BF), (F32, HF)])
def test_quantize_matches_definition(segments, N, group, dtype, sdtype, device):
    from moe_b200.kernels import dequantize_int4, pack_int4, quantize_int4

    K = sum(segments)
    w = weight(K, N, dtype, seed=K + N)
    w[:, 3] = 0  # a column of zeros
    w[0, 5] = 3.0  # one large value a group
    rows = offsets(segments) if len(segments) > 1 else None
    q = quantize_int4(w, group, row_offsets=rows, dtype=sdtype)
    codes, scales = ref.quantize(w, group, segments, sdtype)
    assert q.shape == (K, N) and q.dtype == sdtype
    assert torch.equal(q.scales, scales)
    back = dequantize_int4(q)
    assert torch.equal(back, values(codes, scales, group, segments).to(sdtype))
    p = pack_int4(codes.to(torch.uint8), scales, group, row_offsets=rows)
    assert torch.equal(p.packed, q.packed)


def test_ties_go_to_even(device):
    from moe_b200.kernels import dequantize_int4, quantize_int4

    # scale 1: 7 is the largest, halves in between
    col = torch.tensor([7.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 6.5, -6.5, 3.5, -3.5, 0.0, 4.5, 5.5,
                        -7.0, -4.5])
    w = col[:, None].expand(16, 16).contiguous()
    for dtype in (BF, HF, F32):
        got = dequantize_int4(quantize_int4(w.to(device, dtype), 32)).float().cpu()
        assert torch.equal(got, torch.round(w))
    # just beside a half, closer than fp32 can divide
    x = torch.tensor([7.0, 2.5 * (1 + 2**-23), 2.5 * (1 - 2**-24), 3.5 * (1 - 2**-24)] * 4)
    w = x[:, None].expand(16, 16).contiguous().to(device)
    got = dequantize_int4(quantize_int4(w, 32)).float().cpu()[:4, 0]
    assert got.tolist() == [7.0, 3.0, 2.0, 3.0]


@pytest.mark.parametrize("dtype", [BF, HF])
def test_not_finite_groups(dtype, device):
    from moe_b200.kernels import dequantize_int4, quantize_int4

    w = weight(128, 32, dtype)
    w[40, 2] = float("nan")
    w[70, 4] = float("inf")
    w[3, 6] = float("-inf")
    back = dequantize_int4(quantize_int4(w, 32))
    bad = torch.zeros(128, 32, dtype=torch.bool, device=device)
    bad[32:64, 2] = bad[64:96, 4] = bad[0:32, 6] = True
    assert torch.equal(torch.isnan(back), bad)


def test_tiny_weights(device):
    """Scales at the bottom of the type: zero, or codes held at the ends."""
    from moe_b200.kernels import dequantize_int4, quantize_int4

    w = torch.full((16, 16), 2.0**-24, device=device, dtype=HF)
    w[3, :] = 2.0**-23
    q = quantize_int4(w, 32)
    codes, scales = ref.quantize(w, 32, [16], HF)
    assert torch.equal(q.scales, scales)
    assert torch.equal(dequantize_int4(q), values(codes, scales, 32, [16]).to(HF))


def test_strided_weight(device):
    from moe_b200.kernels import quantize_int4

    w = weight(64, 96, BF)
    a = quantize_int4(w[:, 16:64].contiguous(), 64)
    for view in (w[:, 16:64], w.t().contiguous().t()[:, 16:64]):
        b = quantize_int4(view, 64)
        assert torch.equal(a.packed, b.packed) and torch.equal(a.scales, b.scales)


def quantized(p, act, group):
    """Int4 weights of make()'s layer, their exact values, and their terms' magnitudes."""
    from moe_b200.kernels import quantize_int4

    gated = 2 if act == "swiglu" else 1
    rows = [o // gated for o in p["off"]]
    q1, q2 = quantize_int4(p["w1"], group), quantize_int4(p["w2"], group, row_offsets=rows)
    seg2 = [b - a for a, b in zip(rows, rows[1:])]
    c1, s1 = ref.quantize(p["w1"], group, [p["w1"].shape[0]], p["w1"].dtype)
    c2, s2 = ref.quantize(p["w2"], group, seg2, p["w2"].dtype)
    seg1, dt = [p["w1"].shape[0]], p["w1"].dtype
    return (q1, q2, values(c1, s1, group, seg1), values(c2, s2, group, seg2),
            ref.int4_terms(spread(s1, group, seg1), dt), ref.int4_terms(spread(s2, group, seg2), dt))


LAYERS = [
    (1, 16, [(1, 16)], 1, True, "relu_squared", BF, 32),
    (1, 768, [(4, 512), (8, 256), (4, 128)], 2, True, "relu_squared", BF, 64),
    (7, 256, [(4, 512), (4, 256)], 2, True, "relu_squared", BF, 128),
    (17, 1104, [(3, 336), (5, 176), (3, 16)], 3, False, "swiglu", HF, 32),
    (64, 272, [(2, 48), (3, 144)], 2, True, "none", HF, 64),
    (33, 528, [(5, 80), (2, 272)], 4, True, "relu_squared", BF, 32),
    (64, 64, [(256, 16)], 9, True, "relu_squared", BF, 128),
    (12, 2048, [(16, 320)], 8, True, "swiglu", BF, 128),
    # final sums shared by several threads, with 64-column tiles
    (2, 272, [(5, 80), (2, 272)], 4, True, "relu_squared", HF, 64),
    (3, 528, [(11, 96)], 5, False, "swiglu", BF, 32),
    (4, 144, [(7, 208)], 3, True, "none", BF, 128),
    (64, 32, [(256, 16)], 32, True, "relu_squared", BF, 32),
    # 128-column tiles: 12800 columns or more
    (1, 256, [(4, 2048), (4, 1616)], 8, True, "relu_squared", BF, 64),
    (2, 528, [(10, 1360)], 5, True, "relu_squared", HF, 32),
    (3, 272, [(5, 2720)], 4, False, "swiglu", HF, 32),
    (4, 1040, [(8, 1616)], 6, True, "swiglu", BF, 128),
    (6, 1104, [(7, 2016)], 3, False, "none", BF, 128),
    (8, 2048, [(20, 1024)], 8, True, "relu_squared", BF, 64),
    (9, 96, [(40, 336)], 5, True, "relu_squared", BF, 64),
    (33, 336, [(7, 2080), (30, 48)], 6, True, "swiglu", HF, 32),
    (64, 528, [(3, 4096), (2, 1040), (1, 16)], 2, True, "relu_squared", BF, 64),
    (64, 64, [(256, 64)], 32, True, "relu_squared", BF, 32),
]


@pytest.mark.parametrize("T,H,sizes,k,norm,act,dtype,group", LAYERS)
def test_layer_on_int4_experts(T, H, sizes, k, norm, act, dtype, group, device):
    from moe_b200.kernels import check_device_status, moe_few_tokens

    p = make(T, H, sizes, dtype, act, seed=4, k=k)
    q1, q2, v1, v2, m1, m2 = quantized(p, act, group)
    off = torch.tensor(p["off"], dtype=torch.int32, device=device)
    out = moe_few_tokens(p["x"], p["router"], q1, q2, off, p["max_width"], k, norm, act)
    r, b = ref.layer(p["x"], p["router"], v1, v2, p["off"], k, norm, act, m1, m2)
    ref.assert_within(out, r, b, "out")
    assert torch.equal(out, moe_few_tokens(p["x"], p["router"], q1, q2, off, p["max_width"], k,
                                           norm, act))
    check_device_status(device)


GROUPED = [
    # counts, slack rows after each expert, H, sizes, act, dtype, group
    ([1], 0, 16, [(1, 16)], "none", BF, 32),
    ([0, 3, 0, 1, 2, 0], 0, 256, [(3, 64), (3, 128)], "relu_squared", BF, 64),
    ([5, 0, 17, 40], 3, 528, [(1, 80), (1, 272), (2, 16)], "none", HF, 32),
    ([9, 8, 16, 1], 2, 272, [(4, 144)], "swiglu", BF, 128),
    ([2] * 64, 0, 2048, [(64, 64)], "relu_squared", BF, 128),
    ([300, 0, 1], 5, 96, [(3, 48)], "relu_squared", HF, 64),
    # 128-column tiles in one direction or both
    ([3] * 20, 0, 768, [(20, 688)], "relu_squared", BF, 64),
    ([0, 1, 11, 2, 30], 3, 2640, [(2, 2608), (3, 1328)], "swiglu", HF, 32),
    ([2, 9] * 8, 0, 1040, [(16, 80)], "none", BF, 128),
    # more units a team than its table holds
    ([32767], 1, 32, [(1, 640)], "none", BF, 32),
    ([3100], 0, 32, [(1, 12800)], "relu_squared", BF, 64),
]


@pytest.mark.parametrize("down", [False, True])
@pytest.mark.parametrize("counts,slack,H,sizes,act,dtype,group", GROUPED)
def test_grouped_products(counts, slack, H, sizes, act, dtype, group, down, device):
    from moe_b200.kernels import (check_device_status, grouped_gemv_down_int4,
                                  grouped_gemv_up_int4)

    if down:
        act = "none"
    p = make(1, H, sizes, dtype, act, seed=5)
    q1, q2, v1, v2, m1, m2 = quantized(p, act, group)
    widths, E, mw = widths_of(sizes), len(counts), p["max_width"]
    start = offsets([c + slack for c in counts])
    rows = start[-1] + 2
    g = torch.Generator(device="cpu").manual_seed(1)
    x = torch.randn(rows, mw if down else H, generator=g).to(device, dtype)
    # columns past an expert's width hold anything
    if down:
        for e, (s, w) in enumerate(zip(start, widths)):
            x[s:start[e + 1], w:] = float("nan")
    i32 = dict(dtype=torch.int32, device=device)
    tok, off = torch.tensor(start, **i32), torch.tensor(p["off"], **i32)
    cnt, wid = torch.tensor(counts, **i32), torch.tensor(widths, **i32)
    if down:
        out = grouped_gemv_down_int4(x, q2, tok, off, wid, cnt, H)
    else:
        out = grouped_gemv_up_int4(x, q1, tok, off, wid, cnt, mw, activation=act)
    r, b = ref.grouped(x, v2 if down else v1, list(zip(start, counts)), p["off"], mw, act, down,
                       m2 if down else m1)
    ref.assert_within(out, r, b, "out")
    if slack == 0:  # without counts: all of an expert's rows
        again = (grouped_gemv_down_int4(x, q2, tok, off, wid, None, H) if down else
                 grouped_gemv_up_int4(x, q1, tok, off, wid, None, mw, activation=act))
        assert torch.equal(out, again)
    check_device_status(device)


def test_products_make_the_layer(device):
    """Routing by the framework's own functions around the two products gives the
    whole layer's result (the intermediate and the rows rounded once each)."""
    from moe_b200.kernels import (fused_route, grouped_gemv_down_int4, grouped_gemv_up_int4,
                                  moe_few_tokens, padded_gather, padded_scatter)
    from moe_b200.kernels._ops import router_topk

    p = make(6, 256, [(4, 128), (4, 64)], BF, seed=8)
    q1, q2, *_ = quantized(p, "relu_squared", 64)
    i32 = dict(dtype=torch.int32, device=device)
    off = torch.tensor(p["off"], **i32)
    wid = torch.tensor([128] * 4 + [64] * 4, **i32)
    w, sel = router_topk(torch.sigmoid(p["x"].float() @ p["router"].float().t()), 2, True, BF)
    bin_ids, indices, tpe, bins, padded = fused_route(sel.reshape(-1), 8, block_size=16)
    tok = torch.cat([torch.zeros(1, **i32), padded])
    xg = padded_gather(p["x"], indices, bin_ids, bins, padded, 2)
    h = grouped_gemv_up_int4(xg, q1, tok, off, wid, tpe, 128)
    y = grouped_gemv_down_int4(h, q2, tok, off, wid, tpe, 256)
    out = padded_scatter(y, indices, bin_ids, w.reshape(-1), bins, padded, 2)
    whole = moe_few_tokens(p["x"], p["router"], q1, q2, off, 128, 2)
    scale = float(whole.abs().max())
    # four roundings of half a bf16 step each against one
    assert float((out - whole).abs().max()) <= 5 * 2.0**-8 * 2 * scale


def test_module_on_int4_experts(device):
    m = make_module([(4, 64), (3, 48)], 128, 2, BF)
    x = torch.randn(2, 3, 128, generator=torch.Generator().manual_seed(2)).to(device, BF)
    with torch.no_grad():
        for group in (32, 64, 128):
            q = m.quantize_experts(group_size=group)
            out = m.decode(x, experts=q)
            seg = [64] * 4 + [48] * 3
            c1, s1 = ref.quantize(m.w1, group, [128], BF)
            c2, s2 = ref.quantize(m.w2, group, seg, BF)
            r, b = ref.layer(x.reshape(-1, 128), m.router.weight, values(c1, s1, group, [128]),
                             values(c2, s2, group, seg), m.expert_offsets, 2, True, "relu_squared",
                             ref.int4_terms(spread(s1, group, [128]), BF),
                             ref.int4_terms(spread(s2, group, seg), BF))
            ref.assert_within(out.reshape(-1, 128), r, b, f"group {group}")


def test_grouped_offsets_that_do_not_fit(device):
    from moe_b200._lib import MoEKernelError
    from moe_b200.kernels import check_device_status, grouped_gemv_up_int4

    p = make(1, 64, [(2, 32)], BF)
    q1, *_ = quantized(p, "none", 32)
    i32 = dict(dtype=torch.int32, device=device)
    x = torch.randn(4, 64, device=device, dtype=BF)
    off, wid = torch.tensor([0, 32, 64], **i32), torch.tensor([32, 32], **i32)
    good = grouped_gemv_up_int4(x, q1, torch.tensor([0, 2, 4], **i32), off, wid, None, 32, "none")
    for tok, o in [([0, 2, 5], off), ([0, 3, 2], off), ([-1, 2, 4], off),
                   ([0, 2, 4], torch.tensor([0, 32, 80], **i32)),
                   ([0, 2, 4], torch.tensor([0, 32, 56], **i32))]:
        out = grouped_gemv_up_int4(x, q1, torch.tensor(tok, **i32), o, wid, None, 32, "none")
        assert torch.isfinite(out.float()).all()
        with pytest.raises(MoEKernelError):
            check_device_status(device)
    check_device_status(device)
    assert good.shape == (4, 32)


def test_layer_offsets_that_do_not_fit_the_packed_weight(device):
    """w2 packed for other experts than the offsets name: those beyond its blocks add
    nothing and set the status word."""
    from moe_b200._lib import MoEKernelError
    from moe_b200.kernels import check_device_status, moe_few_tokens, quantize_int4

    p = make(5, 64, [(4, 32)], BF)
    q1, q2, *_ = quantized(p, "relu_squared", 32)
    off = torch.tensor(p["off"], dtype=torch.int32, device=device)
    whole = moe_few_tokens(p["x"], p["router"], q1, q2, off, 32, 4)
    check_device_status(device)
    # two block rows where the offsets need four
    other = quantize_int4(p["w2"], 32, row_offsets=[0, 64, 128, 128, 128])
    out = moe_few_tokens(p["x"], p["router"], q1, other, off, 32, 4)
    with pytest.raises(MoEKernelError):
        check_device_status(device)
    assert bool(torch.isfinite(out).all())
    assert torch.equal(whole, moe_few_tokens(p["x"], p["router"], q1, q2, off, 32, 4))
    check_device_status(device)


@pytest.mark.parametrize("T", [5, 12])
def test_not_finite_tokens_reach_no_other(T, device):
    from moe_b200.kernels import moe_few_tokens

    p = make(T, 128, [(8, 64)], BF, seed=2)
    q1, q2, *_ = quantized(p, "relu_squared", 64)
    off = torch.tensor(p["off"], dtype=torch.int32, device=device)
    clean = moe_few_tokens(p["x"], p["router"], q1, q2, off, 64, 3)
    x = p["x"].clone()
    x[1, 7], x[3, 100] = float("nan"), float("inf")
    out = moe_few_tokens(x, p["router"], q1, q2, off, 64, 3)
    assert bool(torch.isnan(out[1]).all())
    # (the others' experts may share passes otherwise than before: within a rounding)
    keep = [t for t in range(T) if t not in (1, 3)]
    d = (out[keep].float() - clean[keep].float()).abs()
    assert bool((d <= 2 * 2.0**-8 * clean[keep].float().abs().amax()).all())


def test_offsets_of_other_types_and_strides(device):
    from moe_b200.kernels import grouped_gemv_up_int4, moe_few_tokens

    p = make(6, 64, [(4, 32)], BF)
    q1, q2, *_ = quantized(p, "relu_squared", 32)
    i32 = dict(dtype=torch.int32, device=device)
    off, tok = torch.tensor(p["off"], **i32), torch.tensor([0, 2, 2, 5, 6], **i32)
    wid = torch.tensor([32] * 4, **i32)
    apart = torch.stack([off, off], 1)[:, 0]
    layer = moe_few_tokens(p["x"], p["router"], q1, q2, off, 32, 2)
    up = grouped_gemv_up_int4(p["x"], q1, tok, off, wid, None, 32)
    for o in (off.long(), apart):
        assert torch.equal(layer, moe_few_tokens(p["x"], p["router"], q1, q2, o, 32, 2))
        assert torch.equal(up, grouped_gemv_up_int4(p["x"], q1, tok.long(), o, wid, None, 32))


def test_graph_capture_of_products(device):
    from moe_b200.kernels import grouped_gemv_up_int4

    p = make(1, 256, [(4, 128)], BF)
    q1, *_ = quantized(p, "relu_squared", 64)
    i32 = dict(dtype=torch.int32, device=device)
    tok, off = torch.tensor([0, 2, 2, 3, 5], **i32), torch.tensor(p["off"], **i32)
    wid = torch.tensor([128] * 4, **i32)
    x = torch.randn(5, 256, device=device, dtype=BF)
    grouped_gemv_up_int4(x, q1, tok, off, wid, None, 128)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = grouped_gemv_up_int4(x, q1, tok, off, wid, None, 128)
    x.copy_(torch.randn(5, 256, device=device, dtype=BF))
    graph.replay()
    assert torch.equal(y, grouped_gemv_up_int4(x, q1, tok, off, wid, None, 128))


def test_refusals(device):
    from moe_b200.kernels import (Int4Weight, grouped_gemv_down_int4, grouped_gemv_up_int4,
                                  moe_few_tokens, pack_int4, quantize_int4)

    w = weight(64, 64, BF)
    for bad in (dict(group_size=16), dict(group_size=48), dict(row_offsets=[0, 32]),
                dict(row_offsets=[0, 24, 64]), dict(row_offsets=[0, 48, 32, 64]),
                dict(row_offsets=[16, 64]), dict(row_offsets=[0]), dict(row_offsets=[0, 2**40])):
        with pytest.raises(ValueError):
            quantize_int4(w, **bad)
    with pytest.raises(ValueError):
        quantize_int4(w[:24], 32)
    with pytest.raises(ValueError):
        quantize_int4(w[:, :24], 32)
    with pytest.raises(ValueError):
        quantize_int4(w.cpu(), 32)
    with pytest.raises(TypeError):
        quantize_int4(w, 32, dtype=HF)
    with pytest.raises(TypeError):
        quantize_int4(w.double(), 32)
    with pytest.raises(TypeError):
        quantize_int4(w, 32, row_offsets=torch.tensor([0, 64], device=device))
    q = quantize_int4(w, 32)
    with pytest.raises(ValueError):
        pack_int4(torch.zeros(64, 64, dtype=torch.uint8, device=device), q.scales[:1], 32)
    with pytest.raises(TypeError):
        pack_int4(torch.zeros(64, 64, dtype=torch.int32, device=device), q.scales, 32)
    with pytest.raises(ValueError):
        Int4Weight(q.packed[:, :2], q.scales, 64, 64, 32)
    with pytest.raises(TypeError):
        Int4Weight(q.packed, q.scales.float(), 64, 64, 32)
    p = make(2, 64, [(4, 32)], BF)
    q1, q2, *_ = quantized(p, "none", 32)
    off = torch.tensor(p["off"], dtype=torch.int32, device=device)

    def layer(a, b, x=p["x"]):
        return moe_few_tokens(x, p["router"], a, b, off, 32, 2)

    with pytest.raises(TypeError):
        layer(q1, p["w2"])
    with pytest.raises(TypeError):
        layer(q1, q2, p["x"].half())
    with pytest.raises(ValueError):  # w2 without its experts' offsets
        layer(q1, quantize_int4(p["w2"], 32))
    with pytest.raises(ValueError):  # two group sizes
        layer(q1, quantize_int4(p["w2"], 64, row_offsets=p["off"]))
    with pytest.raises(ValueError):
        layer(q2, q2)
    tok = torch.tensor([0, 1, 1, 2, 2], dtype=torch.int32, device=device)
    wid = torch.tensor([32] * 4, dtype=torch.int32, device=device)
    with pytest.raises(TypeError):
        grouped_gemv_up_int4(p["x"], p["w1"], tok, off, wid, None, 32)
    with pytest.raises(ValueError):
        grouped_gemv_up_int4(p["x"][:, :32], q1, tok, off, wid, None, 32)
    with pytest.raises(ValueError):
        grouped_gemv_up_int4(p["x"], q1, tok[:-1], off, wid, None, 32)
    with pytest.raises(ValueError):
        grouped_gemv_down_int4(p["x"][:, :32], quantize_int4(p["w2"], 32), tok, off, wid, None, 64)
    with pytest.raises(ValueError):
        grouped_gemv_down_int4(p["x"][:, :32], q2, tok, off, wid, None, 48)
    with pytest.raises(RuntimeError, match="no_grad"):
        grouped_gemv_up_int4(p["x"].clone().requires_grad_(), q1, tok, off, wid, None, 32)
