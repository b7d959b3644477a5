"""The MoE layer for a few tokens (moe_few_tokens, TritonMoEMLP.decode) against the
layer's definition in 64 bits, at the sizes and inputs where it can go wrong."""

import pytest
import torch

from tests import few_reference as ref

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def widths_of(sizes):
    return [w for c, w in sizes for _ in range(c)]


def make(T, H, sizes, dtype, act="relu_squared", seed=0, device="cuda", k=None):
    """Inputs of the seed, or, given k, of the first seed from it without a near tie."""
    while True:
        p = _make(T, H, sizes, dtype, act, seed, device)
        if k is None or ref.clear_choice(p["x"], p["router"], k):
            return p
        seed += 100


def _make(T, H, sizes, dtype, act, seed, device):
    g = torch.Generator(device="cpu").manual_seed(seed)
    gated = 2 if act == "swiglu" else 1
    widths = widths_of(sizes)
    off = [0]
    for w in widths:
        off.append(off[-1] + gated * w)
    E = len(widths)

    def rnd(*shape, std=1.0):
        return (torch.randn(*shape, generator=g) * std).to(device, dtype)

    return dict(x=rnd(T, H), router=rnd(E, H, std=H**-0.5), w1=rnd(H, off[-1], std=H**-0.5),
                w2=rnd(off[-1] // gated, H, std=0.05), off=off, max_width=max(widths))


def call(p, k, norm=True, act="relu_squared", **kw):
    from moe_b200.kernels import moe_few_tokens

    p = {**p, **kw}
    off = torch.tensor(p["off"], dtype=torch.int32, device=p["x"].device)
    return moe_few_tokens(p["x"], p["router"], p["w1"], p["w2"], off, p["max_width"], k,
                          norm_topk_prob=norm, activation=act)


def want(p, k, norm=True, act="relu_squared"):
    return ref.layer(p["x"], p["router"], p["w1"], p["w2"], p["off"], k, norm, act)


CASES = [
    # T, H, sizes, k, norm, act, dtype
    (1, 16, [(1, 16)], 1, True, "relu_squared", BF),
    (1, 64, [(4, 32)], 2, True, "relu_squared", BF),
    (1, 768, [(4, 512), (8, 256), (4, 128)], 2, True, "relu_squared", BF),
    (3, 768, [(4, 512), (8, 256), (4, 128)], 4, False, "relu_squared", BF),
    (8, 256, [(4, 512), (4, 256)], 2, True, "relu_squared", BF),
    (9, 256, [(4, 512), (4, 256)], 2, True, "relu_squared", BF),
    (17, 1104, [(3, 336), (5, 176), (3, 16)], 3, False, "swiglu", HF),
    (64, 272, [(2, 48)], 1, True, "relu_squared", BF),
    (63, 528, [(1, 80), (2, 272)], 3, True, "none", HF),
    (64, 128, [(17, 64)], 8, True, "relu_squared", BF),
    (33, 64, [(256, 16)], 32, True, "relu_squared", HF),
    (5, 2048, [(64, 128)], 8, True, "relu_squared", BF),
    (2, 4096, [(5, 80)], 2, True, "swiglu", BF),
    (16, 48, [(31, 16)], 7, True, "swiglu", BF),
    (1, 256, [(4, 512), (4, 256)], 2, True, "relu_squared", F32),
    (3, 256, [(4, 512), (4, 256)], 2, True, "swiglu", F32),
    (11, 80, [(3, 48), (2, 144)], 2, False, "relu_squared", F32),
    (64, 272, [(33, 16)], 5, True, "none", F32),
    (64, 1024, [(2, 1040)], 2, True, "relu_squared", F32),
    (64, 64, [(256, 16)], 32, True, "relu_squared", BF),
    (64, 32, [(256, 16)], 32, True, "relu_squared", F32),
    # more units a team than its table holds
    (64, 16, [(80, 32768)], 8, True, "relu_squared", BF),
]


@pytest.mark.parametrize("T,H,sizes,k,norm,act,dtype", CASES)
def test_matches_definition(T, H, sizes, k, norm, act, dtype, device):
    p = make(T, H, sizes, dtype, act, seed=3, k=k)
    out = call(p, k, norm, act)
    assert out.shape == (T, H) and out.dtype == dtype
    r, b = want(p, k, norm, act)
    ref.assert_within(out, r, b, "out")
    from moe_b200.kernels import check_device_status

    check_device_status(device)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_same_bits_every_time(dtype, device):
    p = make(24, 512, [(8, 256), (8, 128)], dtype)
    a = call(p, 4)
    for _ in range(5):
        assert torch.equal(call(p, 4), a)


def test_no_tokens(device):
    p = make(4, 64, [(4, 32)], BF)
    assert call(p, 2, x=p["x"][:0]).shape == (0, 64)


def test_token_does_not_depend_on_the_batch_it_is_in(device):
    """Up to 8 tokens run the same arithmetic per token: only the slicing of the sums
    may change, so compare each within its bound."""
    p = make(8, 256, [(4, 512), (4, 256)], BF)
    r, b = want(p, 2)
    for t in range(8):
        ref.assert_within(call(p, 2, x=p["x"][t:t + 1]), r[t:t + 1], b[t:t + 1], f"token {t}")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strided_and_unaligned_tokens(dtype, device):
    p = make(6, 128, [(6, 64)], dtype)
    a = call(p, 2)
    wide = torch.full((6, 256), float("nan"), dtype=dtype, device=device)
    wide[:, 64:192] = p["x"]
    assert torch.equal(call(p, 2, x=wide[:, 64:192]), a)  # aligned rows, a stride
    odd = torch.full((6 * 131 + 1,), float("nan"), dtype=dtype, device=device)
    view = odd[1:].view(6, 131)[:, :128]
    view.copy_(p["x"])
    assert torch.equal(call(p, 2, x=view), a)  # no row on 16 bytes
    assert torch.equal(call(p, 2, x=p["x"].t().contiguous().t()), a)  # columns first
    one = p["x"][:1].expand(6, 128)
    assert torch.equal(call(p, 2, x=one), call(p, 2, x=one.contiguous()))


def test_equal_logits_go_to_the_lower_expert(device):
    p = make(3, 64, [(8, 32)], BF)
    p["router"].zero_()
    r, b = want(p, 3)  # all logits 0: experts 0, 1, 2
    ref.assert_within(call(p, 3), r, b, "out")


def test_close_logits_are_told_apart(device):
    """Two logits that differ by less than a bf16 step."""
    H = 64
    p = make(1, H, [(4, 32)], BF)
    p["x"].fill_(0)
    p["x"][0, :2] = 1.0
    p["router"].zero_()
    p["router"][:, 0] = torch.tensor([0.25, 1.0, 1.0, 0.5], device=device)
    p["router"][2, 1] = 2.0**-12
    r, b = want(p, 1)
    ref.assert_within(call(p, 1), r, b, "out")


def test_nan_and_infinity_stay_where_they_are(device):
    p = make(6, 128, [(8, 64)], BF)
    clean = call(p, 2)
    sel, _ = ref.choose(p["x"], p["router"], 2)
    # an expert that no token chose may hold anything
    free = sorted(set(range(8)) - set(sel.flatten().tolist()))
    q = make(1, 128, [(8, 64)], BF)
    sel1, _ = ref.choose(q["x"], q["router"], 2)
    free1 = sorted(set(range(8)) - set(sel1.flatten().tolist()))
    one = call(q, 2)
    for e in free1:
        q["w1"][:, 64 * e:64 * e + 64] = float("nan")
        q["w2"][64 * e:64 * e + 64] = float("inf")
    assert torch.equal(call(q, 2), one)
    for e in free:
        p["w1"][:, 64 * e:64 * e + 64] = float("nan")
    assert torch.equal(call(p, 2), clean)
    # tokens that share an expert with others do not see its other tokens' values
    bad = p["x"].clone()
    bad[2, 5] = float("nan")
    out = call(p, 2, x=bad)
    keep = [0, 1, 3, 4, 5]
    assert torch.isnan(out[2]).all()
    r, b = want({**p, "w1": p["w1"].nan_to_num(0)}, 2)
    ref.assert_within(out[keep], r[keep], b[keep], "other tokens")


def test_nan_weight_of_a_chosen_expert_reaches_only_its_tokens(device):
    p = make(6, 128, [(8, 64)], BF, seed=1)
    sel, _ = ref.choose(p["x"], p["router"], 2)
    e = int(sel[0, 0])
    hit = (sel == e).any(1)
    clean = call(p, 2)
    p["w2"][64 * e + 3, :] = float("nan")
    out = call(p, 2)
    assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])


def test_nan_router_row_is_chosen_first(device):
    """torch.topk's order: NaN above all numbers; the token's weights become NaN."""
    p = make(2, 64, [(4, 32)], BF)
    p["router"][3] = float("nan")
    assert torch.isnan(call(p, 2)).all()


def test_huge_and_tiny_logits(device):
    p = make(4, 64, [(8, 32)], F32)
    p["router"] *= 200.0
    r, b = want(p, 3)
    ref.assert_within(call(p, 3), r, b, "out")


def test_experts_without_columns(device):
    p = make(5, 64, [(6, 32)], BF)
    off = [0, 32, 32, 64, 96, 128, 192]
    p.update(off=off, max_width=64)
    r, b = want(p, 6)
    ref.assert_within(call(p, 6), r, b, "out")
    p.update(off=[0] * 7)
    assert torch.equal(call(p, 6), torch.zeros_like(p["x"]))


@pytest.mark.parametrize("off", [[0, 32, 60, 96, 128], [0, 32, 64, 96, 144], [0, 96, 64, 96, 128],
                                 [-16, 32, 64, 96, 128], [0, 32, 128, 128, 128]])
def test_offsets_that_do_not_fit_set_the_status(off, device):
    from moe_b200._lib import MoEKernelError
    from moe_b200.kernels import check_device_status

    p = make(3, 64, [(4, 32)], BF)
    out = call(p, 4, off=off)
    assert torch.isfinite(out.float()).all()
    with pytest.raises(MoEKernelError):
        check_device_status(device)
    check_device_status(device)


def test_graph_capture_and_replay(device):
    from moe_b200.kernels import moe_few_tokens

    p = make(4, 256, [(8, 128)], BF)
    off = torch.tensor(p["off"], dtype=torch.int32, device=device)
    x = p["x"].clone()

    def step(x):
        return moe_few_tokens(x, p["router"], p["w1"], p["w2"], off, p["max_width"], 2)

    step(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y1 = step(x)
        y2 = step(y1)
    for seed in (5, 6):
        x.copy_(make(4, 256, [(8, 128)], BF, seed=seed)["x"])
        graph.replay()
        a = step(x.clone())
        assert torch.equal(y1, a) and torch.equal(y2, step(a))


def test_two_graphs_replayed_together(device):
    p = make(4, 512, [(8, 256)], BF)
    q = make(7, 512, [(8, 256)], BF, seed=9)
    wp, wq = call(p, 2), call(q, 2)
    off = torch.tensor(p["off"], dtype=torch.int32, device=device)
    from moe_b200.kernels import moe_few_tokens

    graphs = []
    for d in (p, q):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = moe_few_tokens(d["x"], d["router"], d["w1"], d["w2"], off, d["max_width"], 2)
        graphs.append((g, y, torch.cuda.Stream()))
    for _ in range(20):
        for g, _y, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], wp) and torch.equal(graphs[1][1], wq)


def test_two_streams(device):
    p = make(4, 512, [(8, 256)], BF)
    q = make(40, 512, [(8, 256)], BF, seed=9)
    wp, wq = call(p, 2), call(q, 2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            got.append((call(p, 2), wp))
        with torch.cuda.stream(s2):
            got.append((call(q, 2), wq))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, b)


def make_module(sizes, H, k, dtype, norm=True, block=16, device="cuda"):
    from moe_b200 import TritonMoEConfig, TritonMoEMLP

    torch.manual_seed(0)
    m = TritonMoEMLP(TritonMoEConfig(n_embd=H, expert_sizes=sizes, num_active_experts=k,
                                     norm_topk_prob=norm, block_size=block))
    with torch.no_grad():
        m.router.weight.normal_(0, H**-0.5)
        m.w1.normal_(0, H**-0.5)
        m.w2.normal_(0, 0.05)
    return m.to(device=device, dtype=dtype)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_module_decode(dtype, device):
    m = make_module([(4, 64), (3, 48)], 128, 2, dtype)
    x = torch.randn(3, 5, 128, generator=torch.Generator().manual_seed(1)).to(device, dtype)
    with torch.no_grad():
        out = m.decode(x)
        fwd, _, _ = m(x)
    assert out.shape == x.shape and out.dtype == dtype
    r, b = ref.layer(x.reshape(-1, 128), m.router.weight, m.w1, m.w2, m.expert_offsets, 2, True,
                     "relu_squared")
    ref.assert_within(out.reshape(-1, 128), r.detach(), b.detach(), "decode")
    # forward rounds logits, weights and the intermediate (fp32: tf32 products) once each
    scale = float(fwd.abs().max())
    assert float((out - fwd).abs().max()) <= 3e-2 * scale
    with torch.no_grad():
        assert torch.equal(m.decode(x[0, 0]), m.decode(x[:1, :1])[0, 0])


def test_decode_step_after_step(device):
    """Tokens through two layers, then 4-bit experts of the second: as a decode loop
    runs them, on one stream with nothing between."""
    a, b = make_module([(8, 64)], 256, 2, BF), make_module([(4, 128)], 256, 2, BF)
    with torch.no_grad():
        q = b.quantize_experts(group_size=64)
        x = torch.randn(2, 1, 256, device=device, dtype=BF)
        outs = []
        for _ in range(4):
            x = x + b.decode(x + a.decode(x), experts=q)
            outs.append(x)
        y = outs[0].clone()
        for want_ in outs[1:]:
            y = y + b.decode(y + a.decode(y), experts=q)
            assert torch.equal(y, want_)
    assert torch.isfinite(outs[-1].float()).all()


def test_refuses_gradients_and_wrong_arguments(device):
    m = make_module([(4, 64)], 128, 2, BF)
    x = torch.randn(2, 1, 128, device=device, dtype=BF)
    with pytest.raises(RuntimeError, match="no_grad"):
        m.decode(x)
    with torch.no_grad():
        with pytest.raises(ValueError, match="64 tokens"):
            m.decode(x[:1].expand(65, 1, 128))
        with pytest.raises(TypeError, match="dtype"):
            m.decode(x.float())
    p = make(2, 64, [(4, 32)], BF)
    for bad, err in [
        (dict(x=p["x"].cpu()), ValueError), (dict(router=p["router"][:, :32]), ValueError),
        (dict(w1=p["w1"][:, ::2]), ValueError), (dict(w2=p["w2"][:64]), ValueError),
        (dict(w1=p["w1"].t().contiguous().t()), ValueError), (dict(off=p["off"][:-1]), ValueError),
        (dict(max_width=24), ValueError), (dict(max_width=0), ValueError),
        (dict(w1=p["w1"].half()), TypeError), (dict(x=p["x"].double()), TypeError),
        (dict(x=p["x"][0]), ValueError),
    ]:
        with pytest.raises(err):
            call(p, 2, **bad)
    for k in (0, 5, 33):
        with pytest.raises(ValueError):
            call(p, k)
    with pytest.raises(NotImplementedError):
        call(p, 2, act="gelu")
    w = torch.empty(64 * 128 + 4, dtype=BF, device=device)[4:].view(64, 128)
    with pytest.raises(ValueError, match="aligned"):
        call(p, 2, w1=w)
