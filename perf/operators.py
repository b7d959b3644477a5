"""Workloads of the few-token (serving) operators.

Four operators, each with a plain form in elementary torch operations:

  layer          the whole MoE layer for up to 64 tokens, dense experts
  layer_int4     the same with 4-bit expert weights and group scales
  grouped_int4   the up or down product of the experts' 4-bit weights over rows
                 grouped by expert
  quantize       rounding weights to 4 bits with group scales, and back

A case names the sizes; `prepare` makes the tensors a program holds before the
call, `run` is one call, `exact` is the definition in 64 bits.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_PACKAGE = str(Path(__file__).resolve().parent.parent / "triton-variable-moe_b200")


def _kernels():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from moe_b200 import kernels

    return kernels


def _widths(case):
    """"4x512+8x256" -> [512] * 4 + [256] * 8."""
    return [int(w) for part in case["experts"].split("+")
            for c, w in [part.split("x")] for _ in range(int(c))]


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a chat through a small variable-width layer (latency only)
        dict(name="layer_1tok_h768", op="layer", dtype="bf16", tokens=1, hidden=768,
             experts="4x512+8x256+4x128", top_k=2, norm=True, activation="relu_squared"),
        # an odd small batch through a fine-grained layer
        dict(name="layer_5tok_h2048", op="layer", dtype="bf16", tokens=5, hidden=2048,
             experts="64x1024", top_k=8, norm=True, activation="relu_squared"),
        # the largest: a full decode batch that touches nearly all experts
        dict(name="layer_64tok_h4096", op="layer", dtype="bf16", tokens=64, hidden=4096,
             experts="32x2048+64x1024+32x512", top_k=8, norm=True, activation="relu_squared"),
        # ragged widths (odd multiples of 16), gated activation, raw router weights
        dict(name="layer_17tok_ragged", op="layer", dtype="fp16", tokens=17, hidden=1104,
             experts="3x336+5x176+3x16", top_k=3, norm=False, activation="swiglu"),
        # a full-precision layer, as in numerical checks of a deployment
        dict(name="layer_3tok_fp32", op="layer", dtype="fp32", tokens=3, hidden=256,
             experts="4x512+4x256", top_k=2, norm=True, activation="relu_squared"),
        # one token through 4-bit experts: the interactive case of a quantised layer
        dict(name="layer_int4_1tok_h4096", op="layer_int4", dtype="bf16", tokens=1, hidden=4096,
             experts="32x2048+64x1024+32x512", top_k=8, norm=True, activation="relu_squared",
             group=128),
        # a decode batch through 4-bit experts
        dict(name="layer_int4_33tok_h2048", op="layer_int4", dtype="bf16", tokens=33, hidden=2048,
             experts="64x1024", top_k=8, norm=True, activation="relu_squared", group=64),
        # ragged widths and a last group shorter than the others
        dict(name="layer_int4_6tok_ragged", op="layer_int4", dtype="fp16", tokens=6, hidden=1104,
             experts="3x336+5x176+3x16", top_k=3, norm=False, activation="swiglu", group=32),
        # the products alone, for programs that route by themselves
        dict(name="up_int4_3tok_h768", op="grouped_int4", dtype="bf16", tokens=3, hidden=768,
             experts="4x512+8x256+4x128", top_k=2, activation="relu_squared", group=64,
             direction="up"),
        dict(name="down_int4_24tok_h2048", op="grouped_int4", dtype="bf16", tokens=24,
             hidden=2048, experts="64x1024", top_k=8, activation="none", group=128,
             direction="down"),
        # quantising a small layer's down weights (a group never spans two experts)
        dict(name="quantize_h768", op="quantize", dtype="bf16", hidden=768,
             experts="4x512+8x256+4x128", group=64, direction="down"),
        # quantising a whole layer's up weights at load time
        dict(name="quantize_h2048", op="quantize", dtype="bf16", hidden=2048, experts="64x1024",
             group=128, direction="up"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layer", "layer", "layer_int4", "layer_int4", "grouped_int4", "quantize"])
    while True:
        hidden = 16 * _log_int(rng, 8, 256)
        parts = []
        for _ in range(rng.randint(1, 3)):
            parts.append((_log_int(rng, 1, 48), 16 * _log_int(rng, 1, 128)))
        total = sum(c * w for c, w in parts)
        # at most about 200 M weights a matrix
        if sum(c for c, _ in parts) >= 2 and total * hidden <= 200e6:
            break
    experts = "+".join(f"{c}x{w}" for c, w in parts)
    num = sum(c for c, _ in parts)
    case = dict(op=op, hidden=hidden, experts=experts)
    if op == "quantize":
        return dict(case, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    group=rng.choice([32, 64, 128]), direction=rng.choice(["up", "down"]))
    case["tokens"] = _log_int(rng, 1, 64)
    case["top_k"] = min(rng.randint(1, 8), num)
    case["activation"] = rng.choice(["relu_squared", "relu_squared", "swiglu", "none"])
    if op == "layer":
        return dict(case, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    norm=rng.random() < 0.7)
    case["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
    case["group"] = rng.choice([32, 64, 128])
    if op == "layer_int4":
        return dict(case, norm=rng.random() < 0.7)
    case["direction"] = rng.choice(["up", "down"])
    if case["direction"] == "down" or case["activation"] == "swiglu":
        case["activation"] = "none" if case["direction"] == "down" else "relu_squared"
    return case


# -------------------------------------------------------------------- inputs
def _group_ids(segments, group):
    """The group of every row: groups of `group` rows start anew in each segment."""
    ids, base = [], 0
    for n in segments:
        ids += [base + i // group for i in range(n)]
        base += -(-n // group)
    return torch.tensor(ids, dtype=torch.int64, device="cuda"), base


def _int4(gen, rows, cols, segments, group, std, dtype):
    """Random codes [rows, cols] in 0..15 and scales [groups, cols] of a weight
    of about the given standard deviation."""
    gid, groups = _group_ids(segments, group)
    codes = torch.randint(0, 16, (rows, cols), dtype=torch.uint8, device="cuda", generator=gen)
    scales = torch.rand(groups, cols, device="cuda", generator=gen) * 0.5 + 0.75
    return codes, (scales * (std / 4.6)).to(dtype), gid


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _DTYPES[case["dtype"]]
    widths = _widths(case)
    hidden, num = case["hidden"], len(widths)
    st = {"case": case, "max_width": max(widths)}

    def normal(*shape, std=1.0):
        return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0, std, generator=gen)

    offsets = [0]
    for w in widths:
        offsets.append(offsets[-1] + w)
    total = offsets[-1]
    if case["op"] == "quantize":
        up = case["direction"] == "up"
        st["w"] = normal(*((hidden, total) if up else (total, hidden)), std=0.02)
        st["row_offsets"] = None if up else offsets
        st["gid"], st["groups"] = _group_ids([hidden] if up else widths, case["group"])
        return st

    gated = 2 if case["activation"] == "swiglu" else 1
    st["off"] = torch.tensor([gated * o for o in offsets], dtype=torch.int32, device="cuda")
    st["widths"] = torch.tensor(widths, dtype=torch.int32, device="cuda")
    # a weight scale that keeps activations near one at any hidden size
    std1, std2 = 1.0 / math.sqrt(hidden), 0.02
    if case["op"] == "grouped_int4":
        T, k = case["tokens"], case["top_k"]
        choice = torch.rand(T, num, device="cuda", generator=gen).argsort(1)[:, :k].reshape(-1)
        counts = torch.bincount(choice, minlength=num)
        st["row_expert"] = torch.sort(choice).values
        st["counts"] = counts.to(torch.int32)
        st["tok_off"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        if case["direction"] == "up":
            st["x"] = normal(T * k, hidden)
            weight = _int4(gen, hidden, total, [hidden], case["group"], std1, dtype)
            rows = None
        else:
            st["x"] = normal(T * k, st["max_width"])
            weight = _int4(gen, total, hidden, widths, case["group"], std2, dtype)
            rows = offsets
        if own:
            st["q"] = _kernels().pack_int4(weight[0], weight[1], case["group"], row_offsets=rows)
        else:
            st["weight"] = weight
        return st

    st["x"] = normal(case["tokens"], hidden)
    st["router"] = normal(num, hidden, std=1.0 / math.sqrt(hidden))
    if case["op"] == "layer":
        st["w1"] = normal(hidden, gated * total, std=std1)
        st["w2"] = normal(total, hidden, std=std2)
        return st
    c1 = _int4(gen, hidden, gated * total, [hidden], case["group"], std1, dtype)
    if own:
        st["w1"] = _kernels().pack_int4(c1[0], c1[1], case["group"])
        del c1
    else:
        st["c1"] = c1
    c2 = _int4(gen, total, hidden, widths, case["group"], std2, dtype)
    if own:
        st["w2"] = _kernels().pack_int4(c2[0], c2[1], case["group"], row_offsets=offsets)
    else:
        st["c2"] = c2
    return st


# --------------------------------------------------------------- plain forms
def _values(weight):
    codes, scales, gid = weight
    return (codes.float() - 8.0) * scales.float()[gid]


def _select(x, router, k, norm):
    """(experts [T, k], weights [T, k]): the k largest logits, in 64 bits since
    neighbouring logits decide which expert runs."""
    logits = x.double() @ router.double().t()
    top, sel = torch.sort(logits, dim=1, descending=True, stable=True)
    p = 1.0 / (1.0 + torch.exp(-top[:, :k]))
    if norm:
        p = p / (p.sum(1, keepdim=True) + 1e-20)
    return sel[:, :k], p.float()


def _activate(u, activation, gate=None):
    if activation == "relu_squared":
        return torch.clamp(u, min=0).square()
    if activation == "swiglu":
        return gate / (1.0 + torch.exp(-gate)) * u
    return u


def _columns(first, widths, max_width):
    """Column indices [rows, max_width] of each row's expert, and which are real."""
    j = torch.arange(max_width, device=first.device)
    real = j[None, :] < widths[:, None]
    return torch.where(real, first[:, None] + j[None, :], 0), real


def _row_products(x, w, cols):
    """x[r] @ w[:, cols[r]] -> [rows, max_width].  Few rows: the columns of each
    row are picked out first; many: all products, then the pick."""
    if 2 * cols.numel() <= w.shape[1]:
        picked = w[:, cols.reshape(-1)].float().reshape(w.shape[0], *cols.shape)
        return torch.einsum("rh,hrj->rj", x.float(), picked)
    return torch.gather(x.float() @ w.float(), 1, cols)


def _row_products_down(h, w, cols, real):
    """sum_j h[r, j] w[cols[r, j]] -> [rows, hidden]."""
    h = torch.where(real, h, 0.0)
    if 2 * cols.numel() <= w.shape[0]:
        picked = w[cols.reshape(-1)].float().reshape(*cols.shape, w.shape[1])
        return torch.einsum("rj,rjn->rn", h, picked)
    wide = torch.zeros(h.shape[0], w.shape[0], device=h.device)
    return wide.scatter_add_(1, cols, h) @ w.float()


def _plain_layer(st, w1, w2):
    case, x = st["case"], st["x"]
    T, k, act = case["tokens"], case["top_k"], case["activation"]
    gated = 2 if act == "swiglu" else 1
    sel, p = _select(x, st["router"], k, case["norm"])
    e = sel.reshape(-1)
    width = st["widths"].long()[e]
    first = st["off"].long()[e]
    cols, real = _columns(first, width, st["max_width"])
    xr = x[torch.arange(T * k, device=x.device) // k]
    if gated == 2:
        gate = _row_products(xr, w1, cols)
        cols_up = torch.where(real, cols + width[:, None], 0)
        h = _activate(_row_products(xr, w1, cols_up), act, gate)
    else:
        h = _activate(_row_products(xr, w1, cols), act)
    cols2, _ = _columns(first // gated, width, st["max_width"])
    y = _row_products_down(h, w2, cols2, real)
    return (y.reshape(T, k, -1) * p[:, :, None]).sum(1).to(x.dtype)


def _plain_grouped(st):
    case, x = st["case"], st["x"]
    e = st["row_expert"]
    cols, real = _columns(st["off"].long()[e], st["widths"].long()[e], st["max_width"])
    w = _values(st["weight"])
    if case["direction"] == "up":
        u = _row_products(x, w, cols)
        return torch.where(real, _activate(u, case["activation"]), 0.0).to(x.dtype)
    return _row_products_down(x.float(), w, cols, real).to(x.dtype)


def _plain_quantize(st):
    w, gid = st["w"], st["gid"]
    scale_dtype = torch.bfloat16 if w.dtype == torch.float32 else w.dtype
    amax = torch.zeros(st["groups"], w.shape[1], device=w.device)
    amax.index_reduce_(0, gid, w.float().abs(), "amax")
    scale = (amax / 7.0).to(scale_dtype).float()[gid]
    q = torch.round(w.double() / scale.double()).clamp(-8, 7)  # 64 bits: quotients near a half
    q = torch.where(scale > 0, q, 0.0)
    return (q.float() * scale).to(scale_dtype)


def run(state):
    case, op = state["case"], state["case"]["op"]
    if not own:
        if op == "layer":
            return _plain_layer(state, state["w1"], state["w2"])
        if op == "layer_int4":
            return _plain_layer(state, _values(state["c1"]), _values(state["c2"]))
        if op == "grouped_int4":
            return _plain_grouped(state)
        return _plain_quantize(state)
    kernels = _kernels()
    if op in ("layer", "layer_int4"):
        return kernels.moe_few_tokens(state["x"], state["router"], state["w1"], state["w2"],
                                      state["off"], state["max_width"], case["top_k"],
                                      norm_topk_prob=case["norm"], activation=case["activation"])
    if op == "grouped_int4":
        if case["direction"] == "up":
            return kernels.grouped_gemv_up_int4(state["x"], state["q"], state["tok_off"],
                                                state["off"], state["widths"], state["counts"],
                                                state["max_width"], activation=case["activation"])
        return kernels.grouped_gemv_down_int4(state["x"], state["q"], state["tok_off"],
                                              state["off"], state["widths"], state["counts"],
                                              case["hidden"])
    q = kernels.quantize_int4(state["w"], case["group"], row_offsets=state["row_offsets"])
    return kernels.dequantize_int4(q)


# ------------------------------------------------------------- work and exact
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    widths, hidden = _widths(case), case["hidden"]
    total, num = sum(widths), len(widths)
    if case["op"] == "quantize":
        n = total * hidden
        packed = n / 2 + n / case["group"] * 2
        # weights in, packed out; packed in, values out
        return {"bytes": n * size + 2 * packed + n * (2 if size == 4 else size), "flops": 6 * n}
    T, k = case["tokens"], case["top_k"]
    # experts that T tokens choosing k of them reach, on average
    active = num * (1.0 - (1.0 - k / num) ** T)
    weights = active * total / num * hidden
    per = size if case["op"] == "layer" else 0.5 + 2.0 / case["group"]
    gated = 2 if case["activation"] == "swiglu" else 1
    rows_flops = 2.0 * T * k * (total / num) * hidden
    if case["op"] == "grouped_int4":
        io = T * k * (hidden + max(widths)) * size
        return {"bytes": weights * per + io, "flops": rows_flops}
    io = 2 * T * hidden * size + num * hidden * size
    return {"bytes": (1 + gated) * weights * per + io,
            "flops": (1 + gated) * rows_flops + 2.0 * T * num * hidden}


def _exact_weight(weight):
    codes, scales, gid = weight
    return lambda rows, cols: ((codes[rows, cols].double() - 8) * scales[:, cols].double()[gid[rows]])


def exact(case, seed):
    global own
    was, own = own, False  # the inputs themselves, not a packed form of them
    try:
        st = prepare(case, seed)
    finally:
        own = was
    widths, op = _widths(case), case["op"]
    everything = slice(None)
    if op == "quantize":
        w, out = st["w"].double(), torch.empty(st["w"].shape, dtype=torch.float64, device="cuda")
        scale_dtype = torch.bfloat16 if st["w"].dtype == torch.float32 else st["w"].dtype
        first = 0
        for n in ([case["hidden"]] if case["direction"] == "up" else widths):
            for r in range(first, first + n, case["group"]):
                part = w[r:min(r + case["group"], first + n)]
                s = (part.abs().amax(0) / 7).to(scale_dtype).double()
                q = torch.where(s > 0, (part / s).round().clamp(-8, 7), 0.0)
                out[r:r + part.shape[0]] = q * s
            first += n
        return out

    if op == "layer":
        w1, w2 = (lambda r, c: st["w1"][r, c].double()), (lambda r, c: st["w2"][r, c].double())
    elif op == "layer_int4":
        w1, w2 = _exact_weight(st["c1"]), _exact_weight(st["c2"])
    else:
        w1 = w2 = _exact_weight(st["weight"])
    gated = 2 if case["activation"] == "swiglu" else 1
    x = st["x"].double()

    def up(xe, a, w):
        u = xe @ w1(everything, slice(gated * a, gated * (a + w)))
        if case["activation"] == "relu_squared":
            return u.relu() ** 2
        if gated == 2:
            return torch.nn.functional.silu(u[:, :w]) * u[:, w:]
        return u

    if op == "grouped_int4":
        up_dir = case["direction"] == "up"
        out = torch.zeros(x.shape[0], st["max_width"] if up_dir else case["hidden"],
                          dtype=torch.float64, device="cuda")
        bounds, a = st["tok_off"].tolist(), 0
        for i, w in enumerate(widths):
            rows = slice(bounds[i], bounds[i + 1])
            if bounds[i + 1] > bounds[i]:
                if up_dir:
                    out[rows, :w] = up(x[rows], a, w)
                else:
                    out[rows] = x[rows, :w] @ w2(slice(a, a + w), everything)
            a += w
        return out

    p = torch.sigmoid(x @ st["router"].double().T)
    chosen = torch.zeros_like(p)
    idx = p.topk(case["top_k"], dim=1).indices
    weight = p.gather(1, idx)
    if case["norm"]:
        weight = weight / (weight.sum(1, keepdim=True) + 1e-20)
    chosen.scatter_(1, idx, weight)
    picked = torch.zeros_like(p, dtype=torch.bool).scatter_(1, idx, True)
    out, a = torch.zeros_like(x), 0
    for i, w in enumerate(widths):
        t = picked[:, i].nonzero().flatten()
        if t.numel():
            y = up(x[t], a, w) @ w2(slice(a, a + w), everything)
            out[t] += y * chosen[t, i:i + 1]
        a += w
    return out
