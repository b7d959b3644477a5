"""The few-token operators in 64 bits, with the error a kernel may have.

Each reference returns (value, bound).  The bound follows the kernels' arithmetic:
  * one rounding of the output: half a step, eps / 2 of the value;
  * fp32 sums of n products: n_adds * 2^-22 of the sum of magnitudes, n_adds being
    the additions in sequence (16 products a tensor-core step, whose alignment may
    drop bits below 2^-22 of the largest; one product an addition in fp32);
  * the intermediate as two 16-bit operands: (eps / 2)^2 of it, and for fp16 the
    smallest step 2^-24;
  * the routing weight: sigmoid and one division, 2^-20 relative, plus the error of
    its logit (its derivative is at most 1/4 of it, absolutely; p(1-p) relative 1-p).
  * 4-bit weights: the sums hold terms of (31 + 24) scales in bf16, (143 + 136) in
    fp16, for a weight (q - 8) scale, so their magnitudes are taken with those.
First-order terms are carried through the activation; nothing is fitted.
"""

import torch

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def adds(n, dtype):
    """Relative error of an fp32 sum of n products, against the sum of magnitudes."""
    return (n / (1 if dtype == torch.float32 else 16) + 40) * 2.0**-22


def activate(u, du, act):
    """(h, its error) for u [..., w] (swiglu: [..., 2 w]) with error du."""
    if act == "relu_squared":
        r = u.clamp(min=0)
        return r * r, 2 * r * du + du * du + r * r * 2.0**-22
    if act == "swiglu":
        w = u.shape[-1] // 2
        g, up, dg, dup = u[..., :w], u[..., w:], du[..., :w], du[..., w:]
        s = torch.sigmoid(g)
        silu = g * s
        h = silu * up
        # |silu'| <= 1.1; expf and the division: 2^-20
        return h, 1.1 * dg * up.abs() + silu.abs() * dup + 1.1 * dg * dup + h.abs() * 2.0**-20
    return u, du


def choose(x, router, k):
    """Experts [T, k] by logit, equal ones in index order."""
    logits = x.double() @ router.double().t()
    return torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k], logits


def clear_choice(x, router, k):
    """Whether every token's k-th and next logit are equal or further apart than both
    may be off in fp32 (otherwise either choice is right)."""
    logits = x.double() @ router.double().t()
    if k >= logits.shape[1]:
        return True
    err = ((x.double().abs() @ router.double().abs().t()) * adds(x.shape[1], x.dtype)).amax(1)
    top = logits.sort(dim=1, descending=True).values
    gap = top[:, k - 1] - top[:, k]
    return bool(((gap > 2 * err) | (gap == 0)).all())


def int4_terms(scales, dtype):
    """Magnitudes of the terms in the sums of 4-bit weights, from the scale of each."""
    return scales.double().abs() * (55 if dtype == torch.bfloat16 else 279)


def layer(x, router, w1, w2, offsets, k, norm, act, m1=None, m2=None):
    """offsets: host list of w1's column offsets; m1, m2: magnitudes of the summed
    terms (default: of the weights).  Returns (out, bound) in fp64."""
    m1, m2 = w1 if m1 is None else m1, w2 if m2 is None else m2
    dt = x.dtype
    half = HALF_STEP[dt]
    gated = 2 if act == "swiglu" else 1
    T, H = x.shape
    xd = x.double()
    sel, logits = choose(x, router, k)
    lerr = (xd.abs() @ router.double().abs().t()) * adds(H, dt)
    assert clear_choice(x, router, k), "the inputs have a near tie"
    p = torch.sigmoid(logits).gather(1, sel)
    perr = p * (1 - p) * lerr.gather(1, sel) + p * 2.0**-20
    if norm:
        s = p.sum(1, keepdim=True) + 1e-20
        perr = perr / s + p / s * (perr.sum(1, keepdim=True) / s + 2.0**-20)
        p = p / s
    out = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    err = torch.zeros_like(out)
    for e in range(len(offsets) - 1):
        t, slot = (sel == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        a, b = offsets[e], offsets[e + 1]
        w1e, w2e = w1[:, a:b].double(), w2[a // gated:b // gated].double()
        m1e, m2e = m1[:, a:b].double().abs(), m2[a // gated:b // gated].double().abs()
        u = xd[t] @ w1e
        h, dh = activate(u, (xd[t].abs() @ m1e) * adds(H, dt), act)
        if dt != torch.float32:
            dh = dh + h.abs() * half * half + (2.0**-24 if dt == torch.float16 else 0.0)
        y = h @ w2e
        mag = h.abs() @ m2e
        dy = dh @ w2e.abs() + mag * adds(b - a, dt)
        g, dg = p[t, slot, None], perr[t, slot, None]
        out[t] += g * y
        err[t] += g * dy + dg * (y.abs() + dy) + g * mag * 2.0**-20
    return out, err + out.abs() * half * (1 + 2.0**-10) + (2.0**-24 if dt == torch.float16 else 1e-38)


def grouped(x, w, row_ranges, offsets, max_width, act, down, m=None):
    """row_ranges: [(first, count)] an expert; w: fp64-able matrix; m: as layer's."""
    m = w if m is None else m
    dt = x.dtype
    half = HALF_STEP[dt]
    gated = 2 if act == "swiglu" else 1
    cols = w.shape[1] if down else max_width
    out = torch.zeros(x.shape[0], cols, dtype=torch.float64, device=x.device)
    err = torch.zeros_like(out)
    for e, (r, n) in enumerate(row_ranges):
        a, b = offsets[e], offsets[e + 1]
        if n == 0 or a == b:
            continue
        xe = x[r:r + n].double()
        we = w[a:b].double() if down else w[:, a:b].double()
        if down:
            xe = xe[:, :b - a]
        u = xe @ we
        me = (m[a:b] if down else m[:, a:b]).double().abs()
        h, dh = activate(u, (xe.abs() @ me) * adds(xe.shape[1], dt), act)
        c = cols if down else (b - a) // gated
        out[r:r + n, :c] = h
        err[r:r + n, :c] = dh + h.abs() * half * (1 + 2.0**-10)
    return out, err + (2.0**-24 if dt == torch.float16 else 1e-38)


def quantize(w, group, segments, scale_dtype):
    """(codes int64 [K, N], scales [groups, N]) by the definition, in 64 bits."""
    codes, scales, first = [], [], 0
    for n in segments:
        for r in range(first, first + n, group):
            part = w[r:min(r + group, first + n)].double()
            s = (part.abs().amax(0) / 7).to(scale_dtype)
            sd = s.double()
            q = torch.where(sd > 0, (part / sd).round().clamp(-8, 7), 0.0)
            codes.append(q.long() + 8)
            scales.append(s)
        first += n
    return torch.cat(codes), torch.stack(scales)


def assert_within(got, ref, bound, what):
    d = (got.double() - ref).abs()
    bad = ~(d <= bound)
    if bool(bad.any()):
        i = int((d / bound).nan_to_num(float("inf")).argmax())
        raise AssertionError(
            f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst at {i}: got "
            f"{float(got.flatten()[i])}, want {float(ref.flatten()[i])}, bound "
            f"{float(bound.flatten()[i])}")
