"""The whole MoE layer for a few tokens (decode), in two launches (four above 8
tokens; three up to 8 with an fp32 router beside 4-bit experts).

No counterpart in the reference: its layer (triton_moe/moe.py:148-249) sorts the
tokens and pads every expert's rows to a tile, which at a few tokens is mostly
padding and launches.  `moe_few_tokens` computes the same layer output for up to
FEW_TOKENS_MAX tokens (csrc/few_tokens.cu): routing, up product, activation, down
product and weighted sum.  It never synchronises the host and can be captured in
a CUDA graph.

What differs from the training forward is only rounding: logits and routing weights
stay fp32 (the forward rounds each to the storage type), so two experts whose logits
differ by less than that rounding may be ranked differently.  Experts are ranked by logit
where the forward ranks fp32 sigmoids: those of logits above about 17 are all 1 and of
logits below -88 all 0, and the forward then takes the lower index however far apart the
logits are (the weights are the same).  The intermediate keeps twice the digits of the
storage type (2^-16 relative in bf16; in fp16 2^-22 relative or 2^-25, whichever is more).
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from .._lib import ACT_CODE, DTYPE_CODE, check, lib
from . import _ops
from ._ops import _meta, status_buffer
from .int4 import Int4Weight, eager_only, on_device, refuse_grad, row_view, stream_of

FEW_TOKENS_MAX = 64

# What the sizes and types of a call come to, worked out and checked at the first call
# with them: (tokens, hidden, experts, group, columns of w1, workspace bytes, codes).
_signatures: dict[tuple, tuple] = {}


def _signature(x_shape, dt, router_shape, w1, w2, offsets, max_width, top_k, activation):
    if len(x_shape) != 2:
        raise ValueError(f"moe_few_tokens: x must be [tokens, hidden], got {tuple(x_shape)}")
    T, H = x_shape
    if T > FEW_TOKENS_MAX:
        raise ValueError(f"moe_few_tokens: at most {FEW_TOKENS_MAX} tokens, got {T} (use the "
                         "layer's forward)")
    if dt not in DTYPE_CODE:
        raise TypeError(f"moe_few_tokens: bf16, fp16 or fp32, got {dt}")
    if activation not in ACT_CODE:
        raise NotImplementedError(f"activation {activation!r} is not supported "
                                  f"(supported: {tuple(ACT_CODE)})")
    if len(router_shape) != 2 or router_shape[1] != H:
        raise ValueError(f"moe_few_tokens: router_weight must be [experts, {H}], got "
                         f"{tuple(router_shape)}")
    E = router_shape[0]
    if not 1 <= E <= 256 or not 1 <= top_k <= min(E, 32):
        raise ValueError(f"moe_few_tokens: 1 to 256 experts and top_k up to 32 of them, got {E} and "
                         f"{top_k}")
    if H % 16 or not 16 <= H <= 32768 or max_width % 16 or not 16 <= max_width <= 32768:
        raise ValueError("moe_few_tokens: hidden size and expert widths must be multiples of 16 up "
                         f"to 32768, got {H} and {max_width}")
    if offsets != E + 1:
        raise ValueError(f"moe_few_tokens: expert_weight_offsets needs {E + 1} entries, got {offsets}")
    gated = 2 if activation == "swiglu" else 1
    packed = isinstance(w1, Int4Weight)
    if packed != isinstance(w2, Int4Weight):
        raise TypeError("moe_few_tokens: w1 and w2 must both be tensors or both be Int4Weight")
    if len(w1.shape) != 2 or w1.shape[0] != H or w1.shape[1] % (16 * gated) or w1.shape[1] < 16:
        raise ValueError(f"moe_few_tokens: w1 must be [{H}, total width in multiples of "
                         f"{16 * gated}], got {tuple(w1.shape)}")
    total = w1.shape[1]
    if tuple(w2.shape) != (total // gated, H):
        raise ValueError(f"moe_few_tokens: w2 must be {(total // gated, H)}, got {tuple(w2.shape)}")
    group = 0
    if packed:
        if w1.group_size != w2.group_size:
            raise ValueError("moe_few_tokens: w1 and w2 must have one group size, got "
                             f"{w1.group_size} and {w2.group_size}")
        if w1.row_offsets is not None and len(w1.row_offsets) > 2:
            raise ValueError("moe_few_tokens: a 4-bit w1 is one segment (no row_offsets)")
        if len(w2.row_offsets or (0, 0)) != E + 1:
            raise ValueError(f"moe_few_tokens: a 4-bit w2 needs row_offsets of its {E} experts")
        group = w1.group_size
    act = ACT_CODE[activation]
    ws_bytes = int(lib.moe_few_tokens_workspace_bytes(T, H, E, top_k, max_width, act))
    return T, H, E, group, total, ws_bytes, act, DTYPE_CODE[dt]


@eager_only
def moe_few_tokens(
    x: torch.Tensor,
    router_weight: torch.Tensor,
    w1: torch.Tensor | Int4Weight,
    w2: torch.Tensor | Int4Weight,
    expert_weight_offsets: torch.Tensor,
    max_expert_width: int,
    top_k: int,
    norm_topk_prob: bool = True,
    activation: str = "relu_squared",
) -> torch.Tensor:
    """Output [T, H] of the MoE layer for x [T, H], T <= 64.

    router_weight [E, H]; w1 [H, total width] and w2 [total width, H] with the
    experts side by side at expert_weight_offsets (device, [E + 1]), in bf16, fp16
    or fp32 (fp32 products are fp32, not tf32), or both Int4Weight (x in the
    scales' bf16 or fp16, the router in that or fp32; w2 quantised with the experts'
    row offsets).  activation "relu_squared", "none" or "swiglu" (then w1 holds each
    expert's gate columns and up columns, the offsets step by 2 w_e and w2 has half as
    many rows as w1 columns).  Hidden size and widths are multiples of 16; an expert
    whose offsets do not fit (with 4-bit weights: are not those that w2 was quantised
    with) adds nothing and sets the device status word.  In fp16 an intermediate above
    65504 is infinite, as in the training forward; 4-bit products make a NaN of an
    infinite x or intermediate, and in bf16 can of one from 2^115 on.  Inference only."""
    dt, dev = x.dtype, x.device
    packed = w1.__class__ is Int4Weight and w2.__class__ is Int4Weight
    if packed:
        t1, t2 = w1.packed, w2.packed
        key = (x.shape, dt, router_weight.shape, w1.shape, w2.shape, w1.group_size, w2.group_size,
               w1.row_offsets is None or len(w1.row_offsets), w2.row_offsets is None or
               len(w2.row_offsets), expert_weight_offsets.numel(), max_expert_width, top_k,
               activation)
    else:
        t1, t2 = w1, w2
        key = (x.shape, dt, router_weight.shape, w1.shape, w2.shape, w1.__class__ is Int4Weight,
               w2.__class__ is Int4Weight, expert_weight_offsets.numel(), max_expert_width, top_k,
               activation)
    sig = _signatures.get(key)
    if sig is None:
        sig = _signature(x.shape, dt, router_weight.shape, w1, w2, expert_weight_offsets.numel(),
                         max_expert_width, top_k, activation)
        if len(_signatures) >= 4096:
            _signatures.clear()
        _signatures[key] = sig
    T, H, E, group, total, ws_bytes, act, dt_code = sig
    if not x.is_cuda:
        raise ValueError("moe_b200 kernels need CUDA tensors (no CPU fallback)")
    rdt = router_weight.dtype
    if w1.dtype is not dt or w2.dtype is not dt or (
            rdt is not dt and not (packed and rdt is torch.float32)):
        raise TypeError(f"moe_few_tokens: x, router_weight, w1 and w2 must share a dtype, got {dt}, "
                        f"{rdt}, {w1.dtype} and {w2.dtype}")
    idx = x.get_device()
    if (router_weight.get_device() != idx or t1.get_device() != idx or t2.get_device() != idx
            or expert_weight_offsets.get_device() != idx):
        raise ValueError("moe_few_tokens: all tensors must be on one device")
    if not (t1.is_contiguous() and t2.is_contiguous() and router_weight.is_contiguous()):
        raise ValueError("moe_few_tokens: router_weight, w1 and w2 must be contiguous")
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        if packed:
            refuse_grad("moe_few_tokens", x, router_weight, w1.scales, w2.scales)
        else:
            refuse_grad("moe_few_tokens", x, router_weight, t1, t2)
    out = torch.empty((T, H), dtype=dt, device=dev)
    if T == 0:
        return out
    x = row_view(x)
    off = _meta(expert_weight_offsets)
    p1, p2, pr = t1.data_ptr(), t2.data_ptr(), router_weight.data_ptr()
    if (p1 | p2 | pr) & 15:
        raise ValueError("moe_few_tokens: weights must be 16-byte aligned")
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    with on_device(dev):
        ev = _ops._ev_begin()
        if packed:
            rc = lib.moe_few_tokens_int4(
                x.data_ptr(), T, x.stride(0) if T > 1 else H, H, pr, DTYPE_CODE[rdt], E, p1,
                w1.scales.data_ptr(), p2, w2.scales.data_ptr(), group, w2._host_offsets, total,
                off.data_ptr(), max_expert_width, top_k, 1 if norm_topk_prob else 0, act,
                out.data_ptr(), H, ws.data_ptr(), ws_bytes, dt_code, status_buffer(dev).data_ptr(),
                stream_of(dev))
        else:
            rc = lib.moe_few_tokens(
                x.data_ptr(), T, x.stride(0) if T > 1 else H, H, pr, E, p1, None, p2, None, 0, 0, 0,
                total, off.data_ptr(), max_expert_width, top_k, 1 if norm_topk_prob else 0, act,
                out.data_ptr(), H, ws.data_ptr(), ws_bytes, dt_code, status_buffer(dev).data_ptr(),
                stream_of(dev))
        _ops._ev_end(ev, "few_tokens")
    if rc:
        check(rc, "moe_few_tokens")
    _ops._count((2 if T <= 8 else 4) + (T <= 8 and rdt is not dt))
    return out
