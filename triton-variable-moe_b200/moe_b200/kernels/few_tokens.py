"""The whole MoE layer for a few tokens (decode), in two launches.

No counterpart in the reference: its layer (triton_moe/moe.py:148-249) sorts the
tokens and pads every expert's rows to a tile, which at a few tokens is mostly
padding and launches.  `moe_few_tokens` computes the same layer output for up to
FEW_TOKENS_MAX tokens (csrc/few_tokens.cu): routing, up product, activation, down
product and weighted sum.  It never synchronises the host and can be captured in
a CUDA graph.

What differs from the training forward is only rounding: logits, routing weights
and the intermediate stay fp32 (the forward rounds each to the storage type), so
two experts whose logits differ by less than that rounding may be ranked
differently.
"""

from __future__ import annotations

import torch

from .._lib import ACT_CODE, DTYPE_CODE, check, lib
from ._ops import _count, _ev_begin, _ev_end, _meta, status_buffer
from .int4 import Int4Weight, eager_only, on_device, refuse_grad, row_view, stream_of

FEW_TOKENS_MAX = 64

_workspace_bytes: dict[tuple, int] = {}


def _check_weights(x, router, w1, w2, num_experts, hidden, max_width, gated):
    """(w1 tensor, its scales, w2 tensor, its scales, group, blocks, groups, columns of w1)."""
    if isinstance(w1, Int4Weight) != isinstance(w2, Int4Weight):
        raise TypeError("moe_few_tokens: w1 and w2 must both be tensors or both be Int4Weight")
    dt, dev = x.dtype, x.device
    if router.dtype != dt or w1.dtype != dt or w2.dtype != dt:
        raise TypeError(f"moe_few_tokens: x, router_weight, w1 and w2 must share a dtype, got {dt}, "
                        f"{router.dtype}, {w1.dtype} and {w2.dtype}")
    if router.device != dev or w1.device != dev or w2.device != dev:
        raise ValueError("moe_few_tokens: all tensors must be on one device")
    if len(w1.shape) != 2 or w1.shape[0] != hidden or w1.shape[1] % (16 * gated) or w1.shape[1] < 16:
        raise ValueError(f"moe_few_tokens: w1 must be [{hidden}, total width in multiples of "
                         f"{16 * gated}], got {tuple(w1.shape)}")
    total = w1.shape[1]
    if tuple(w2.shape) != (total // gated, hidden):
        raise ValueError(f"moe_few_tokens: w2 must be {(total // gated, hidden)}, got "
                         f"{tuple(w2.shape)}")
    if isinstance(w1, Int4Weight):
        if w1.group_size != w2.group_size:
            raise ValueError("moe_few_tokens: w1 and w2 must have one group size, got "
                             f"{w1.group_size} and {w2.group_size}")
        if w1.row_offsets is not None and len(w1.row_offsets) > 2:
            raise ValueError("moe_few_tokens: a 4-bit w1 is one segment (no row_offsets)")
        offs = w2.row_offsets if w2.row_offsets is not None else (0, w2.rows)
        if len(offs) != num_experts + 1:
            raise ValueError(f"moe_few_tokens: a 4-bit w2 needs row_offsets of its {num_experts} "
                             "experts")
        return (w1.packed, w1.scales.data_ptr(), w2.packed, w2.scales.data_ptr(), w1.group_size,
                w2.packed.shape[0], w2.scales.shape[0], total)
    if not (w1.is_contiguous() and w2.is_contiguous()):
        raise ValueError("moe_few_tokens: w1 and w2 must be contiguous")
    return w1, None, w2, None, 0, 0, 0, total


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
    scales' bf16 or fp16).  activation "relu_squared", "none" or "swiglu" (then w1
    holds each expert's gate columns and up columns, the offsets step by 2 w_e and
    w2 has half as many rows as w1 columns).  Hidden size and widths are multiples
    of 16; an expert whose offsets do not fit adds nothing and sets the device
    status word.  In fp16 an intermediate above 65504 is infinite, as in the
    training forward.  Inference only."""
    if x.dim() != 2:
        raise ValueError(f"moe_few_tokens: x must be [tokens, hidden], got {tuple(x.shape)}")
    T, H = x.shape
    if T > FEW_TOKENS_MAX:
        raise ValueError(f"moe_few_tokens: at most {FEW_TOKENS_MAX} tokens, got {T} (use the "
                         "layer's forward)")
    if not (x.is_cuda and expert_weight_offsets.is_cuda):
        raise ValueError("moe_b200 kernels need CUDA tensors (no CPU fallback)")
    if x.dtype not in DTYPE_CODE:
        raise TypeError(f"moe_few_tokens: bf16, fp16 or fp32, got {x.dtype}")
    if activation not in ACT_CODE:
        raise NotImplementedError(f"activation {activation!r} is not supported "
                                  f"(supported: {tuple(ACT_CODE)})")
    E = router_weight.shape[0]
    if router_weight.dim() != 2 or router_weight.shape[1] != H or not router_weight.is_contiguous():
        raise ValueError(f"moe_few_tokens: router_weight must be contiguous [experts, {H}], got "
                         f"{tuple(router_weight.shape)}")
    if not 1 <= E <= 256 or not 1 <= top_k <= min(E, 32):
        raise ValueError(f"moe_few_tokens: 1 to 256 experts and top_k up to 32 of them, got {E} and "
                         f"{top_k}")
    if (H % 16 or not 16 <= H <= 32768 or max_expert_width % 16
            or not 16 <= max_expert_width <= 32768):
        raise ValueError("moe_few_tokens: hidden size and expert widths must be multiples of 16 up "
                         f"to 32768, got {H} and {max_expert_width}")
    if expert_weight_offsets.numel() != E + 1 or expert_weight_offsets.device != x.device:
        raise ValueError(f"moe_few_tokens: expert_weight_offsets needs {E + 1} entries on x's device")
    gated = 2 if activation == "swiglu" else 1
    w1t, s1, w2t, s2, group, blocks, groups, total = _check_weights(
        x, router_weight, w1, w2, E, H, max_expert_width, gated)
    if group:
        refuse_grad("moe_few_tokens", x, router_weight)
    else:
        refuse_grad("moe_few_tokens", x, router_weight, w1, w2)
    dev = x.device
    out = torch.empty(T, H, dtype=x.dtype, device=dev)
    if T == 0:
        return out
    x = row_view(x)
    off = _meta(expert_weight_offsets)
    p1, p2, pr = w1t.data_ptr(), w2t.data_ptr(), router_weight.data_ptr()
    if (p1 | p2 | pr) & 15:
        raise ValueError("moe_few_tokens: weights must be 16-byte aligned")
    act = ACT_CODE[activation]
    key = (T, H, E, top_k, max_expert_width, act)
    ws_bytes = _workspace_bytes.get(key)
    if ws_bytes is None:
        ws_bytes = int(lib.moe_few_tokens_workspace_bytes(*key))
        if len(_workspace_bytes) > 4096:
            _workspace_bytes.clear()
        _workspace_bytes[key] = ws_bytes
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    with on_device(dev):
        ev = _ev_begin()
        rc = lib.moe_few_tokens(
            x.data_ptr(), T, x.stride(0) if T > 1 else H, H, pr, E, p1, s1, p2, s2, group, blocks,
            groups, total, off.data_ptr(), max_expert_width, top_k, 1 if norm_topk_prob else 0, act,
            out.data_ptr(), H, ws.data_ptr(), ws_bytes, DTYPE_CODE[x.dtype],
            status_buffer(dev).data_ptr(), stream_of(dev))
        _ev_end(ev, "few_tokens")
    check(rc, "moe_few_tokens")
    _count(2)
    return out
