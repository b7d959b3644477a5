"""4-bit expert weights with group scales, and the grouped products that read them.

No counterpart in the reference, whose weights are bf16/fp16/fp32.  A weight
[K, N] is (q - 8) * scale with q in 0..15 and one scale for `group_size` rows of
a column; `Int4Weight` holds it in the order in which the kernels multiply
(csrc/int4.cu).  `quantize_int4` rounds a weight, `pack_int4` takes codes and
scales from elsewhere (a checkpoint quantised by another program), and
`dequantize_int4` gives the values back.

`grouped_gemv_up_int4` / `grouped_gemv_down_int4` stand beside `grouped_gemm_up`
/ `grouped_gemm_down` (same arguments, an Int4Weight in place of the weight) for
a few rows an expert, as a decode step has: the weights are read once for every
8 rows of an expert.  The whole layer on 4-bit experts is `moe_few_tokens`.
Sums are fp32, with an error of a few 2^-22 of 55 (fp16: 279) scales times the sum of
|x|, whatever the codes (a column of codes 8 comes out at that, not at zero); an infinite
x, and in bf16 one from 2^115 on, can make a NaN.
All of it is for inference: nothing here is differentiable.
"""

from __future__ import annotations

import ctypes
import functools
from collections.abc import Sequence
from contextlib import nullcontext
from dataclasses import dataclass, field

import torch
from torch.autograd import forward_ad

from .._lib import ACT_CODE, DTYPE_CODE, check, lib, ptr
from ._ops import _count, _ev_begin, _ev_end, _meta, status_buffer

GROUP_SIZES = (32, 64, 128)
MAX_GEMV_ROWS = 65536


def eager_only(fn):
    """torch.compiler.disable for calls of a few microseconds: the disabled wrapper
    (8 us a call) is taken only while a graph is being traced."""
    disabled = torch.compiler.disable(fn)

    @functools.wraps(fn)
    def call(*args, **kwargs):
        if torch.compiler.is_compiling():
            return disabled(*args, **kwargs)
        return fn(*args, **kwargs)

    return call


def refuse_tangent(name: str, *tensors: torch.Tensor) -> None:
    """Forward-mode derivatives, which torch.no_grad() leaves on."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no forward-mode derivative, and an argument has a "
                               "tangent: pass its primal value")


def refuse_grad(name: str, *tensors: torch.Tensor) -> None:
    if forward_ad._current_level >= 0:
        refuse_tangent(name, *tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError(f"{name} is for inference and has no backward: call it under "
                                   "torch.no_grad() or torch.inference_mode()")


_here = nullcontext()


def on_device(device: torch.device):
    """Context in which `device` is the current CUDA device."""
    return _here if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def stream_of(device: torch.device) -> int:
    """The current stream's handle (torch.cuda.current_stream builds an object first,
    2 us a call)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def row_view(x: torch.Tensor) -> torch.Tensor:
    """x [rows, cols] itself where its rows are contiguous 16-byte vectors, else a copy."""
    vec = 16 // x.element_size()
    rows = x.shape[0]
    if (x.stride(1) == 1 and x.data_ptr() % 16 == 0
            and (rows == 1 or (x.stride(0) >= x.shape[1] and x.stride(0) % vec == 0))):
        return x
    return x.clone(memory_format=torch.contiguous_format)


@dataclass(frozen=True, eq=False)
class Int4Weight:
    """A [rows, cols] weight in 4 bits.

    packed: uint8 [block rows, cols / 16, 512]; scales: [groups, cols] in `dtype`;
    row_offsets: where groups start anew (None: only at row 0)."""

    packed: torch.Tensor
    scales: torch.Tensor
    rows: int
    cols: int
    group_size: int
    row_offsets: tuple[int, ...] | None = None
    _host_offsets: object = field(init=False, repr=False, compare=False, default=None)

    def __post_init__(self):
        blocks, groups, host = _layout(self.rows, self.cols, self.group_size, self.row_offsets)
        if (self.packed.shape != (blocks, self.cols // 16, 512) or self.packed.dtype != torch.uint8
                or not self.packed.is_contiguous()):
            raise ValueError(f"packed must be contiguous uint8 {(blocks, self.cols // 16, 512)}, "
                             f"got {self.packed.dtype} {tuple(self.packed.shape)}")
        if self.scales.shape != (groups, self.cols) or not self.scales.is_contiguous():
            raise ValueError(f"scales must be contiguous {(groups, self.cols)}, "
                             f"got {tuple(self.scales.shape)}")
        if self.scales.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"scales must be bf16 or fp16, got {self.scales.dtype}")
        if self.packed.device != self.scales.device:
            raise ValueError("packed and scales must be on one device")
        if self.packed.data_ptr() % 16 or self.scales.data_ptr() % 16:
            raise ValueError("packed and scales must be 16-byte aligned")
        object.__setattr__(self, "_host_offsets", host)

    @classmethod
    def _trusted(cls, packed, scales, rows, cols, group_size, row_offsets, host) -> "Int4Weight":
        """From parts that this module has just made."""
        self = object.__new__(cls)
        self.__dict__.update(packed=packed, scales=scales, rows=rows, cols=cols,
                             group_size=group_size, row_offsets=row_offsets, _host_offsets=host)
        return self

    def __reduce__(self):  # copies and pickles: all but the host offsets, made again
        return (Int4Weight, (self.packed, self.scales, self.rows, self.cols, self.group_size,
                             self.row_offsets))

    @property
    def dtype(self) -> torch.dtype:
        return self.scales.dtype

    @property
    def device(self) -> torch.device:
        return self.packed.device

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.cols

    def to(self, device) -> "Int4Weight":
        """The same weight on another device."""
        return Int4Weight(self.packed.to(device), self.scales.to(device), self.rows, self.cols,
                          self.group_size, self.row_offsets)

    def _segments(self):
        n = 1 if self._host_offsets is None else len(self.row_offsets) - 1
        return self._host_offsets, n


@functools.lru_cache(maxsize=256)
def _layout(rows: int, cols: int, group_size: int, row_offsets: tuple[int, ...] | None):
    """(block rows, groups, host offset array) of a weight; ValueError if it cannot be packed."""
    if group_size not in GROUP_SIZES:
        raise ValueError(f"group_size must be one of {GROUP_SIZES}, got {group_size}")
    if rows < 16 or rows % 16 or cols < 16 or cols % 16:
        raise ValueError(f"4-bit weights need rows and columns in multiples of 16, got {rows} x {cols}")
    host, n = None, 1
    if row_offsets is not None:
        n = len(row_offsets) - 1
        if not 1 <= n <= 256:
            raise ValueError(f"row_offsets must name 1 to 256 segments, got {n}")
        if min(row_offsets) < 0 or max(row_offsets) >= 2**31:
            raise ValueError(f"row_offsets must lie in 0..{rows}")
        host = (ctypes.c_int32 * (n + 1))(*row_offsets)
    blocks, groups = ctypes.c_int64(), ctypes.c_int64()
    rc = lib.moe_int4_rows(rows, group_size, host, n, ctypes.addressof(blocks),
                           ctypes.addressof(groups))
    if rc != 0:
        raise ValueError("row_offsets must ascend in multiples of 16 from 0 to the number of rows "
                         f"({rows})")
    return blocks.value, groups.value, host


def _offsets_tuple(row_offsets: Sequence[int] | None) -> tuple[int, ...] | None:
    if row_offsets is None:
        return None
    if isinstance(row_offsets, torch.Tensor):
        if row_offsets.is_cuda:
            raise TypeError("row_offsets are read on the host: pass a list, not a CUDA tensor")
        row_offsets = row_offsets.tolist()
    return tuple(row_offsets)


@eager_only
def quantize_int4(w: torch.Tensor, group_size: int = 64, row_offsets: Sequence[int] | None = None,
                  dtype: torch.dtype | None = None) -> Int4Weight:
    """Round w [K, N] to 4 bits: in each column, for every `group_size` rows,
    scale = amax / 7 (rounded to `dtype`: w's own, bf16 for an fp32 w unless fp16
    is asked for) and q = rint(w / scale), ties to even, within -8..7.

    row_offsets: host integers [0, ..., K] at which groups start anew, for a
    weight of stacked experts (w2).  A group of zeros is exact; one that holds a
    NaN or an infinity, or whose scale is above `dtype`'s range, reads back as NaN."""
    if not w.is_cuda:
        raise ValueError("moe_b200 kernels need CUDA tensors (no CPU fallback)")
    if w.dim() != 2 or w.dtype not in DTYPE_CODE:
        raise TypeError(f"quantize_int4 takes a bf16, fp16 or fp32 matrix, got {w.dtype} "
                        f"{tuple(w.shape)}")
    if dtype is None:
        dtype = torch.bfloat16 if w.dtype == torch.float32 else w.dtype
    if dtype not in (torch.bfloat16, torch.float16) or w.dtype not in (dtype, torch.float32):
        raise TypeError(f"a {w.dtype} weight cannot be quantised with {dtype} scales")
    K, N = w.shape
    offsets = _offsets_tuple(row_offsets)
    blocks, groups, host = _layout(K, N, group_size, offsets)
    refuse_tangent("quantize_int4", w)
    w = row_view(w.detach())
    dev = w.device
    packed = torch.empty(blocks, N // 16, 512, dtype=torch.uint8, device=dev)
    scales = torch.empty(groups, N, dtype=dtype, device=dev)
    with on_device(dev):
        ev = _ev_begin()
        rc = lib.moe_int4_quantize(ptr(w), K, N, w.stride(0) if K > 1 else N, DTYPE_CODE[w.dtype],
                                   group_size, host, 1 if host is None else len(offsets) - 1,
                                   ptr(packed), ptr(scales), DTYPE_CODE[dtype], stream_of(dev))
        _ev_end(ev, "quantize_int4")
    check(rc, "moe_int4_quantize")
    _count(1)
    return Int4Weight._trusted(packed, scales, K, N, group_size, offsets, host)


@eager_only
def pack_int4(codes: torch.Tensor, scales: torch.Tensor, group_size: int,
              row_offsets: Sequence[int] | None = None) -> Int4Weight:
    """An Int4Weight from uint8 codes [K, N] (the low 4 bits; 8 stands for zero)
    and scales [groups, N] (bf16 or fp16; groups start anew at row_offsets)."""
    if not codes.is_cuda:
        raise ValueError("moe_b200 kernels need CUDA tensors (no CPU fallback)")
    if codes.dim() != 2 or codes.dtype != torch.uint8:
        raise TypeError(f"codes must be a uint8 matrix, got {codes.dtype} {tuple(codes.shape)}")
    K, N = codes.shape
    offsets = _offsets_tuple(row_offsets)
    blocks, groups, host = _layout(K, N, group_size, offsets)
    if scales.shape != (groups, N) or scales.device != codes.device:
        raise ValueError(f"scales must be {(groups, N)} on {codes.device}, got "
                         f"{tuple(scales.shape)} on {scales.device}")
    refuse_tangent("pack_int4", scales)
    codes = row_view(codes)
    scales = scales.detach()
    if not scales.is_contiguous() or scales.data_ptr() % 16:
        scales = scales.clone(memory_format=torch.contiguous_format)
    dev = codes.device
    packed = torch.empty(blocks, N // 16, 512, dtype=torch.uint8, device=dev)
    with on_device(dev):
        ev = _ev_begin()
        rc = lib.moe_int4_pack(ptr(codes), K, N, codes.stride(0) if K > 1 else N, group_size, host,
                               1 if host is None else len(offsets) - 1, ptr(packed),
                               stream_of(dev))
        _ev_end(ev, "pack_int4")
    check(rc, "moe_int4_pack")
    _count(1)
    return Int4Weight(packed, scales, K, N, group_size, offsets)


@eager_only
def dequantize_int4(q: Int4Weight) -> torch.Tensor:
    """The values (q - 8) * scale [K, N], rounded to the scales' type."""
    if not q.packed.is_cuda:
        raise ValueError("moe_b200 kernels need CUDA tensors (no CPU fallback)")
    out = torch.empty(q.rows, q.cols, dtype=q.dtype, device=q.device)
    refuse_grad("dequantize_int4", q.scales)
    host, n = q._segments()
    with on_device(q.device):
        ev = _ev_begin()
        rc = lib.moe_int4_dequantize(ptr(q.packed), ptr(q.scales), q.rows, q.cols, q.group_size,
                                     host, n, ptr(out), q.cols, DTYPE_CODE[q.dtype],
                                     stream_of(q.device))
        _ev_end(ev, "dequantize_int4")
    check(rc, "moe_int4_dequantize")
    _count(1)
    return out


def _gemv(name, x, q, tok_off, w_off, expert_widths, tok_cnt, hidden, max_width, activation, down):
    E = len(expert_widths)
    if not isinstance(q, Int4Weight):
        raise TypeError(f"{name} takes an Int4Weight, got {type(q).__name__}")
    if not (x.is_cuda and q.packed.is_cuda and tok_off.is_cuda and w_off.is_cuda
            and (tok_cnt is None or tok_cnt.is_cuda)):
        raise ValueError("moe_b200 kernels need CUDA tensors (no CPU fallback)")
    if not (x.device == q.device == tok_off.device == w_off.device) or (
            tok_cnt is not None and tok_cnt.device != x.device):
        raise ValueError(f"{name}: all tensors must be on one device")
    if x.dtype != q.dtype:
        raise TypeError(f"{name}: x is {x.dtype}, the weight's scales are {q.dtype}")
    if activation not in ACT_CODE:
        raise NotImplementedError(f"activation {activation!r} is not supported "
                                  f"(supported: {tuple(ACT_CODE)})")
    if not 1 <= E <= 256:
        raise ValueError(f"{name}: 1 to 256 experts, got {E}")
    if tok_off.numel() != E + 1 or w_off.numel() != E + 1 or (
            tok_cnt is not None and tok_cnt.numel() != E):
        raise ValueError(f"{name}: expert_token_offsets and expert_weight_offsets need {E + 1} "
                         f"entries, tokens_per_expert {E}")
    if max_width < 16 or max_width % 16 or max_width > 32768 or hidden > 32768:
        raise ValueError(f"{name}: hidden size and expert widths must be multiples of 16 up to "
                         f"32768, got {hidden} and {max_width}")
    if x.dim() != 2 or x.shape[1] != (max_width if down else hidden):
        raise ValueError(f"{name}: x must be [rows, {max_width if down else hidden}], got "
                         f"{tuple(x.shape)}")
    if down:
        if q.cols != hidden:
            raise ValueError(f"{name}: the weight has {q.cols} columns, hidden_size is {hidden}")
        if (E if q.row_offsets is not None else 1) != (
                1 if q.row_offsets is None else len(q.row_offsets) - 1) or (
                q.row_offsets is None and E != 1):
            raise ValueError(f"{name}: the weight needs row_offsets of its {E} experts")
    elif q.row_offsets is not None and len(q.row_offsets) > 2:
        raise ValueError(f"{name}: the up weight is one segment (no row_offsets)")
    rows = x.shape[0]
    if rows > MAX_GEMV_ROWS:
        raise ValueError(f"{name}: at most {MAX_GEMV_ROWS} rows, got {rows}")
    refuse_grad(name, x, q.scales)
    dev = x.device
    out_cols = hidden if down else max_width
    out = torch.empty(rows, out_cols, dtype=x.dtype, device=dev)
    if rows == 0:
        return out
    x = row_view(x)
    tok_off, w_off, tok_cnt = _meta(tok_off), _meta(w_off), _meta(tok_cnt)
    ws_bytes = int(lib.moe_grouped_gemv_int4_workspace_bytes(
        rows, hidden, max_width, ACT_CODE[activation], 1 if down else 0))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    with on_device(dev):
        ev = _ev_begin()
        ldx = x.stride(0) if rows > 1 else x.shape[1]
        if down:
            rc = lib.moe_grouped_gemv_down_int4(
                ptr(x), rows, ldx, ptr(q.packed), ptr(q.scales), q.group_size, q._host_offsets,
                hidden, q.rows, ptr(tok_off), ptr(w_off), ptr(tok_cnt), E, max_width, ptr(out),
                out_cols, ptr(ws), ws_bytes, DTYPE_CODE[x.dtype], ptr(status_buffer(dev)),
                stream_of(dev))
        else:
            rc = lib.moe_grouped_gemv_int4(
                ptr(x), rows, ldx, ptr(q.packed), ptr(q.scales), q.group_size, q.packed.shape[0],
                q.scales.shape[0], hidden, q.cols, ptr(tok_off), ptr(w_off), ptr(tok_cnt), E,
                max_width, ACT_CODE[activation], 0, ptr(out), out_cols, ptr(ws), ws_bytes,
                DTYPE_CODE[x.dtype], ptr(status_buffer(dev)), stream_of(dev))
        _ev_end(ev, name)
    check(rc, name)
    _count(2)
    return out


@eager_only
def grouped_gemv_up_int4(
    x: torch.Tensor,
    w1: Int4Weight,
    expert_token_offsets: torch.Tensor,
    expert_weight_offsets: torch.Tensor,
    expert_widths: torch.Tensor,
    tokens_per_expert: torch.Tensor | None,
    max_expert_width: int,
    activation: str = "relu_squared",
) -> torch.Tensor:
    """grouped_gemm_up on 4-bit weights for a few rows an expert.

    x [rows, hidden] holds expert e's rows from expert_token_offsets[e], of which
    the first tokens_per_expert[e] (None: all) are computed.  Returns act(x @ W1_e)
    [rows, max_expert_width]; rows of no expert and columns past an expert's width
    are zero.  "swiglu": expert_weight_offsets step by 2 w_e (gate columns, then
    up columns).  Never reads the offsets on the host; an expert whose offsets do
    not fit gets zeros and sets the device status word."""
    return _gemv("grouped_gemv_up_int4", x, w1, expert_token_offsets, expert_weight_offsets,
                 expert_widths, tokens_per_expert, getattr(w1, "rows", 0), int(max_expert_width),
                 activation, False)


@eager_only
def grouped_gemv_down_int4(
    intermediate: torch.Tensor,
    w2: Int4Weight,
    expert_token_offsets: torch.Tensor,
    expert_weight_offsets: torch.Tensor,
    expert_widths: torch.Tensor,
    tokens_per_expert: torch.Tensor | None,
    hidden_size: int,
) -> torch.Tensor:
    """grouped_gemm_down on 4-bit weights for a few rows an expert:
    out[rows_e] = intermediate[rows_e, :w_e] @ W2_e, zero elsewhere.  w2 is
    quantised with the experts' row offsets; expert_weight_offsets are those
    offsets on the device (an expert with others gets zeros and sets the device
    status word)."""
    return _gemv("grouped_gemv_down_int4", intermediate, w2, expert_token_offsets,
                 expert_weight_offsets, expert_widths, tokens_per_expert, int(hidden_size),
                 intermediate.shape[1] if intermediate.dim() == 2 else 0, "none", True)
