"""Rotary positions on gfx950 (mambo_amd/csrc/kv_cache.hip). The reference has no counterpart.

    pair (a, b) -> magnitude * (a cos - b sin, a sin + b cos) of the angle position * frequency
"""

from __future__ import annotations

import torch

from mambo_amd import _native
from mambo_amd.kernels.fp8_block import ROW_DTYPES
from mambo_amd.utils.rotary_table import MAX_ROTARY_DIM, RotaryTable


def heads_in_place(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """`t` [T,H,D] itself where heads do not overlap and their values are next to each other, else a contiguous
    copy, and the strides of its tokens and heads (of a single one, whose stride torch leaves open, its length)."""
    tokens, heads, dim = t.shape
    if not t.is_contiguous():
        token, head, value = t.stride()
        if heads == 1:
            head = dim
        if tokens == 1:
            token = head * heads
        if (dim <= 1 or value == 1) and head >= dim and token >= head * (heads - 1) + dim:
            return t, token, head
        t = t.contiguous()
    return t, heads * dim, dim


def check_heads(t, dim: int | None, dev, what: str) -> None:
    if not isinstance(t, torch.Tensor) or t.ndim != 3 or t.dtype not in ROW_DTYPES or t.shape[1] < 1 \
            or (dim is not None and t.shape[2] != dim):
        raise ValueError(f"{what} must be float32 or bfloat16 [T,H,{'D' if dim is None else dim}]")
    if not t.is_cuda:
        raise ValueError(f"{what} must be a GPU tensor")
    if dev is not None and t.device != dev:
        raise ValueError(f"{what} must be on the same device")


def check_int32(t, size: int, dev, what: str) -> None:
    if not isinstance(t, torch.Tensor) or t.shape != (size,) or t.dtype != torch.int32 or t.device != dev \
            or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous int32 [{size}] on the rows' device")


def output_heads(out, shape, dtype, dev) -> tuple[torch.Tensor, int, int]:
    """The given output, checked, or a new one, and its strides."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=dev), shape[1] * shape[2], shape[2]
    if isinstance(out, torch.Tensor) and out.shape == shape and out.dtype == dtype and out.device == dev:
        same, token, head = heads_in_place(out)
        if same is out:
            return out, token, head
    raise ValueError(f"out must be {dtype} {list(shape)} with heads that do not overlap, on the rows' device")


def launch_rotary(x: torch.Tensor, positions: torch.Tensor, table: RotaryTable, *, out_dtype: torch.dtype | None = None,
                  stream=None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate the heads of ``x`` [T,H,D] (float32 or bfloat16, D up to 1024) by int32 ``positions`` [T].

    The first ``table.size`` values of a head are rotated in float32 and multiplied by the table's magnitude,
    the others copied; each is rounded once to ``out_dtype`` (default: that of ``x``). T may be 0. Tokens and heads
    may be apart; other strides are copied first. ``out`` optionally supplies the output; it may be ``x``
    itself, and must not overlap it otherwise."""
    check_heads(x, None, None, "x")
    if not isinstance(table, RotaryTable):
        raise TypeError("prepare the angles with prepare_rotary_table before launch")
    shape, dev = x.shape, x.device
    tokens, heads, dim = shape
    if dim > MAX_ROTARY_DIM or table.size > dim:
        raise ValueError(f"heads of {table.size} to {MAX_ROTARY_DIM} values, got {dim}")
    if table.turns.device != dev:
        raise ValueError("the angles must be on the rows' device")
    check_int32(positions, tokens, dev, "positions")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in ROW_DTYPES:
        raise ValueError("out_dtype must be float32 or bfloat16")
    with _native.launch_on(dev, stream):
        x, ldt, ldh = heads_in_place(x)
        out, ldot, ldoh = output_heads(out, shape, out_dtype, dev)
        _native.check(_native.lib().mambo_rotary(
            x.data_ptr(), ROW_DTYPES[x.dtype], tokens, heads, dim, ldt, ldh, positions.data_ptr(), table.args,
            out.data_ptr(), ROW_DTYPES[out_dtype], ldot, ldoh, _native.stream_handle(stream, dev)),
            "launch_rotary")
    return out
