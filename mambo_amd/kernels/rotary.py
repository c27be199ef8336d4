"""Rotary positions on gfx950 (mambo_amd/csrc/kv_cache.hip). The reference has no counterpart.

    pair (a, b) -> magnitude * (a cos - b sin, a sin + b cos) of the angle position * frequency
"""

from __future__ import annotations

import torch

from mambo_amd import _native
from mambo_amd.kernels.fp8_block import ROW_DTYPES
from mambo_amd.utils.rotary_table import MAX_ROTARY_DIM, RotaryTable


def heads_in_place(t: torch.Tensor) -> torch.Tensor:
    """`t` [T,H,D] itself where heads do not overlap and their values are next to each other, else a
    contiguous copy."""
    tokens, heads, dim = t.shape
    if (dim <= 1 or t.stride(2) == 1) and (heads <= 1 or t.stride(1) >= dim) \
            and (tokens <= 1 or t.stride(0) >= (t.stride(1) * (heads - 1) + dim if heads > 1 else dim)):
        return t
    return t.contiguous()


def head_strides(t: torch.Tensor) -> tuple[int, int]:
    """Strides of the tokens and the heads; of a single one, whose stride torch leaves open, its length."""
    tokens, heads, dim = t.shape
    head = t.stride(1) if heads > 1 else dim
    return (t.stride(0) if tokens > 1 else head * heads), head


def check_heads(t, dim: int | None, dev, what: str) -> None:
    if not isinstance(t, torch.Tensor) or t.ndim != 3 or t.dtype not in ROW_DTYPES or t.shape[1] < 1 \
            or (dim is not None and t.shape[2] != dim):
        raise ValueError(f"{what} must be float32 or bfloat16 [T,H,{'D' if dim is None else dim}]")
    if not t.is_cuda:
        raise ValueError(f"{what} must be a GPU tensor")
    if dev is not None and t.device != dev:
        raise ValueError(f"{what} must be on the same device")


def check_int32(t, shape: tuple[int, ...], dev, what: str) -> None:
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != shape or t.dtype != torch.int32 or t.device != dev \
            or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous int32 {list(shape)} on the rows' device")


def output_heads(out, shape, dtype, dev) -> torch.Tensor:
    """The given output, checked, or a new one."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    if not isinstance(out, torch.Tensor) or tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != dev \
            or heads_in_place(out) is not out:
        raise ValueError(f"out must be {dtype} {list(shape)} with heads that do not overlap, on the rows' device")
    return out


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
    (tokens, heads, dim), dev = x.shape, x.device
    if dim > MAX_ROTARY_DIM or table.size > dim:
        raise ValueError(f"heads of {table.size} to {MAX_ROTARY_DIM} values, got {dim}")
    if table.turns.device != dev:
        raise ValueError("the angles must be on the rows' device")
    check_int32(positions, (tokens,), dev, "positions")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in ROW_DTYPES:
        raise ValueError("out_dtype must be float32 or bfloat16")
    with _native.launch_on(dev, stream):
        x = heads_in_place(x)
        out = output_heads(out, (tokens, heads, dim), out_dtype, dev)
        _native.check(_native.lib().mambo_rotary(
            x.data_ptr(), ROW_DTYPES[x.dtype], tokens, heads, dim, *head_strides(x), positions.data_ptr(), table.args,
            out.data_ptr(), ROW_DTYPES[out_dtype], *head_strides(out), _native.stream_handle(stream, dev)),
            "launch_rotary")
    return out
