"""The operators of a layer of experts on gfx950: the router's plan, the products grouped by
expert and the join of their rows (mambo_amd/csrc/experts.hip, fp8_block.hip, iq3s_experts.hip).
Nothing is read back to the host: how many rows an expert has stays on the device. The reference has
no counterpart.

    plan = launch_route_experts(logits, top_k)
    values, scales = launch_quantize_fp8_block(x)                       # a token's row once
    y = launch_fp8_block_matmul_experts(values, scales, w, plan.offsets, rows=plan.rows)
    out = launch_combine_experts(y, plan.slots, plan.weights)
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from mambo_amd import _native
from mambo_amd.kernels.fp8_block import (ROW_DTYPES, block_activations, plain_rows, product_output, row_stride,
                                         rows_in_place)
from mambo_amd.utils.fp8_block_weight import Fp8BlockWeight
from mambo_amd.utils.iq3_s_weight import IQ3SExperts, IQ3_S_BLOCK_VALUES

MAX_EXPERTS = 1024  # MAMBO_MAX_EXPERTS
MAX_TOP_K = 64  # MAMBO_MAX_TOP_K


class ExpertPlan(NamedTuple):
    """What launch_route_experts decides for M tokens of ``top_k`` choices, R = M * top_k rows.

    ids: int32 [M, top_k], the chosen experts in falling order (-1: none was left)
    weights: float32 [M, top_k], their weights (0 beside -1)
    offsets: int32 [E + 1]; expert e has the rows offsets[e] to offsets[e + 1]
    rows: int32 [R], the token of each row, ascending within an expert (-1 past offsets[E])
    slots: int32 [M, top_k], the row of each choice (-1: none)
    """

    ids: torch.Tensor
    weights: torch.Tensor
    offsets: torch.Tensor
    rows: torch.Tensor
    slots: torch.Tensor


def launch_route_experts(logits: torch.Tensor, top_k: int, *, renormalize: bool = True, stream=None) -> ExpertPlan:
    """Choose each token's ``top_k`` experts from router logits [M, E] (float32 or bfloat16, E <= 1024,
    top_k <= min(E, 64)) and lay the rows out by expert.

    The largest logits are chosen, ties to the lowest expert; one that is -inf or NaN never is, so a
    token may have fewer choices, or none. ``weights`` is the softmax over the chosen experts
    (``renormalize``) or over all that the token may take. M may be 0.
    """
    if not isinstance(logits, torch.Tensor) or logits.ndim != 2 or logits.dtype not in ROW_DTYPES:
        raise ValueError("logits must be float32 or bfloat16 [M,E]")
    if not logits.is_cuda:
        raise ValueError("logits must be a GPU tensor")
    (m, experts), dev = logits.shape, logits.device
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"between 1 and {MAX_EXPERTS} experts, got {experts}")
    if not 1 <= top_k <= min(experts, MAX_TOP_K):
        raise ValueError(f"top_k must be in [1, min(E, {MAX_TOP_K})], got {top_k}")
    with _native.launch_on(dev, stream):
        if not logits.is_contiguous() and not plain_rows(logits):
            logits = logits.contiguous()
        # int32 planes of one buffer: allocated and taken apart in few calls
        ids, slots, rows, weights = torch.empty((4, m, top_k), dtype=torch.int32, device=dev).unbind(0)
        rows, weights = rows.view(-1), weights.view(torch.float32)
        offsets = torch.empty(experts + 1, dtype=torch.int32, device=dev)
        _native.check(_native.lib().mambo_route_experts(
            logits.data_ptr(), ROW_DTYPES[logits.dtype], row_stride(logits), m, experts, top_k, bool(renormalize),
            ids.data_ptr(), weights.data_ptr(), offsets.data_ptr(), rows.data_ptr(), slots.data_ptr(),
            _native.stream_handle(stream, dev)), "launch_route_experts")
    return ExpertPlan(ids, weights, offsets, rows, slots)


def _plan_tensors(offsets, rows, m: int, experts: int, dev) -> int:
    """Validate the plan of a grouped product; return its number of output rows."""
    if not isinstance(offsets, torch.Tensor) or offsets.shape != (experts + 1,) or offsets.dtype != torch.int32 \
            or not offsets.is_contiguous() or offsets.device != dev:
        raise ValueError(f"offsets must be contiguous int32 [{experts + 1}] on the rows' device")
    if rows is None:
        return m
    if not isinstance(rows, torch.Tensor) or rows.ndim != 1 or rows.dtype != torch.int32 or not rows.is_contiguous() \
            or rows.device != dev:
        raise ValueError("rows must be contiguous int32 [R] on the rows' device")
    if m == 0 and rows.shape[0]:
        raise ValueError("rows of no tokens")
    return rows.shape[0]


def launch_fp8_block_matmul_experts(x_values: torch.Tensor, x_scales: torch.Tensor, weight: Fp8BlockWeight,
                                    offsets: torch.Tensor, *, rows: torch.Tensor | None = None,
                                    out_dtype: torch.dtype = torch.float32, stream=None,
                                    out: torch.Tensor | None = None) -> torch.Tensor:
    """launch_fp8_block_matmul grouped by expert: output row i, of expert e where
    offsets[e] <= i < offsets[e + 1], is input row rows[i] times weight e. Returns [R,N].

    ``x_values`` / ``x_scales``: the tokens' rows, read where ``rows`` points, or (``rows`` None) the
    rows in the experts' order themselves. Rows past offsets[E] come out as zeros; experts without
    rows cost nothing. ``offsets`` and ``rows`` are a plan's (launch_route_experts)."""
    if not isinstance(weight, Fp8BlockWeight):
        raise TypeError("prepare FP8 weights with prepare_fp8_block_weight before launch")
    dev = weight.packed.device
    with _native.launch_on(dev, stream):
        x_values, x_scales, strides, m = block_activations(x_values, x_scales, weight.k, dev)
        r = _plan_tensors(offsets, rows, m, weight.experts, dev)
        out = product_output(out, r, weight.n, out_dtype, dev)
        _native.check(_native.lib().mambo_fp8_block_matmul_experts(
            x_values.data_ptr(), row_stride(x_values), x_scales.data_ptr(), *strides, m,
            None if rows is None else rows.data_ptr(), r, offsets.data_ptr(), weight.experts, weight.packed.data_ptr(),
            weight.scales.data_ptr(), weight.n, weight.k, out.data_ptr(), ROW_DTYPES[out_dtype], row_stride(out),
            _native.stream_handle(stream, dev)), "launch_fp8_block_matmul_experts")
    return out


def launch_iq3_s_fp8_matmul_experts(x_values: torch.Tensor, x_scales: torch.Tensor, weight: IQ3SExperts,
                                    offsets: torch.Tensor, *, rows: torch.Tensor | None = None,
                                    out_dtype: torch.dtype = torch.float32, stream=None,
                                    out: torch.Tensor | None = None) -> torch.Tensor:
    """launch_iq3_s_fp8_matmul grouped by expert, as launch_fp8_block_matmul_experts is:
    ``x_values`` / ``x_scales`` from launch_quantize_fp8 (MXFP8), ``weight`` from
    prepare_iq3_s_experts."""
    if not isinstance(weight, IQ3SExperts):
        raise TypeError("prepare IQ3_S experts with prepare_iq3_s_experts before launch")
    k, dev = weight.blocks * IQ3_S_BLOCK_VALUES, weight.packed.device
    with _native.launch_on(dev, stream):
        if not isinstance(x_values, torch.Tensor) or x_values.ndim != 2 or x_values.dtype != torch.uint8 \
                or x_values.shape[1] != k:
            raise ValueError(f"x_values must be uint8 [M,{k}]")
        m = x_values.shape[0]
        if not isinstance(x_scales, torch.Tensor) or tuple(x_scales.shape) != (m, k // 32) \
                or x_scales.dtype != torch.uint8:
            raise ValueError("x_scales must be uint8 [M,K/32]")
        if x_values.device != dev or x_scales.device != dev:
            raise ValueError("the rows, their scales and the weight must be on the same device")
        x_values, x_scales = rows_in_place(x_values, 16), rows_in_place(x_scales, 8)
        r = _plan_tensors(offsets, rows, m, weight.experts, dev)
        out = product_output(out, r, weight.n, out_dtype, dev)
        _native.check(_native.lib().mambo_iq3s_fp8_matmul_experts(
            x_values.data_ptr(), row_stride(x_values), x_scales.data_ptr(), row_stride(x_scales), m,
            None if rows is None else rows.data_ptr(), r, offsets.data_ptr(), weight.experts, weight.packed.data_ptr(),
            weight.packed.stride(0), weight.n, weight.blocks, out.data_ptr(), ROW_DTYPES[out_dtype], row_stride(out),
            _native.stream_handle(stream, dev)), "launch_iq3_s_fp8_matmul_experts")
    return out


def launch_combine_experts(y: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor, *,
                           out_dtype: torch.dtype | None = None, stream=None,
                           out: torch.Tensor | None = None) -> torch.Tensor:
    """Return out[t] = sum_j weights[t, j] * y[slots[t, j]] as [M,N] of ``out_dtype`` (default: that of
    ``y``), added in float32 in order of j.

    ``y`` [R,N] float32 or bfloat16, ``slots`` int32 and ``weights`` float32 [M, top_k] as in a plan; a
    choice whose slot is -1 (or outside y) adds nothing, and a token without any becomes zeros."""
    if not isinstance(y, torch.Tensor) or y.ndim != 2 or y.dtype not in ROW_DTYPES or y.shape[1] < 1:
        raise ValueError("y must be float32 or bfloat16 [R,N]")
    if not y.is_cuda:
        raise ValueError("y must be a GPU tensor")
    dev = y.device
    if not isinstance(slots, torch.Tensor) or slots.ndim != 2 or slots.dtype != torch.int32 \
            or not 1 <= slots.shape[1] <= MAX_TOP_K or slots.device != dev:
        raise ValueError(f"slots must be int32 [M,top_k] with top_k in [1, {MAX_TOP_K}] on y's device")
    if not isinstance(weights, torch.Tensor) or weights.shape != slots.shape or weights.dtype != torch.float32 \
            or weights.device != dev:
        raise ValueError("weights must be float32 of the shape of slots on y's device")
    m, top_k = slots.shape
    out_dtype = y.dtype if out_dtype is None else out_dtype
    with _native.launch_on(dev, stream):
        y = y if y.is_contiguous() or plain_rows(y) else y.contiguous()
        slots, weights = slots.contiguous(), weights.contiguous()
        out = product_output(out, m, y.shape[1], out_dtype, dev)
        _native.check(_native.lib().mambo_combine_experts(
            y.data_ptr(), ROW_DTYPES[y.dtype], row_stride(y), y.shape[0], slots.data_ptr(), weights.data_ptr(), m,
            top_k, y.shape[1], out.data_ptr(), ROW_DTYPES[out_dtype], row_stride(out),
            _native.stream_handle(stream, dev)), "launch_combine_experts")
    return out
