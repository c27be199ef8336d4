"""E4M3 products with an f32 scale for each block of 128 on gfx950: the quantizer of the rows
and the product with a prepared weight (mambo_amd.utils.fp8_block_weight). The kernels are
hand-written HIP (mambo_amd/csrc/fp8_block.hip) behind the C ABI. The reference has no counterpart.

    out[m, n] = sum_g xs[m, g] * ws[n // 128, g] * sum_{k in group g} xv[m, k] * w[n, k]

over the groups g of 128 along K, summed in float32 in a fixed order.
"""

from __future__ import annotations

import torch

from mambo_amd import _native
from mambo_amd.utils.fp8_block_weight import FP8_BLOCK, Fp8BlockWeight

ROW_DTYPES = {torch.float32: _native.DTYPE_F32, torch.bfloat16: _native.DTYPE_BF16}


def launch_quantize_fp8_block(x: torch.Tensor, *, stream=None, out: tuple[torch.Tensor, torch.Tensor] | None = None
                              ) -> tuple[torch.Tensor, torch.Tensor]:
    """Return uint8 [M,K] E4M3 codes and float32 [M,ceil(K/128)] scales of ``x``.

    ``x`` is float32 or bfloat16 [M,K] on the GPU, K a multiple of 16, M >= 0. A group of 128 along K
    (the last may be shorter) has the scale max(amax / 448, 2^-100) and the codes of x / scale,
    which is 448 x / amax in float32, rounded to nearest even; a group that holds a NaN or an infinity becomes NaN. Row-strided
    inputs are read in place. The scales are laid out group by group (strides (1, M)); ``out``
    optionally supplies codes with unit column stride and scales of either order.
    """
    if not isinstance(x, torch.Tensor) or x.ndim != 2 or x.dtype not in ROW_DTYPES or x.shape[1] % 16 or x.shape[1] < 16:
        raise ValueError("activation must be float32 or bfloat16 [M,K] with K a multiple of 16")
    if not x.is_cuda:
        raise ValueError("activation must be a GPU tensor")
    (m, k), dev = x.shape, x.device
    groups = -(-k // FP8_BLOCK)
    with _native.launch_on(dev, stream):
        if not x.is_contiguous() and not plain_rows(x):
            x = x.contiguous()
        if out is None:
            values = torch.empty((m, k), dtype=torch.uint8, device=dev)
            # a group's scales next to each other: the products copy those of 64 rows in one piece
            scales = torch.empty_strided((m, groups), (1, m), dtype=torch.float32, device=dev)
            ldv, (lds, gss) = k, (1, m)
        else:
            values, scales = out
            if values.shape != (m, k) or values.dtype != torch.uint8 or scales.shape != (m, groups) \
                    or scales.dtype != torch.float32 or values.device != dev or scales.device != dev \
                    or not plain_rows(values) or not (plain_rows(scales) or plain_rows(scales.t())):
                raise ValueError("out must be (uint8 [M,K] with unit column stride, float32 [M,ceil(K/128)] with unit "
                                 "row or column stride) on the activation's device")
            ldv, (lds, gss) = row_stride(values), scale_strides(scales)
        _native.check(_native.lib().mambo_quantize_fp8_block(
            x.data_ptr(), ROW_DTYPES[x.dtype], m, k, row_stride(x), values.data_ptr(), ldv, scales.data_ptr(), lds, gss,
            _native.stream_handle(stream, dev)), "launch_quantize_fp8_block")
    return values, scales


def row_stride(t: torch.Tensor) -> int:
    """Stride of the rows; of a single row, whose stride torch leaves open, its length."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def plain_rows(t: torch.Tensor) -> bool:
    """Whether rows do not overlap and their elements are next to each other."""
    return (t.shape[1] <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1])


def scale_strides(t: torch.Tensor) -> tuple[int, int]:
    """Strides of the rows and the groups of scales [M,G] that are plain rows of groups or of rows."""
    if t.shape[1] <= 1 or t.stride(1) == 1:
        return row_stride(t), 1
    return 1, t.stride(1)


def rows_in_place(t: torch.Tensor, align: int) -> torch.Tensor:
    """`t` itself where the kernels can read its rows as they lie (elements next to each other, rows
    apart and `align` bytes aligned), else a contiguous copy."""
    if t.is_contiguous():
        if t.data_ptr() % align == 0 and t.shape[1] * t.element_size() % align == 0:
            return t
    elif plain_rows(t) and t.data_ptr() % align == 0 and row_stride(t) * t.element_size() % align == 0:
        return t
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def block_activations(x_values, x_scales, k: int, dev) -> tuple[torch.Tensor, torch.Tensor, tuple[int, int], int]:
    """Validate E4M3 rows [M,K] and scales [M,ceil(K/128)] on `dev`; return them in a form that the
    kernels read in place, the scales' strides, and M."""
    if not isinstance(x_values, torch.Tensor) or x_values.ndim != 2 or x_values.dtype != torch.uint8 \
            or x_values.shape[1] != k:
        raise ValueError(f"x_values must be uint8 [M,{k}]")
    m = x_values.shape[0]
    if not isinstance(x_scales, torch.Tensor) or x_scales.shape != (m, -(-k // FP8_BLOCK)) \
            or x_scales.dtype != torch.float32:
        raise ValueError("x_scales must be float32 [M,ceil(K/128)]")
    if x_values.device != dev or x_scales.device != dev:
        raise ValueError("x_values and x_scales must be on the weight's device")
    strides = x_scales.stride()
    if strides != (1, m):  # as the quantizer lays them out
        if not plain_rows(x_scales) and not plain_rows(x_scales.t()):
            x_scales = x_scales.contiguous()
        strides = scale_strides(x_scales)
    return rows_in_place(x_values, 16), x_scales, strides, m


def product_output(out, rows: int, n: int, dtype, dev) -> torch.Tensor:
    """The given output, checked, or a new one."""
    if dtype not in ROW_DTYPES:
        raise ValueError("out_dtype must be float32 or bfloat16")
    if out is None:
        return torch.empty((rows, n), dtype=dtype, device=dev)
    if not isinstance(out, torch.Tensor) or tuple(out.shape) != (rows, n) or out.dtype != dtype or out.device != dev \
            or not plain_rows(out):
        raise ValueError(f"out must be {dtype} [{rows},{n}] with unit column stride on the rows' device")
    return out


def launch_fp8_block_matmul(x_values: torch.Tensor, x_scales: torch.Tensor, weight: Fp8BlockWeight, *,
                            out_dtype: torch.dtype = torch.float32, stream=None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """Multiply rows from launch_quantize_fp8_block by a prepared weight: [M,N] of ``out_dtype``
    (float32 or bfloat16, rounded once from the float32 sums). bfloat16 outputs are computed by the
    FP8 matrix instructions, which leave out up to 8.5e-4 of the largest of eight consecutive products
    (5e-5 of the sums in the 2-norm), float32 ones by the bfloat16 instructions, which add more exactly
    and at half the rate. M may be 0. Rows that are not 16-byte aligned are copied first; ``out`` optionally
    supplies the output."""
    if not isinstance(weight, Fp8BlockWeight):
        raise TypeError("prepare FP8 weights with prepare_fp8_block_weight before launch")
    if weight.experts != 1:
        raise ValueError("a weight of several experts takes launch_fp8_block_matmul_experts")
    packed, n, k = weight.packed, weight.n, weight.k
    dev = packed.device
    with _native.launch_on(dev, stream):
        x_values, x_scales, strides, m = block_activations(x_values, x_scales, k, dev)
        out = product_output(out, m, n, out_dtype, dev)
        _native.check(_native.lib().mambo_fp8_block_matmul(
            x_values.data_ptr(), row_stride(x_values), x_scales.data_ptr(), *strides, m, packed.data_ptr(),
            weight.scales.data_ptr(), n, k, out.data_ptr(), ROW_DTYPES[out_dtype], row_stride(out),
            _native.stream_handle(stream, dev)), "launch_fp8_block_matmul")
    return out
