"""E4M3 weights with an f32 scale for each block of 128 x 128, as 8-bit checkpoints hold them.

``prepare_fp8_block_weight`` brings the codes once into the layout that the products read (tiles
of 32 rows x 128 of K in the order of the matrix instruction's operand, mambo_amd/csrc/fp8_block.hip),
for one weight or for one per expert. The reference has no counterpart.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from mambo_amd import _native

FP8_BLOCK = 128


@dataclass(frozen=True)
class Fp8BlockWeight:
    """A prepared weight: ``packed`` uint8 (private layout), ``scales`` float32
    [experts, ceil(N/128), ceil(K/128)], and the shape of the codes."""

    packed: torch.Tensor
    scales: torch.Tensor
    experts: int
    n: int
    k: int


def prepare_fp8_block_weight(codes: torch.Tensor, scales: torch.Tensor, *, stream=None) -> Fp8BlockWeight:
    """Prepare E4M3 codes [N, K], or [E, N, K] for experts, with scales float32
    [.., ceil(N/128), ceil(K/128)]: a weight is code * scale of its block.

    ``codes`` is uint8 or float8_e4m3fn on the GPU, K a multiple of 16; other strides than a
    contiguous K are copied first. The result holds the codes once more and its own copy of the
    scales, so that the arguments can be freed or changed.
    """
    if not isinstance(codes, torch.Tensor) or codes.dtype not in (torch.uint8, torch.float8_e4m3fn) \
            or codes.ndim not in (2, 3):
        raise ValueError("codes must be uint8 or float8_e4m3fn [N,K] or [E,N,K]")
    if not codes.is_cuda:
        raise ValueError("codes must be a GPU tensor")
    n, k = int(codes.shape[-2]), int(codes.shape[-1])
    blocks = (-(-n // FP8_BLOCK), -(-k // FP8_BLOCK))
    if not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32 \
            or tuple(scales.shape) != (*codes.shape[:-2], *blocks):
        raise ValueError(f"scales must be float32 {[*codes.shape[:-2], *blocks]}")
    if scales.device != codes.device:
        raise ValueError("codes and scales must be on the same device")
    dev = codes.device
    with _native.launch_on(dev, stream):
        codes = codes.view(torch.uint8) if codes.dtype != torch.uint8 else codes
        if codes.ndim == 2:
            codes, scales = codes[None], scales[None]
        if codes.stride(2) != 1:
            codes = codes.contiguous()
        lib = _native.lib()
        size = lib.mambo_fp8_block_packed_bytes(codes.shape[0], n, k)
        packed = torch.empty(size, dtype=torch.uint8, device=dev)
        _native.check(lib.mambo_fp8_block_pack(codes.data_ptr(), codes.shape[0], n, k, codes.stride(0), codes.stride(1),
                                               packed.data_ptr(), _native.stream_handle(stream)),
                      "prepare_fp8_block_weight")
        return Fp8BlockWeight(packed, scales.clone(memory_format=torch.contiguous_format), int(codes.shape[0]), n, k)
