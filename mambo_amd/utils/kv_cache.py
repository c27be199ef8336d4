"""The paged 8-bit cache of keys and values that the append writes and attention reads.

Pages of ``page_size`` tokens, in any order; a block of 32 tokens of one key/value head holds E4M3 codes
and two powers of two, one for its keys and one for its values. The order of the codes in a block is
private (mambo_amd/csrc/kv_cache.h); pages may be copied whole, [page] of both tensors. The reference has no
counterpart.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from mambo_amd import _native

KV_BLOCK = 32  # MAMBO_KV_BLOCK
MAX_HEAD_DIM = 256  # MAMBO_KV_MAX_DIM


@dataclass(frozen=True)
class KVCache:
    """``codes`` uint8 [pages, heads, page_size / 32, 2 * 32 * D] (D: head_dim rounded up to 32) and ``scales``
    uint8 [pages, heads, page_size / 32, 2], E8M0 of the keys and the values of each block."""

    codes: torch.Tensor
    scales: torch.Tensor
    heads: int
    head_dim: int
    page_size: int

    def __post_init__(self):
        pages, blocks = self.codes.shape[0], self.page_size // KV_BLOCK
        size = _native.lib().mambo_kv_cache_bytes(pages, self.heads, self.head_dim, self.page_size)
        shape = (pages, self.heads, blocks, size // max(1, pages * self.heads * blocks))
        for t, want in ((self.codes, shape), (self.scales, (*shape[:3], 2))):
            if size == 0 or tuple(t.shape) != want or t.dtype != torch.uint8 or not t.is_contiguous() \
                    or t.device != self.codes.device:
                raise ValueError(f"a cache of these sizes has contiguous uint8 tensors on one device, one of them {list(want)}")
        object.__setattr__(self, "args", _native.KVCacheArgs(
            self.codes.data_ptr(), self.scales.data_ptr(), self.codes.shape[0], self.heads, self.head_dim,
            self.page_size, 0))

    def __reduce__(self):  # a copy's tensors are its own, and so are the addresses that it hands to the kernels
        return KVCache, (self.codes, self.scales, self.heads, self.head_dim, self.page_size)

    @property
    def pages(self) -> int:
        return self.codes.shape[0]


def allocate_kv_cache(pages: int, heads: int, head_dim: int, *, page_size: int = 64, device=None) -> KVCache:
    """An empty cache on a GPU (default: the current one): ``head_dim`` a multiple of 8 up to 256, ``page_size``
    a power of two from 32 to 65536 tokens. A page takes 2 * heads * page_size * D bytes (D: head_dim rounded
    up to 32) and a 512th of that for the scales of heads of 128 or so."""
    pages, heads, head_dim, page_size = int(pages), int(heads), int(head_dim), int(page_size)
    size = _native.lib().mambo_kv_cache_bytes(pages, heads, head_dim, page_size)
    if size == 0:
        raise ValueError(f"no cache of {pages} pages of {page_size} tokens, {heads} heads of {head_dim}: head_dim must be a "
                         f"multiple of 8 up to {MAX_HEAD_DIM}, page_size a power of two from {KV_BLOCK} to 65536")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if device.type != "cuda":
        raise ValueError("the cache must be on a GPU")
    blocks = page_size // KV_BLOCK
    codes = torch.zeros((pages, heads, blocks, size // (pages * heads * blocks)), dtype=torch.uint8, device=device)
    scales = torch.zeros((pages, heads, blocks, 2), dtype=torch.uint8, device=device)
    return KVCache(codes, scales, heads, head_dim, page_size)
