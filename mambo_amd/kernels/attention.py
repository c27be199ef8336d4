"""Attention over the paged 8-bit cache on gfx950 (mambo_amd/csrc/attention_rows.hip for few rows of a sequence,
attention_tiles.hip for many). The reference has no counterpart.

    out[t, h] = sum_j p_j v_j,  p = softmax_j(scale * q[t, h] . k_j)   over the cached tokens j that the row sees

Sequences are told as for launch_append_kv (mambo_amd.kernels.kv_cache).
"""

from __future__ import annotations

from functools import lru_cache

import torch

from mambo_amd import _native
from mambo_amd.kernels.kv_cache import batch_args, check_cache
from mambo_amd.kernels.rotary import check_heads, heads_in_place, output_heads
from mambo_amd.utils.kv_cache import KVCache


@lru_cache(maxsize=1024)
def _workspace(pages: int, kv_heads: int, dim: int, page_size: int, seqs: int, width: int, ragged: bool, tokens: int, heads: int,
               window: int) -> int:
    """Bytes that a call of these sizes needs (asked once of each: a call of its own is a tenth of an eager launch)."""
    unused = 256  # an address that is not looked at
    cache = _native.KVCacheArgs(unused, unused, pages, kv_heads, dim, page_size, 0)
    batch = _native.KVBatchArgs(unused, width, width, unused, unused if ragged else None, seqs)
    size = _native.lib().mambo_kv_attention_workspace(cache, batch, tokens, heads, window)
    if size < 0:
        _native.check(size, "launch_attention_kv")
    return size


def launch_attention_kv(q: torch.Tensor, cache: KVCache, tables: torch.Tensor, lengths: torch.Tensor, *,
                        offsets: torch.Tensor | None = None, scale: float | None = None, causal: bool = True,
                        window: int = 0, return_lse: bool = False, stream=None, out: torch.Tensor | None = None):
    """Attention of bfloat16 queries ``q`` [T,Hq,D] over the cached keys and values of their sequences; query head h
    reads key/value head h // (Hq / H). Returns bfloat16 [T,Hq,D], or (that, float32 [T,Hq]) with
    ``return_lse``: the logarithm of the sum of the exponentials of a row's scores.

    Row i of a sequence's n stands at position lengths[s] - n + i and sees the tokens up to itself (``causal``), no more
    than the last ``window`` of them where that is not 0, or all of the sequence's. A row that sees none (a sequence of length
    0, more rows than tokens, no page) becomes zeros, its lse -inf. ``scale`` (positive) defaults to D ** -0.5.

    Scores, the running sum and the output are float32; the probabilities are rounded to bfloat16 (2^-8 of each at most) for the
    product with the values, the result once to bfloat16. Results do not vary from run to run. Rows of no sequence are not
    written: they stay what they were in ``out``, and are undefined without. ``out`` must not overlap ``q``. T may be 0."""
    cache = check_cache(cache)
    dev, dim = cache.codes.device, cache.head_dim
    check_heads(q, dim, dev, "q")
    if q.dtype != torch.bfloat16:
        raise ValueError("q must be bfloat16")
    shape = q.shape
    tokens, heads, _ = shape
    if heads % cache.heads:
        raise ValueError(f"q must have a multiple of the cache's {cache.heads} heads, got {heads}")
    scale = dim ** -0.5 if scale is None else float(scale)
    window = int(window)
    if window < 0 or (window and not causal):
        raise ValueError("a window is positive, and of causal attention")
    with _native.launch_on(dev, stream):
        batch = batch_args(tables, lengths, offsets, tokens, dev)
        q, ldqt, ldqh = heads_in_place(q)
        if q.data_ptr() % 16 or ldqt % 8 or ldqh % 8:
            q, ldqt, ldqh = torch.empty(shape, dtype=q.dtype, device=dev).copy_(q), heads * dim, dim
        out, ldot, ldoh = output_heads(out, shape, torch.bfloat16, dev)
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=dev) if return_lse else None
        size = _workspace(cache.pages, cache.heads, dim, cache.page_size, batch.seqs, batch.width, offsets is not None, tokens,
                          heads, window)
        workspace = torch.empty(size, dtype=torch.uint8, device=dev).data_ptr() if size else None
        _native.check(_native.lib().mambo_kv_attention(
            q.data_ptr(), tokens, heads, dim, ldqt, ldqh, cache.args, batch, scale, bool(causal), window, out.data_ptr(),
            ldot, ldoh, None if lse is None else lse.data_ptr(), workspace, size,
            _native.stream_handle(stream, dev)), "launch_attention_kv")
    return (out, lse) if return_lse else out
