"""Writing and reading the paged 8-bit cache on gfx950 (mambo_amd/csrc/kv_cache.hip). The reference has
no counterpart.

A call's sequences are told by ``tables`` int32 [S, C] (the page that holds a sequence's tokens
[c * page_size, ...), any value outside the cache: none), ``lengths`` int32 [S] (cached tokens, the call's own
included) and, unless every sequence has as many rows, ``offsets`` int32 [S + 1] (sequence s has the rows
offsets[s] to offsets[s + 1], the last at position lengths[s] - 1). A sequence may be longer than its row of the
table: there is no page for what lies past it. All of it stays on the device: nothing is
read back, so that a step can be recorded into a HIP graph and replayed with other lengths; while a call
runs they must not change.

    cache = allocate_kv_cache(pages, kv_heads, head_dim)
    q = launch_append_kv(k, v, cache, tables, lengths, rotary=table, q=q)
    out = launch_attention_kv(q, cache, tables, lengths)                  # mambo_amd.kernels.attention
"""

from __future__ import annotations

import torch

from mambo_amd import _native
from mambo_amd.kernels.fp8_block import ROW_DTYPES
from mambo_amd.kernels.rotary import check_heads, check_int32, heads_in_place, output_heads
from mambo_amd.utils.kv_cache import KVCache
from mambo_amd.utils.rotary_table import RotaryTable


def check_cache(cache) -> KVCache:
    if not isinstance(cache, KVCache):
        raise TypeError("allocate the cache with allocate_kv_cache before launch")
    return cache


def check_tables(tables, dev) -> tuple[int, int, int]:
    """Sequences, columns and the stride of the rows of `tables`, checked."""
    if isinstance(tables, torch.Tensor) and tables.ndim == 2 and tables.dtype == torch.int32 and tables.device == dev:
        seqs, columns = tables.shape
        if seqs and columns:
            if tables.is_contiguous():
                return seqs, columns, columns
            row, value = tables.stride()
            if (columns == 1 or value == 1) and (seqs == 1 or row >= columns):
                return seqs, columns, row if seqs > 1 else columns
    raise ValueError("tables must be int32 [S,C] with unit column stride on the cache's device")


def batch_args(tables, lengths, offsets, tokens: int, dev) -> _native.KVBatchArgs:
    """The sequences of a call of `tokens` rows, checked."""
    seqs, columns, row = check_tables(tables, dev)
    check_int32(lengths, seqs, dev, "lengths")
    if offsets is not None:
        check_int32(offsets, seqs + 1, dev, "offsets")
        offsets = offsets.data_ptr()
    elif tokens % seqs:
        raise ValueError(f"without offsets every sequence has as many rows: {tokens} rows of {seqs} sequences")
    return _native.KVBatchArgs(tables.data_ptr(), row, columns, lengths.data_ptr(), offsets, seqs)


def launch_append_kv(k: torch.Tensor, v: torch.Tensor, cache: KVCache, tables: torch.Tensor, lengths: torch.Tensor, *,
                     offsets: torch.Tensor | None = None, rotary: RotaryTable | None = None,
                     positions: torch.Tensor | None = None, q: torch.Tensor | None = None, stream=None,
                     out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Store keys ``k`` and values ``v`` [T,H,D] (both float32 or both bfloat16) as the last tokens of their
    sequences, the keys rotated by ``rotary``; return the queries ``q`` [T,Hq,D] (the same type) rotated
    with them as bfloat16, or None without.

    A block of 32 tokens and a head gets the exponent e = max(ceil(log2(amax / 448)), -100) and the codes
    E4M3(x 2^-e), to nearest even. One that older tokens of the sequence are in keeps them: its exponent is the larger of the
    two, and where it grows the older codes are rounded again. A token's head with a key or value that is not finite is held
    as NaN keys and zero values, so that what sees it becomes NaN and nothing else does. Values beyond 240 * 2^120 (3.2e38) are
    held as that.

    ``positions`` int32 [T] are the rotary positions, by default those in the sequence. Rows whose position in the
    sequence would be negative (more rows than ``lengths``), or that no page is for, are not stored; rows of no
    sequence are left alone, and so are their queries in ``out``. Sequences of a call may share pages that none of
    them writes in this call. ``out`` may be ``q`` itself (bfloat16). T may be 0."""
    cache = check_cache(cache)
    dev, dim = cache.codes.device, cache.head_dim
    check_heads(k, dim, dev, "k")
    tokens = k.shape[0]
    if k.shape[1] != cache.heads:
        raise ValueError(f"k must have the cache's {cache.heads} heads")
    check_heads(v, dim, dev, "v")
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError("v must be of k's shape and type")
    if rotary is not None:
        if not isinstance(rotary, RotaryTable):
            raise TypeError("prepare the angles with prepare_rotary_table before launch")
        if rotary.size > dim or rotary.turns.device != dev:
            raise ValueError(f"angles of at most {dim} values on the cache's device")
    if positions is not None:
        if rotary is None:
            raise ValueError("positions are those of the rotation, and there is none")
        check_int32(positions, tokens, dev, "positions")
    if q is not None:
        if rotary is None:
            raise ValueError("queries are taken to be rotated: they need angles")
        check_heads(q, dim, dev, "q")
        if q.shape[0] != tokens or q.dtype != k.dtype or q.shape[1] % cache.heads:
            raise ValueError(f"q must be of k's type, [{tokens},Hq,{dim}] with a multiple of the cache's {cache.heads} heads")
    elif out is not None:
        raise ValueError("out is for queries, and there are none")
    with _native.launch_on(dev, stream):
        batch = batch_args(tables, lengths, offsets, tokens, dev)
        k, ldkt, ldkh = heads_in_place(k)
        v, ldvt, ldvh = heads_in_place(v)
        dtype = ROW_DTYPES[k.dtype]
        if q is None:
            rows = _native.KVRowsArgs(k.data_ptr(), v.data_ptr(), None, ldkt, ldkh, ldvt, ldvh, 0, 0, None, 0, 0, 0, dtype)
        else:
            shape = q.shape
            q, ldqt, ldqh = heads_in_place(q)
            out, ldot, ldoh = output_heads(out, shape, torch.bfloat16, dev)
            rows = _native.KVRowsArgs(k.data_ptr(), v.data_ptr(), q.data_ptr() if tokens else None, ldkt, ldkh, ldvt, ldvh,
                                      ldqt, ldqh, out.data_ptr(), ldot, ldoh, shape[1], dtype)
        _native.check(_native.lib().mambo_kv_append(
            rows, tokens, cache.args, batch, None if rotary is None else rotary.args,
            None if positions is None else positions.data_ptr(), _native.stream_handle(stream, dev)), "launch_append_kv")
    return out


def launch_read_kv(cache: KVCache, tables: torch.Tensor, sequences: torch.Tensor, positions: torch.Tensor, *,
                   stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values, bfloat16 [N,H,D] each, that the cache holds of the tokens at int32 ``positions`` [N]
    of int32 ``sequences`` [N] (rows of ``tables``): code * 2^e, which bfloat16 holds exactly where it is a
    normal number of its. Zeros where there is no such sequence or page; what a page holds past a sequence's tokens is
    anything. For moving a prefix elsewhere and for looking at a cache."""
    cache = check_cache(cache)
    dev = cache.codes.device
    seqs, columns, row = check_tables(tables, dev)
    if not isinstance(sequences, torch.Tensor) or sequences.ndim != 1:
        raise ValueError("sequences must be int32 [N]")
    n = sequences.shape[0]
    check_int32(sequences, n, dev, "sequences")
    check_int32(positions, n, dev, "positions")
    with _native.launch_on(dev, stream):
        batch = _native.KVBatchArgs(tables.data_ptr(), row, columns, None, None, seqs)
        k, v = torch.empty((2, n, cache.heads, cache.head_dim), dtype=torch.bfloat16, device=dev).unbind(0)
        _native.check(_native.lib().mambo_kv_read(
            cache.args, batch, sequences.data_ptr(), positions.data_ptr(), n, cache.heads, cache.head_dim, k.data_ptr(),
            v.data_ptr(), _native.stream_handle(stream, dev)), "launch_read_kv")
    return k, v
