"""Attention over the paged 8-bit cache on the GPU against 64 bits, within what its roundings allow: single tokens,
drafts, prompts and pieces of them, windows, empty sequences, pages that are missing."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import kv_reference as ref
from test_gpu_kv_cache import new_cache, read_all, rows_of

pytestmark = pytest.mark.gpu


def attention():
    from mambo_amd.kernels.attention import launch_attention_kv
    return launch_attention_kv


def filled(gpu, rng, lengths, heads, dim, page, extra=1):
    """(cache, tables, keys and values that it holds by sequence)."""
    from mambo_amd.kernels.kv_cache import launch_append_kv
    host, pages = ref.tables_of(rng, lengths, page, extra=extra)
    tables, cache = ref.device(gpu, host)[0], new_cache(pages, heads, dim, page)
    n = sum(lengths)
    k, v = rows_of(rng, n, heads, dim, torch.bfloat16).to(gpu), rows_of(rng, n, heads, dim, torch.bfloat16).to(gpu)
    launch_append_kv(k, v, cache, tables, *ref.device(gpu, np.array(lengths, np.int32)),
                     offsets=ref.device(gpu, ref.offsets_of(lengths))[0])
    return cache, tables, *read_all(cache, tables, lengths)


def check(out, lse, q, keys, values, counts, group, scale=None, causal=True, window=0, left_out=None):
    cuts = ref.offsets_of(counts)
    got, got_lse, q64 = out.double().cpu().numpy(), lse.double().cpu().numpy(), q.double().cpu().numpy()
    scale = q.shape[2] ** -0.5 if scale is None else scale
    for s in range(len(counts)):
        part = slice(cuts[s], cuts[s + 1])
        want, want_lse, bound, lse_bound = ref.attend(q64[part], keys[s], values[s], group, scale, causal, window,
                                                      None if left_out is None else left_out[s])
        off = np.abs(got[part] - want)
        assert (off <= bound).all(), (s, float((off / np.maximum(bound, 1e-300)).max()))
        some = np.isfinite(want_lse)
        assert np.array_equal(some, np.isfinite(got_lse[part])) and (got_lse[part][~some] == -np.inf).all()
        assert (np.abs(got_lse[part][some] - want_lse[some]) <= lse_bound[some]).all()


# lengths, rows of each sequence, key/value heads, group, head size, page, window
UNIFORM = [
    ([1], 1, 1, 1, 8, 32, 0), ([31], 1, 2, 4, 64, 32, 0), ([32], 1, 1, 1, 32, 32, 0), ([33, 7], 1, 8, 4, 128, 64, 0),
    ([1000], 1, 8, 4, 128, 64, 0), ([500, 0, 3, 129], 1, 2, 8, 128, 32, 0), ([70, 300], 1, 3, 7, 80, 128, 0),
    ([200], 1, 2, 16, 96, 32, 0), ([200, 90], 1, 2, 32, 64, 32, 0), ([150], 1, 1, 5, 256, 64, 0), ([150], 1, 2, 3, 160, 64, 0),
    ([90], 1, 1, 2, 192, 32, 0), ([90, 45], 1, 1, 2, 224, 32, 0), ([300, 290, 44], 5, 2, 6, 64, 32, 0), ([300, 280], 4, 2, 4, 128, 64, 0),
    ([400, 30], 8, 1, 8, 40, 32, 0), ([3, 6], 6, 2, 2, 64, 32, 0), ([700, 650], 3, 2, 4, 64, 32, 100), ([64], 2, 1, 1, 64, 32, 1),
    ([1000, 900], 1, 2, 4, 128, 256, 33), ([2000], 1, 1, 1, 64, 32, 0), ([5000, 1, 64, 3000], 1, 2, 4, 64, 128, 0),
    # many rows of a sequence
    ([40], 40, 2, 4, 64, 32, 0), ([300], 300, 1, 2, 128, 64, 0), ([100, 130], 33, 2, 3, 96, 32, 0), ([65], 65, 1, 1, 32, 32, 0),
    ([260], 129, 2, 1, 80, 32, 0), ([200], 70, 1, 16, 256, 64, 0), ([150], 150, 1, 3, 160, 32, 0), ([90], 90, 1, 2, 192, 32, 0),
    ([90], 90, 1, 2, 224, 32, 0), ([600], 200, 1, 2, 64, 32, 50), ([1500], 64, 1, 8, 64, 64, 0), ([1100, 20], 100, 1, 1, 128, 32, 0),
    ([50, 0, 70], 60, 2, 4, 64, 32, 0), ([2000], 17, 1, 16, 128, 128, 0),
]


@pytest.mark.parametrize("lengths,n,heads,group,dim,page,window", UNIFORM)
def test_uniform(gpu, lengths, n, heads, group, dim, page, window):
    rng = np.random.default_rng(sum(lengths) + dim)
    cache, tables, keys, values = filled(gpu, rng, lengths, heads, dim, page)
    q = rows_of(rng, n * len(lengths), heads * group, dim, torch.bfloat16, 2.0).to(gpu)
    out, lse = attention()(q, cache, tables, *ref.device(gpu, np.array(lengths, np.int32)), window=window, return_lse=True)
    check(out, lse, q, keys, values, [n] * len(lengths), group, window=window)


RAGGED = [
    # lengths, rows
    ([300, 77, 600, 1, 0, 33], [1, 77, 130, 1, 0, 20], 2, 4, 64, 32, 0),
    ([300, 77, 600], [1, 1, 1], 2, 4, 128, 64, 0),
    ([80, 200, 64, 90], [80, 3, 0, 90], 3, 5, 96, 32, 0),
    ([500, 40], [400, 5], 1, 8, 128, 64, 64),
    ([10, 500], [30, 260], 1, 2, 64, 32, 0),  # more rows than tokens
    ([400], [300], 2, 1, 256, 128, 0),
    ([129, 140], [40, 7], 1, 48, 64, 32, 0),
    ([90, 120], [9, 100], 1, 24, 256, 32, 0),
    ([0, 0], [3, 100], 1, 2, 64, 32, 0),
    ([129, 40, 1], [1, 30, 1], 1, 40, 128, 32, 0),  # more heads than the kernel for few rows takes
    ([40] * 300, [1] * 299 + [20], 1, 2, 32, 32, 0),  # more sequences than a wave looks at in one go
    ([33] * 130, [2] * 60 + [0] * 9 + [33] + [1] * 60, 1, 8, 64, 32, 0),
]


@pytest.mark.parametrize("lengths,counts,heads,group,dim,page,window", RAGGED)
def test_ragged(gpu, lengths, counts, heads, group, dim, page, window):
    rng = np.random.default_rng(sum(lengths) + dim)
    cache, tables, keys, values = filled(gpu, rng, lengths, heads, dim, page)
    n = sum(counts)
    q = rows_of(rng, n + 5, heads * group, dim, torch.bfloat16, 2.0).to(gpu)
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=gpu)
    got, lse = attention()(q, cache, tables, *ref.device(gpu, np.array(lengths, np.int32)), window=window, return_lse=True,
                           offsets=ref.device(gpu, ref.offsets_of(counts))[0], out=out)
    assert got is out and (out[n:] == 7.0).all()  # rows of no sequence
    check(out, lse, q, keys, values, counts, group, window=window)


@pytest.mark.parametrize("lengths,n,heads,group,dim", [([300, 41], 1, 2, 4, 64), ([300, 41], 6, 1, 8, 128), ([200, 90], 90, 2, 2, 64)])
def test_all_of_the_sequence_is_seen_without_causal(gpu, lengths, n, heads, group, dim):
    rng = np.random.default_rng(dim + n)
    cache, tables, keys, values = filled(gpu, rng, lengths, heads, dim, 64)
    q = rows_of(rng, n * len(lengths), heads * group, dim, torch.bfloat16).to(gpu)
    out, lse = attention()(q, cache, tables, *ref.device(gpu, np.array(lengths, np.int32)), causal=False, scale=0.3, return_lse=True)
    check(out, lse, q, keys, values, [n] * len(lengths), group, scale=0.3, causal=False)


@pytest.mark.parametrize("n", [1, 60])
def test_missing_pages_are_left_out(gpu, n):
    rng = np.random.default_rng(n)
    lengths, heads, group, dim, page = [500, 200], 2, 4, 64, 32
    cache, tables, keys, values = filled(gpu, rng, lengths, heads, dim, page)
    tables[0, 3], tables[0, 7], tables[1, :] = -1, 2**31 - 1, -5
    gone = [np.zeros(x, dtype=bool) for x in lengths]
    gone[0][96:128] = gone[0][224:256] = gone[1][:] = True
    q = rows_of(rng, n * 2, heads * group, dim, torch.bfloat16).to(gpu)
    out, lse = attention()(q, cache, tables, *ref.device(gpu, np.array(lengths, np.int32)), return_lse=True)
    check(out, lse, q, keys, values, [n] * 2, group, left_out=gone)


@pytest.mark.parametrize("n", [1, 3, 50, 300])
def test_what_a_row_does_not_see_does_not_reach_it(gpu, n):
    """NaN in keys and values: of tokens behind a row, before its window, and in the pages behind a sequence."""
    from mambo_amd.kernels.kv_cache import launch_append_kv
    rng = np.random.default_rng(n)
    heads, group, dim, page, length = 1, 2, 64, 32, 330
    cache = new_cache(12, heads, dim, page)  # NaN codes and scales everywhere
    tables = torch.from_numpy(rng.permutation(12).astype(np.int32)[None]).to(gpu)
    k, v = rows_of(rng, length, heads, dim, torch.float32), rows_of(rng, length, heads, dim, torch.float32)
    bad = length - n + n // 2  # the middle row's own token
    k[bad, 0, 5], v[20, 0, 3] = float("nan"), float("inf")
    lengths = torch.tensor([length], dtype=torch.int32, device=gpu)
    launch_append_kv(k.to(gpu), v.to(gpu), cache, tables, lengths)
    q = rows_of(rng, n, heads * group, dim, torch.bfloat16).to(gpu)
    out, lse = attention()(q, cache, tables, lengths, window=25, return_lse=True)
    spoiled = np.array([bad <= p and bad > p - 25 or 20 <= p and 20 > p - 25 for p in range(length - n, length)])
    nan = torch.isnan(out).all(2).all(1).cpu().numpy()
    assert np.array_equal(nan, spoiled) and np.array_equal(torch.isnan(out).any(2).any(1).cpu().numpy(), spoiled)
    assert np.array_equal(torch.isnan(lse).all(1).cpu().numpy(), spoiled)
    got_k, got_v = read_all(cache, tables, [length])
    keys, values = np.nan_to_num(got_k[0]), got_v[0]
    want, _, bound, _ = ref.attend(q.double().cpu().numpy(), keys, values, group, dim ** -0.5, True, 25)
    off = np.abs(out.double().cpu().numpy() - want)
    assert (off[~spoiled] <= bound[~spoiled]).all()


@pytest.mark.parametrize("n", [1, 100])
def test_large_scores(gpu, n):
    """Scores of hundreds, where one token takes everything, and rows of equal ones."""
    rng = np.random.default_rng(9)
    cache, tables, keys, values = filled(gpu, rng, [400], 2, 64, 32)
    q = rows_of(rng, n, 4, 64, torch.bfloat16, 60.0).to(gpu)
    q[0, 0] = 0.0
    out, lse = attention()(q, cache, tables, *ref.device(gpu, np.array([400], np.int32)), return_lse=True)
    check(out, lse, q, keys, values, [n], 2)


def test_strides_alignment_and_repeats(gpu):
    rng = np.random.default_rng(10)
    lengths = [300, 45, 1]
    cache, tables, keys, values = filled(gpu, rng, lengths, 2, 64, 32)
    on = ref.device(gpu, np.array(lengths, np.int32))[0]
    for n in (1, 70):
        base = rows_of(rng, 3 * n, 10, 72, torch.bfloat16).to(gpu)
        for q in (base[:, :4, :64], base[:, 1:5, 3:67], base[:, ::2, 8:72][:, :4], base[:, :4, :64].flip(2)):
            whole = torch.full((3 * n, 6, 67), 7.0, dtype=torch.bfloat16, device=gpu)
            out = whole[:, 1:5, 3:67]
            first = attention()(q.contiguous(), cache, tables, on)
            assert attention()(q, cache, tables, on, out=out) is out
            assert torch.equal(out, first)
            for _ in range(3):
                assert torch.equal(attention()(q, cache, tables, on), first)
            whole[:, 1:5, 3:67] = 7.0
            assert (whole == 7.0).all()
    assert attention()(q[:0], cache, tables, on).shape == (0, 4, 64)


def test_arrays_of_any_values_stay_within_the_tensors(gpu):
    rng = np.random.default_rng(11)
    cache, tables, _, _ = filled(gpu, rng, [300, 45, 100], 2, 64, 32)
    q = rows_of(rng, 90, 4, 64, torch.bfloat16).to(gpu)
    for bad in ([-5, 70, 3], [2**31 - 1] * 3, [-2**31] * 3):
        for cuts in (None, [0, 5, 3, 90], [-9, 4, 99, 2**31 - 1], [90, 10, 5, 0], [7, 7, 7, 7]):
            attention()(q, cache, tables, torch.tensor(bad, dtype=torch.int32, device=gpu),
                        offsets=None if cuts is None else torch.tensor(cuts, dtype=torch.int32, device=gpu))
    torch.cuda.synchronize()


def test_a_long_cache_is_split(gpu):
    """Tens of thousands of tokens, in parts of many workgroups, against a product in float64 on the GPU."""
    rng = np.random.default_rng(12)
    for n, heads, group, dim, length in ((1, 2, 4, 64, 40011), (3, 1, 5, 128, 20000), (130, 1, 2, 64, 9000)):
        cache, tables, keys, values = filled(gpu, rng, [length], heads, dim, 128)
        q = rows_of(rng, n, heads * group, dim, torch.bfloat16, 2.0).to(gpu)
        out, lse = attention()(q, cache, tables, *ref.device(gpu, np.array([length], np.int32)), return_lse=True)
        check(out, lse, q, keys, values, [n], group)


def test_offsets_past_32_bits(gpu):
    """A pool of more than 4 GiB of codes, the sequence's pages at its end."""
    from mambo_amd.kernels.kv_cache import launch_append_kv
    from mambo_amd.utils.kv_cache import allocate_kv_cache
    rng = np.random.default_rng(13)
    heads, dim, page = 8, 128, 256
    pages = (5 << 30) // (2 * heads * dim * page)
    cache = allocate_kv_cache(pages, heads, dim, page_size=page)
    tables = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device=gpu)
    lengths = torch.tensor([300], dtype=torch.int32, device=gpu)
    k, v = rows_of(rng, 300, heads, dim, torch.bfloat16), rows_of(rng, 300, heads, dim, torch.bfloat16)
    launch_append_kv(k.to(gpu), v.to(gpu), cache, tables, lengths)
    model = ref.Model(heads, dim)
    model.append(k.double().numpy(), v.double().numpy(), 0)
    for n in (1, 40):
        q = rows_of(rng, n, heads * 2, dim, torch.bfloat16).to(gpu)
        out, lse = attention()(q, cache, tables, lengths, return_lse=True)
        check(out, lse, q, [model.k], [model.v], [n], 2)
    assert not cache.codes[0].any() and math.isfinite(float(out.float().sum()))


def test_rows_before_the_first_sequence(gpu):
    rng = np.random.default_rng(14)
    for lengths, counts, skip in (([200, 90], [1, 2], 40), ([300, 100], [150, 60], 7), ([40, 2500], [1, 90], 300)):
        cache, tables, keys, values = filled(gpu, rng, lengths, 2, 64, 32)
        n = sum(counts)
        q = rows_of(rng, n + skip, 8, 64, torch.bfloat16).to(gpu)
        out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=gpu)
        out, lse = attention()(q, cache, tables, *ref.device(gpu, np.array(lengths, np.int32)), return_lse=True, out=out,
                               offsets=ref.device(gpu, ref.offsets_of(counts) + skip)[0])
        assert (out[:skip] == 7.0).all()
        check(out[skip:], lse[skip:], q[skip:], keys, values, counts, 4)


def test_refusals(gpu):
    from mambo_amd.utils.kv_cache import allocate_kv_cache
    cache = allocate_kv_cache(2, 2, 64, page_size=32)
    tables, lengths = torch.zeros((2, 1), dtype=torch.int32, device=gpu), torch.ones(2, dtype=torch.int32, device=gpu)
    q = torch.zeros((4, 4, 64), dtype=torch.bfloat16, device=gpu)
    good = dict(q=q, cache=cache, tables=tables, lengths=lengths)
    attention()(**good)
    for change in ({"q": q.float()}, {"q": q[..., :32]}, {"q": q[:, :3]}, {"q": q[:3]}, {"q": q.cpu()}, {"scale": 0.0}, {"scale": float("nan")},
                   {"scale": -1.0}, {"scale": 3.0e38}, {"window": -1}, {"window": 4, "causal": False}, {"tables": tables.long()},
                   {"lengths": lengths[:1]}, {"offsets": lengths}, {"offsets": torch.zeros(3, device=gpu)}, {"out": q.float()},
                   {"out": q[:2]}, {"out": q[:1].expand(4, 4, 64)}):
        with pytest.raises(ValueError):
            attention()(**(good | change))
    with pytest.raises(TypeError):
        attention()(**(good | {"cache": cache.codes}))


def plan_of(cache, tables, tokens, q_heads, ragged, window=0):
    import ctypes
    from mambo_amd import _native
    out = (ctypes.c_int32 * 4)()
    batch = _native.KVBatchArgs(256, tables.shape[1], tables.shape[1], 256, 256 if ragged else None, tables.shape[0])
    _native.check(_native.lib().mambo_kv_attention_plan(cache.args, batch, tokens, q_heads, window, out))
    return list(out)


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("dim", [24, 64, 88, 128, 160, 184, 224, 256])
def test_every_kernel_for_few_rows(gpu, dim, split):
    """16, 32 and 64 rows a sequence where the head's size allows it, by one workgroup and by shares that are joined
    (tables wide enough for long sequences)."""
    rng = np.random.default_rng(dim)
    lengths = [300, 33, 0, 170]
    cache, tables, keys, values = filled(gpu, rng, lengths, 1, dim, 32, extra=100 if split else 1)
    for group, seqs in [(11, 4), (27, 4)] + [(61, 3), (61, 4)] * (dim <= 64):
        q = rows_of(rng, seqs, group, dim, torch.bfloat16, 2.0).to(gpu)
        plan = plan_of(cache, tables[:seqs], seqs, group, False)
        if split and (group, seqs) == (61, 4):  # from four sequences on
            assert plan[:3] == [0, 0, 256]
        else:
            assert plan[0] == (16 if group == 11 else 32 if group == 27 else 64) and plan[2] == 0
            assert (plan[1] > 0) == (split or (group == 27 and dim > 128))
        out, lse = attention()(q, cache, tables[:seqs], *ref.device(gpu, np.array(lengths[:seqs], np.int32)), return_lse=True)
        check(out, lse, q, keys[:seqs], values[:seqs], [1] * seqs, group)


@pytest.mark.parametrize("dim", [24, 64, 88, 128, 160, 184, 224, 256])
def test_every_kernel_for_many_rows(gpu, dim):
    """With the keys in one part and in several, of one sequence and of ragged ones, of odd numbers of blocks."""
    rng = np.random.default_rng(dim + 1)
    for lengths, counts, parts in (([1100], [70], 3), ([290], [90], 1), ([1090, 40, 300], [66, 40, 9], 3)):
        cache, tables, keys, values = filled(gpu, rng, lengths, 1, dim, 32)
        n, ragged = sum(counts), len(counts) > 1
        q = rows_of(rng, n, 2, dim, torch.bfloat16, 2.0).to(gpu)
        plan = plan_of(cache, tables, n, 2, ragged)
        assert plan[2] == (256 if dim <= 192 else 128) and plan[3] == parts
        out, lse = attention()(q, cache, tables, *ref.device(gpu, np.array(lengths, np.int32)), return_lse=True,
                               offsets=ref.device(gpu, ref.offsets_of(counts))[0] if ragged else None)
        check(out, lse, q, keys, values, counts, 2)


@pytest.mark.parametrize("ragged", [False, True])
def test_many_sequences_share_the_work(gpu, ragged):
    """More sequences than a wave adds up at once, long, short and empty, some of them without rows."""
    rng = np.random.default_rng(15)
    lengths = [int(n) for n in rng.integers(0, 70, 700)]
    lengths[5], lengths[300], lengths[699] = 3000, 1500, 900
    lengths[310:600] = [0] * 290
    counts = [int(c) for c in rng.integers(0, 3, 700)] if ragged else [1] * 700
    counts[300] = 1
    cache, tables, keys, values = filled(gpu, rng, lengths, 1, 32, 64)
    n = sum(counts)
    q = rows_of(rng, n, 4, 32, torch.bfloat16, 2.0).to(gpu)
    assert plan_of(cache, tables, n, 4, ragged)[1] > 0
    out, lse = attention()(q, cache, tables, *ref.device(gpu, np.array(lengths, np.int32)), return_lse=True,
                           offsets=ref.device(gpu, ref.offsets_of(counts))[0] if ragged else None)
    check(out, lse, q, keys, values, counts, 4)


def test_probabilities_add_up_over_a_rising_sequence_of_scores(gpu):
    """Every later key scores higher than all before it: the running largest grows at every step, by less and by more
    than the lag that the kernel for many rows allows itself."""
    from mambo_amd.kernels.kv_cache import launch_append_kv
    rng = np.random.default_rng(16)
    dim, page, length = 64, 64, 700
    for rise in (0.02, 0.4):
        for order in (1, -1):
            cache = new_cache(11, 1, dim, page)
            tables = torch.arange(11, dtype=torch.int32, device=gpu)[None]
            k = torch.ones((length, 1, dim)) * (rise * torch.arange(length)[:, None, None] / 8.0)
            k = k.flip(0) if order < 0 else k
            v = rows_of(rng, length, 1, dim, torch.bfloat16)
            lengths = torch.tensor([length], dtype=torch.int32, device=gpu)
            launch_append_kv(k.bfloat16().to(gpu), v.to(gpu), cache, tables, lengths)
            keys, values = read_all(cache, tables, [length])
            for n in (1, 80):
                q = torch.ones((n, 2, dim), dtype=torch.bfloat16, device=gpu)
                out, lse = attention()(q, cache, tables, lengths, return_lse=True)
                check(out, lse, q, keys, values, [n], 2)


@pytest.mark.parametrize("n,group,columns", [(1, 4, 3), (10, 4, 3), (90, 4, 3), (1, 4, 60), (10, 4, 60), (100, 2, 60)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 8), (True, 70), (False, 0)])
def test_rows_past_a_table_keep_their_positions(gpu, n, group, columns, causal, window):
    """Sequences that are longer than their tables: a row sees the cached tokens up to its own position and within its
    window, which may be none. By every kernel."""
    rng = np.random.default_rng(n + columns)
    held, heads, dim = 32 * columns, 1, 64
    cache, tables, keys, values = filled(gpu, rng, [held, held], heads, dim, 32, extra=0)
    assert tables.shape == (2, columns)
    q = rows_of(rng, 2 * n, heads * group, dim, torch.bfloat16, 2.0).to(gpu)
    for past in ([1, 6], [n, 0], [n + 3, 75], [2**31 - 1 - held, 33]):
        out, lse = attention()(q, cache, tables, *ref.device(gpu, np.array([held + p for p in past], np.int32)), causal=causal,
                               window=window, return_lse=True)
        for s, p in enumerate(past):
            # far behind the table every row sees all of it, or nothing
            p = min(p, held + 2 * n + window)
            gone = np.arange(held + p) >= held
            there = [np.concatenate([t[s], np.zeros((p, heads, dim))]) for t in (keys, values)]
            part = slice(n * s, n * (s + 1))
            check(out[part], lse[part], q[part], [there[0]], [there[1]], [n], group, causal=causal, window=window, left_out=[gone])


@pytest.mark.parametrize("n,group,seqs,few", [(1, 16, 2**20, 16), (64, 32, 2**13, 0), (1, 64, 2**18 + 5, 64)])
def test_two_to_the_24_rows_and_more(gpu, n, group, seqs, few):
    """The same sequences over and over: every repeat has the rows of the first, which are checked."""
    rng = np.random.default_rng(30)
    lengths, dim = [64, 40, 3, 0, 33, 1, 64, 50], 8
    cache, tables, keys, values = filled(gpu, rng, lengths, 1, dim, 32)
    times = -(-seqs // 8)
    on = ref.device(gpu, np.array(lengths, np.int32))[0].repeat(times)[:seqs]
    tables = tables.repeat(times, 1)[:seqs]
    first = rows_of(rng, 8 * n, group, dim, torch.bfloat16, 2.0).to(gpu)
    q = first.repeat(times, 1, 1)[:seqs * n]
    assert q.shape[0] * group >= 2**24 and plan_of(cache, tables, seqs * n, group, False)[:2] == [few, 0]
    out, lse = attention()(q, cache, tables, on, return_lse=True)
    check(out[:8 * n], lse[:8 * n], first, keys, values, [n] * 8, group)
    assert torch.equal(out, out[:8 * n].repeat(times, 1, 1)[:seqs * n]) and torch.equal(lse, lse[:8 * n].repeat(times, 1)[:seqs * n])


# lengths, rows of each sequence, key/value heads, group, head size, page, tables in pages more than needed, causal, window,
# the kernel for few rows (by shares, by one workgroup a sequence, or not launched), whether that for many has several parts
BLOCKS = [
    ([131149], [1], 1, 8, 128, 128, 1, True, 0, "shares", False),
    ([40011], [1], 2, 6, 64, 128, 1, True, 0, "shares", False),
    ([20000], [3], 1, 5, 128, 128, 1, True, 0, "shares", False),
    ([20000, 5000, 9000], [1] * 3, 1, 4, 128, 32, 1, True, 4096, "shares", False),  # windows of many blocks
    ([20000], [5], 2, 6, 64, 64, 1, True, 4100, "shares", False),
    ([9000, 40, 0, 20000], [2, 16, 1, 5], 1, 2, 96, 32, 1, True, 4096, "shares", True),
    ([9000, 6000], [1, 1], 3, 31, 256, 64, 1, True, 3000, "shares", False),
    ([20000, 7000], [3, 3], 1, 4, 96, 32, 1, False, 0, "shares", False),  # all of the sequence, split
    ([40011], [1], 1, 60, 40, 128, 1, False, 0, "shares", False),
    ([5000, 9000], [2, 1], 2, 3, 128, 64, 1, False, 0, "shares", False),
    ([5000] * 4, [4] * 4, 1, 12, 64, 32, 1, True, 2000, None, True),
    ([9000], [130], 1, 2, 64, 128, 1, True, 0, None, True),
    ([9000], [130], 1, 2, 64, 128, 1, True, 4096, None, True),
    ([9000, 300, 7000], [100, 2, 90], 1, 3, 128, 32, 1, True, 3333, "shares", True),
    ([9000], [130], 1, 2, 96, 128, 1, False, 0, None, True),
    ([6000, 5000], [70, 70], 1, 4, 192, 64, 1, True, 2000, None, True),
    ([6000, 70, 5000], [40, 70, 90], 1, 3, 256, 64, 1, True, 1500, "shares", True),
    ([6000, 5000], [150, 30], 1, 2, 256, 64, 1, False, 0, "shares", True),
    ([30001], [600], 2, 2, 64, 128, 1, True, 8000, None, True),
    ([1200], [3], 1, 5, 64, 32, 1, True, 0, "one", False),  # by one workgroup
    ([9000], [3], 1, 5, 64, 32, 1, True, 1000, "one", False),
    ([1200, 30], [4, 4], 2, 4, 128, 32, 1, False, 0, "one", False),
]


@pytest.mark.parametrize("lengths,counts,heads,group,dim,page,extra,causal,window,few,several", BLOCKS)
def test_every_block_of_a_long_cache_counts_once(gpu, lengths, counts, heads, group, dim, page, extra, causal, window, few, several):
    """Long caches, windows of thousands and rows that see all of their sequence, by shares and by parts that are joined: the
    comparison (kv_reference.block_rows) shows a block that is lost or counted twice, or whose values come with other keys."""
    from mambo_amd.kernels.kv_cache import launch_append_kv
    rng = np.random.default_rng(sum(lengths) + dim)
    host, pages = ref.tables_of(rng, lengths, page, extra=extra)
    tables, cache = ref.device(gpu, host)[0], new_cache(pages, heads, dim, page)
    rows = [ref.block_rows(rng, n, heads, dim) for n in lengths]
    k, v = (torch.from_numpy(np.concatenate([r[i] for r in rows])).bfloat16().to(gpu) for i in (0, 1))
    on = ref.device(gpu, np.array(lengths, np.int32))[0]
    launch_append_kv(k, v, cache, tables, on, offsets=ref.device(gpu, ref.offsets_of(lengths))[0])
    ragged, n = len(set(counts)) > 1, sum(counts)
    plan = plan_of(cache, tables, n, heads * group, ragged, window)
    assert (few is None) == (plan[0] == 0) and (few == "shares") == (plan[1] > 0) and several == (plan[2] > 0 and plan[3] > 1), plan
    q = torch.from_numpy(np.concatenate([ref.block_queries(c, heads * group, dim) for c in counts])).bfloat16().to(gpu)
    out, lse = attention()(q, cache, tables, on, causal=causal, window=window, scale=math.log(2.0), return_lse=True,
                           offsets=ref.device(gpu, ref.offsets_of(counts))[0] if ragged else None)
    cuts = ref.offsets_of(counts)
    for s, c in enumerate(counts):
        part = slice(cuts[s], cuts[s + 1])
        want, want_lse, bound, lse_bound = ref.block_attend(*rows[s], c, group, causal, window)
        got, got_lse = out[part].double().cpu().numpy(), lse[part].double().cpu().numpy()
        some = np.isfinite(want_lse)
        assert (np.abs(got - want) <= bound).all(), s
        assert np.array_equal(some, np.isfinite(got_lse)) and (np.abs(got_lse[some] - want_lse[some]) <= lse_bound[some]).all(), s


class Guarded:
    """A tensor in the middle of a larger one, whose ends must stay as they are."""

    def __init__(self, gpu, shape, dtype, fill):
        n = math.prod(shape)
        self.margin = 1 << 16  # 128 KiB and more
        self.whole = torch.full((n + 2 * self.margin,), fill, dtype=dtype, device=gpu)
        self.ends = self.whole[:self.margin].clone()
        self.inner = self.whole[self.margin:self.margin + n].view(shape)

    def untouched(self):
        bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[self.whole.element_size()]
        return all(torch.equal(part.view(bits), self.ends.view(bits)) for part in (self.whole[:self.margin], self.whole[-self.margin:]))


HOSTILE_LENGTHS = ([-5, 70, 3], [2**31 - 1] * 3, [-2**31] * 3, [5000, 0, 2**31 - 40], [2**30, 3200, 31])
HOSTILE_OFFSETS = (None, [0, 5, 3, 90], [-9, 4, 99, 2**31 - 1], [90, 10, 5, 0], [7, 7, 7, 7], [-2**31, 0, 2**31 - 1, 40], [0, 1, 2, 3])


@pytest.mark.parametrize("columns,tokens,plan", [(4, 90, [16, 0, 256, 1]), (4, 3, [16, 0, 0, 1]), (100, 90, [16, 75, 256, 7]), (100, 3, [16, 75, 0, 1])])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 1), (True, 40), (False, 0)])
def test_arrays_of_any_values_write_nothing_elsewhere(gpu, columns, tokens, plan, causal, window):
    """Lengths, offsets and pages of any values: what lies around the output, the lse and the workspace stays, and so do the cache and
    the tables; rows that no sequence can have stay as well."""
    from mambo_amd import _native
    rng = np.random.default_rng(31)
    lengths, heads, group, dim = [32 * columns, 45, 100], 2, 2, 64
    cache, tables, _, _ = filled(gpu, rng, lengths, heads, dim, 32, extra=0)
    tables = tables.clone()
    tables[1, 1:], tables[2] = 2**31 - 1, torch.from_numpy(rng.integers(-2**31, 2**31, columns).astype(np.int32)).to(gpu)
    before = [t.clone() for t in (cache.codes, cache.scales, tables)]
    q = rows_of(rng, tokens, heads * group, dim, torch.bfloat16).to(gpu)
    assert plan_of(cache, tables, tokens, heads * group, True, window) == [16, 0 if window else plan[1], *plan[2:]]
    for bad in HOSTILE_LENGTHS:
        on = torch.tensor(bad, dtype=torch.int64, device=gpu).int()
        for cuts in HOSTILE_OFFSETS:
            offsets = None if cuts is None else torch.tensor(cuts, dtype=torch.int64, device=gpu).int()
            batch = _native.KVBatchArgs(tables.data_ptr(), columns, columns, on.data_ptr(), None if cuts is None else offsets.data_ptr(), 3)
            size = _native.lib().mambo_kv_attention_workspace(cache.args, batch, tokens, heads * group, window)
            out = Guarded(gpu, q.shape, torch.bfloat16, 7.0)
            lse = Guarded(gpu, q.shape[:2], torch.float32, 7.0)
            work = Guarded(gpu, (size,), torch.uint8, 77)
            assert work.inner.data_ptr() % 16 == 0
            _native.check(_native.lib().mambo_kv_attention(
                q.data_ptr(), tokens, heads * group, dim, heads * group * dim, dim, cache.args, batch, 0.125, causal, window,
                out.inner.data_ptr(), heads * group * dim, dim, lse.inner.data_ptr(), work.inner.data_ptr(), size,
                _native.stream_handle(None)), "attention")
            torch.cuda.synchronize()
            assert out.untouched() and lse.untouched() and work.untouched(), (bad, cuts)
            if cuts == [7, 7, 7, 7]:
                assert (out.inner == 7.0).all() and (lse.inner == 7.0).all()
            if cuts == [0, 1, 2, 3]:
                assert (out.inner[3:] == 7.0).all() and (lse.inner[3:] == 7.0).all()
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.codes, cache.scales, tables)))
