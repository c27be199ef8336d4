"""The paged 8-bit cache on the GPU: appends against a model of the blocks, bit for bit without a rotation, and
within a rounding step with one; growth of a block's exponent, pages, strides, values that are not finite."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu


def ops():
    from mambo_amd.kernels import kv_cache
    return kv_cache


def new_cache(pages, heads, dim, page):
    from mambo_amd.utils.kv_cache import allocate_kv_cache
    cache = allocate_kv_cache(pages, heads, dim, page_size=page)
    cache.codes.fill_(0x7F)  # what pages hold before is anything
    cache.scales.fill_(0xFF)
    return cache


def rows_of(rng, n, heads, dim, dtype, scale=1.0):
    x = torch.from_numpy((scale * rng.standard_normal((n, heads, dim))).astype(np.float32)).to(dtype)
    return x


def read_all(cache, tables, lengths):
    seqs = np.concatenate([np.full(n, s) for s, n in enumerate(lengths)]).astype(np.int32)
    at = np.concatenate([np.arange(n) for n in lengths]).astype(np.int32)
    k, v = ops().launch_read_kv(cache, tables, *ref.device(tables.device, seqs, at))
    cuts = ref.offsets_of(lengths)
    split = lambda t: [t[a:b].double().cpu().numpy() for a, b in zip(cuts[:-1], cuts[1:])]  # noqa: E731
    return split(k), split(v)


def same(a, b):
    assert a.shape == b.shape and np.array_equal(np.isnan(a), np.isnan(b))
    assert np.array_equal(np.nan_to_num(a), np.nan_to_num(b))


# head size, heads, page, type, rounds of new tokens of each sequence
STEPS = [
    (64, 2, 64, torch.bfloat16, [[5, 1, 40], [1, 1, 1], [30, 0, 31], [1, 2, 64]]),
    (128, 1, 32, torch.float32, [[33], [1], [31], [64], [1]]),
    (80, 3, 128, torch.float32, [[0, 3], [200, 1], [1, 0], [7, 129]]),
    (8, 1, 32, torch.bfloat16, [[1, 1], [40, 1]]),
    (256, 2, 256, torch.bfloat16, [[31, 65], [1, 1], [2, 300]]),
    (136, 2, 32, torch.float32, [[10, 1, 1, 1], [1, 1, 1, 32]]),
]


@pytest.mark.parametrize("spread", [1.0, 8.0])
@pytest.mark.parametrize("dim,heads,page,dtype,rounds", STEPS)
def test_appends_follow_the_model(gpu, dim, heads, page, dtype, rounds, spread):
    rng = np.random.default_rng(dim)
    seqs = len(rounds[0])
    totals = np.sum(rounds, axis=0)
    host, pages = ref.tables_of(rng, totals, page)
    tables = ref.device(gpu, host)[0]
    cache = new_cache(pages, heads, dim, page)
    models, lengths = [ref.Model(heads, dim) for _ in range(seqs)], np.zeros(seqs, dtype=np.int32)
    for step, counts in enumerate(rounds):
        n = sum(counts)
        scale = spread ** step
        k, v = rows_of(rng, n, heads, dim, dtype, scale), rows_of(rng, n, heads, dim, dtype, 1.0 / scale)
        starts = lengths.copy()
        lengths += np.array(counts, dtype=np.int32)
        offsets = ref.offsets_of(counts)
        uniform = len(set(counts)) == 1
        got = ops().launch_append_kv(k.to(gpu), v.to(gpu), cache, tables, ref.device(gpu, lengths)[0],
                                     offsets=None if uniform and step % 2 else ref.device(gpu, offsets)[0])
        assert got is None
        for s in range(seqs):
            part = slice(offsets[s], offsets[s + 1])
            models[s].append(k[part].double().numpy(), v[part].double().numpy(), int(starts[s]))
        got_k, got_v = read_all(cache, tables, lengths)
        for s in range(seqs):
            same(got_k[s], models[s].k)
            same(got_v[s], models[s].v)


@pytest.mark.parametrize("vectors", [True, False])
@pytest.mark.parametrize("dim,size,interleaved", [(64, 64, False), (64, 32, True), (128, 128, False), (80, 40, False),
                                                  (80, 20, False), (72, 18, True), (256, 256, True), (96, 96, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotated_keys_and_queries(gpu, dim, size, interleaved, dtype, vectors):
    """Stored keys are within half a step of the rotated ones, values exactly rounded, queries as
    launch_rotary rotates them."""
    from mambo_amd.kernels.rotary import launch_rotary
    from mambo_amd.utils.rotary_table import prepare_rotary_table, rotary_frequencies
    scaling = {"type": "yarn", "factor": 16.0, "original_length": 4096}
    frequencies, magnitude = rotary_frequencies(size, scaling=scaling)
    table = prepare_rotary_table(size, scaling=scaling, interleaved=interleaved)
    rng = np.random.default_rng(size)
    heads, group, page, counts, starts = 2, 3, 32, [40, 1, 7], [3, 95, 0]
    lengths = np.array(starts, dtype=np.int32) + np.array(counts, dtype=np.int32)
    host, pages = ref.tables_of(rng, lengths, page)
    tables, cache = ref.device(gpu, host)[0], new_cache(pages, heads, dim, page)
    n, offsets = sum(counts), ref.offsets_of(counts)
    pad = 0 if vectors else 1  # rows that are aligned to their type alone

    def rows(h):
        return rows_of(rng, n, h, dim + pad, dtype).to(gpu)[..., pad:]

    k, v, q = rows(heads), rows(heads), rows(heads * group)
    for given in (None, np.array(rng.integers(0, 50000, n), dtype=np.int32)):
        # the blocks of what was cached are entered anew
        past = ref.offsets_of(starts)
        z = torch.zeros((sum(starts), heads, dim), dtype=dtype, device=gpu)
        ops().launch_append_kv(z, z, cache, tables, ref.device(gpu, np.array(starts, dtype=np.int32))[0],
                               offsets=ref.device(gpu, past)[0])
        got = ops().launch_append_kv(k, v, cache, tables, ref.device(gpu, lengths)[0], offsets=ref.device(gpu, offsets)[0],
                                     rotary=table, q=q, positions=None if given is None else ref.device(gpu, given)[0])
        positions = np.concatenate([np.arange(s, s + c) for s, c in zip(starts, counts)]).astype(np.int32) if given is None else given
        assert got.dtype == torch.bfloat16
        assert torch.equal(got, launch_rotary(q, ref.device(gpu, positions)[0], table, out_dtype=torch.bfloat16))
        got_k, got_v = read_all(cache, tables, lengths)
        k64 = k.double().cpu().numpy()
        turned, off = ref.rotate(k64, positions, frequencies, interleaved, magnitude), ref.rotation_bound(k64, size, interleaved, magnitude)
        for s in range(3):
            part, new = slice(offsets[s], offsets[s + 1]), slice(starts[s], lengths[s])
            model = ref.Model(heads, dim)
            zeros = np.zeros((starts[s], heads, dim))
            model.append(zeros, zeros, 0)
            model.append(turned[part], v[part].double().cpu().numpy(), starts[s])
            same(got_v[s], model.v)
            steps = np.zeros((counts[s], heads, 1))
            for i in range(counts[s]):
                for h in range(heads):
                    steps[i, h] = 2.0 ** (model.e[(starts[s] + i) // 32, h, "k"] + 1 - 10)
            bound = np.abs(turned[part]) * 2.0**-4 + steps + off[part]
            assert (np.abs(got_k[s][new] - turned[part]) <= bound).all()
            assert not got_k[s][:starts[s]].any()


def test_growth_by_single_tokens_is_exact_where_codes_stay_normal(gpu):
    """A token a call with keys of growing powers of two: every older code is moved by powers of two."""
    rng = np.random.default_rng(4)
    heads, dim, page = 1, 64, 32
    cache = new_cache(3, heads, dim, page)
    tables = torch.tensor([[2, 0]], dtype=torch.int32, device=gpu)
    model = ref.Model(heads, dim)
    for t in range(40):
        k = rows_of(rng, 1, heads, dim, torch.float32, 1.5 ** t)
        v = rows_of(rng, 1, heads, dim, torch.float32, 2.0 ** -t)
        ops().launch_append_kv(k.to(gpu), v.to(gpu), cache, tables, torch.tensor([t + 1], dtype=torch.int32, device=gpu))
        model.append(k.double().numpy(), v.double().numpy(), t)
    got_k, got_v = read_all(cache, tables, [40])
    same(got_k[0], model.k)
    same(got_v[0], model.v)


def test_a_prefix_is_kept_and_a_tail_overwritten(gpu):
    """Going back to an earlier length and appending from there: the block keeps its exponent."""
    rng = np.random.default_rng(5)
    cache = new_cache(4, 2, 64, 64)
    tables = torch.tensor([[3, 1]], dtype=torch.int32, device=gpu)
    model = ref.Model(2, 64)
    for start, n, scale in ((0, 50, 1.0), (50, 14, 30.0), (40, 9, 0.1), (32, 3, 1.0), (35, 60, 2.0)):
        k, v = rows_of(rng, n, 2, 64, torch.bfloat16, scale), rows_of(rng, n, 2, 64, torch.bfloat16, scale)
        ops().launch_append_kv(k.to(gpu), v.to(gpu), cache, tables, torch.tensor([start + n], dtype=torch.int32, device=gpu),
                               offsets=torch.tensor([0, n], dtype=torch.int32, device=gpu))
        model.append(k.double().numpy(), v.double().numpy(), start)
        got_k, got_v = read_all(cache, tables, [start + n])
        same(got_k[0], model.k)
        same(got_v[0], model.v)


def test_extreme_values(gpu):
    inf, nan = float("inf"), float("nan")
    heads, dim = 2, 40
    k, v = torch.ones((6, heads, dim)), torch.ones((6, heads, dim))
    k[0, 0, 3], v[1, 1, 39], k[2, 0, 0], v[3, 0, 7] = nan, inf, -inf, nan
    k[2, 0, 1] = 1e30  # of a token that counts for nothing
    k[4, 1], v[4, 1] = 3.4e38, -3.4e38  # would round to 2^128
    k[4, 1, 0], v[4, 1, 0] = 3.0e38, 3.18e38
    k[5, 0], v[5, 0] = 1e-38, 0.0
    cache = new_cache(2, heads, dim, 32)
    tables = torch.tensor([[1]], dtype=torch.int32, device=gpu)
    model = ref.Model(heads, dim)
    model.append(k.double().numpy(), v.double().numpy(), 0)
    ops().launch_append_kv(k.to(gpu), v.to(gpu), cache, tables, torch.tensor([6], dtype=torch.int32, device=gpu),
                           offsets=torch.tensor([0, 6], dtype=torch.int32, device=gpu))
    got_k, got_v = read_all(cache, tables, [6])
    same(got_k[0], model.k)
    same(got_v[0], model.v)
    # NaN keys stay NaN when the block's exponent grows
    more = torch.full((1, heads, dim), 1e20)
    model.append(more.double().numpy(), more.double().numpy(), 6)
    ops().launch_append_kv(more.to(gpu), more.to(gpu), cache, tables, torch.tensor([7], dtype=torch.int32, device=gpu))
    got_k, got_v = read_all(cache, tables, [7])
    same(got_k[0], model.k)
    same(got_v[0], model.v)
    zeros = torch.zeros((32, heads, dim), device=gpu)
    ops().launch_append_kv(zeros, zeros, cache, tables, torch.tensor([32], dtype=torch.int32, device=gpu))
    assert not any(t.any() for t in ops().launch_read_kv(cache, tables, *ref.device(gpu, np.zeros(32, np.int32), np.arange(32, dtype=np.int32))))
    assert (cache.scales[1] == 127 + ref.LOWEST).all()


def test_nothing_but_the_rows_of_the_call_is_written(gpu):
    """Pages of others, blocks that no new token is in, queries of no sequence, tokens that no page is for."""
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    rng = np.random.default_rng(6)
    heads, dim, page = 2, 64, 64
    cache = new_cache(6, heads, dim, page)
    before = cache.codes.clone(), cache.scales.clone()
    tables = torch.tensor([[4, 99], [2, 0], [-1, 5]], dtype=torch.int32, device=gpu)
    # sequence 0: 10 tokens from 60, of which the last 6 have no page; 1: none; 2: 3 tokens without a page; rows 13.. of nobody
    lengths = torch.tensor([70, 40, 3], dtype=torch.int32, device=gpu)
    offsets = torch.tensor([0, 10, 10, 13], dtype=torch.int32, device=gpu)
    k, v, q = (rows_of(rng, 20, h, dim, torch.bfloat16).to(gpu) for h in (heads, heads, 4))
    out = torch.full((20, 4, dim), 7.0, dtype=torch.bfloat16, device=gpu)
    ops().launch_append_kv(k, v, cache, tables, lengths, offsets=offsets, rotary=prepare_rotary_table(64), q=q, out=out)
    changed = (cache.codes != before[0]).flatten(2).any(2) | (cache.scales != before[1]).flatten(2).any(2)
    assert changed[4].all() and not changed[[0, 1, 2, 3, 5]].any()
    assert not (cache.codes[4, :, 0] != before[0][4, :, 0]).any()
    assert (out[13:] == 7.0).all() and not (out[:13] == 7.0).all(2).any()
    # more rows than the length: those before the start are not stored
    before = cache.codes.clone()
    ops().launch_append_kv(k[:5], v[:5], cache, tables[1:2], torch.tensor([2], dtype=torch.int32, device=gpu),
                           offsets=torch.tensor([0, 5], dtype=torch.int32, device=gpu))
    model = ref.Model(heads, dim)
    model.append(k[3:5].double().cpu().numpy(), v[3:5].double().cpu().numpy(), 0)
    got_k, got_v = read_all(cache, tables[1:2], [2])
    same(got_k[0], model.k)
    same(got_v[0], model.v)
    # arrays of any values stay within the tensors
    for bad in ([-5, 70, 3], [2**31 - 1] * 3, [-2**31] * 3):
        for cuts in ([0, 5, 3, 20], [-9, 4, 99, 2**31 - 1], [20, 10, 5, 0], [7, 7, 7, 7]):
            ops().launch_append_kv(k, v, cache, torch.tensor([[4, 99], [2, -7], [2**31 - 1, -2**31]], dtype=torch.int32, device=gpu),
                                   torch.tensor(bad, dtype=torch.int32, device=gpu), q=q, rotary=prepare_rotary_table(64),
                                   offsets=torch.tensor(cuts, dtype=torch.int32, device=gpu))
    got = ops().launch_read_kv(cache, tables, *ref.device(gpu, np.array([-1, 3, 0, 0, 0, 2, 2**31 - 1], np.int32),
                                                          np.array([0, 0, -1, 128, 64, 0, 5], np.int32)))
    assert not got[0].any() and not got[1].any()
    torch.cuda.synchronize()


def test_strided_rows(gpu):
    """Parts of one fused projection, in both types; tables with a stride."""
    rng = np.random.default_rng(7)
    heads, group, dim, n = 2, 2, 64, 37
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    table = prepare_rotary_table(64)
    lengths = torch.tensor([n], dtype=torch.int32, device=gpu)
    for dtype in (torch.float32, torch.bfloat16):
        fused = rows_of(rng, n, heads * (group + 2), dim, dtype).to(gpu)
        q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:]
        wide = torch.tensor([[1, 0, 9, 9]], dtype=torch.int32, device=gpu)
        caches = [new_cache(2, heads, dim, 32) for _ in range(3)]
        a = ops().launch_append_kv(q=q, k=k, v=v, cache=caches[0], tables=wide[:, :2], lengths=lengths, rotary=table)
        b = ops().launch_append_kv(q=q.contiguous(), k=k.contiguous(), v=v.contiguous(), cache=caches[1], tables=wide[:, :2].contiguous(),
                                   lengths=lengths, rotary=table)
        apart = fused.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost: copied first
        c = ops().launch_append_kv(q=apart[:, :4], k=apart[:, 4:6], v=apart[:, 6:], cache=caches[2], tables=wide[:, :2],
                                   lengths=lengths, rotary=table)
        assert torch.equal(a, b) and torch.equal(a, c)
        at = ref.device(gpu, np.zeros(n, np.int32), np.arange(n, dtype=np.int32))
        reads = [ops().launch_read_kv(cache, wide[:, :2], *at) for cache in caches]
        assert all(torch.equal(x, y) for r in reads[1:] for x, y in zip(reads[0], r))


def test_rows_before_the_first_sequence_and_queries_in_place(gpu):
    """Offsets that do not begin at 0; out that is q itself."""
    from mambo_amd.kernels.rotary import launch_rotary
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    rng = np.random.default_rng(8)
    heads, dim, page = 2, 64, 32
    table = prepare_rotary_table(dim)
    for counts, skip in (([40, 3], 70), ([1, 1], 3), ([0, 100], 33)):
        n = sum(counts) + skip
        host, pages = ref.tables_of(rng, counts, page)
        tables, cache = ref.device(gpu, host)[0], new_cache(pages, heads, dim, page)
        k, v, q = (rows_of(rng, n, h, dim, torch.bfloat16).to(gpu) for h in (heads, heads, 4))
        before, offsets = q.clone(), ref.offsets_of(counts) + skip
        got = ops().launch_append_kv(k, v, cache, tables, *ref.device(gpu, np.array(counts, np.int32)), offsets=ref.device(gpu, offsets)[0],
                                     rotary=table, q=q, out=q, positions=torch.zeros(n, dtype=torch.int32, device=gpu) + 9)
        assert got is q and torch.equal(q[:skip], before[:skip])
        nine = torch.full((n,), 9, dtype=torch.int32, device=gpu)
        assert torch.equal(q[skip:], launch_rotary(before, nine, table)[skip:])
        got_k, got_v = read_all(cache, tables, counts)
        turned = launch_rotary(k.float(), nine, table).double().cpu().numpy()
        for s, c in enumerate(counts):
            model = ref.Model(heads, dim)
            if c:
                model.append(turned[offsets[s]:offsets[s + 1]], v[offsets[s]:offsets[s + 1]].double().cpu().numpy(), 0)
            same(got_k[s], model.k)
            same(got_v[s], model.v)


def test_copies_of_a_cache_are_their_own(gpu):
    import copy
    import dataclasses
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    rng = np.random.default_rng(9)
    cache = new_cache(1, 1, 32, 32)
    tables, lengths = torch.zeros((1, 1), dtype=torch.int32, device=gpu), torch.tensor([5], dtype=torch.int32, device=gpu)
    other, table = copy.deepcopy(cache), copy.deepcopy(prepare_rotary_table(32))
    assert other.args.codes == other.codes.data_ptr() != cache.codes.data_ptr() and table.args.turns == table.turns.data_ptr()
    x = rows_of(rng, 5, 1, 32, torch.float32).to(gpu)
    ops().launch_append_kv(x, x, other, tables, lengths, rotary=table)
    assert (cache.codes == 0x7F).all() and not (other.codes == 0x7F).all()
    for wrong in ({"page_size": 64}, {"heads": 2}, {"head_dim": 64}, {"codes": cache.codes[..., :-64]}, {"scales": cache.scales.float()},
                  {"scales": cache.scales.cpu()}, {"head_dim": 20}):
        with pytest.raises(ValueError):
            dataclasses.replace(cache, **wrong)
    with pytest.raises(ValueError):
        dataclasses.replace(table, size=64)


def test_refusals(gpu):
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    cache, table = new_cache(2, 2, 64, 32), prepare_rotary_table(64)
    tables, lengths = torch.zeros((2, 1), dtype=torch.int32, device=gpu), torch.ones(2, dtype=torch.int32, device=gpu)
    k, q = torch.zeros((4, 2, 64), device=gpu), torch.zeros((4, 4, 64), device=gpu)
    good = dict(k=k, v=k, cache=cache, tables=tables, lengths=lengths)
    ops().launch_append_kv(**good)
    for change in ({"k": k.half()}, {"k": k[..., :32]}, {"k": q}, {"v": k.bfloat16()}, {"v": k[:2]}, {"k": k.cpu()}, {"v": k.cpu()},
                   {"tables": tables.long()}, {"tables": tables[0]}, {"tables": tables.cpu()}, {"tables": tables[:0]},
                   {"tables": torch.zeros((2, 4), dtype=torch.int32, device=gpu)[:, ::2]}, {"lengths": lengths[:1]}, {"lengths": lengths.long()},
                   {"offsets": lengths}, {"k": k[:3], "v": k[:3]}, {"q": q}, {"rotary": table, "q": q.bfloat16()}, {"rotary": table, "q": q[:, :3]},
                   {"rotary": table, "q": q[:2]}, {"positions": torch.zeros(4, dtype=torch.int32, device=gpu)},
                   {"rotary": table, "positions": lengths}, {"rotary": prepare_rotary_table(128)}, {"out": q.bfloat16()},
                   {"rotary": table, "q": q, "out": q}, {"rotary": table, "q": q, "out": q.bfloat16()[:2]},
                   {"rotary": table, "q": q, "out": torch.zeros((1, 4, 64), dtype=torch.bfloat16, device=gpu).expand(4, 4, 64)}):
        with pytest.raises(ValueError):
            ops().launch_append_kv(**(good | change))
    for change in ({"cache": None}, {"rotary": "angles"}):
        with pytest.raises(TypeError):
            ops().launch_append_kv(**(good | change))
    assert ops().launch_append_kv(**(good | {"k": k[:0], "v": k[:0]}), rotary=table, q=q[:0]).shape == (0, 4, 64)
    for args in ((lengths.long(), lengths), (lengths, lengths[:1]), (lengths[None], lengths)):
        with pytest.raises(ValueError):
            ops().launch_read_kv(cache, tables, *args)
    assert ops().launch_read_kv(cache, tables, lengths[:0], lengths[:0])[0].shape == (0, 2, 64)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("start,n", [(64, 1), (96, 3), (40, 40), (0, 200), (63, 2), (70, 100), (5000, 1), (2**31 - 41, 40), (2**31 - 2, 1),
                                     (-20, 300)])
def test_tokens_past_a_table_are_dropped(gpu, start, n, ragged):
    """A table of 64 tokens whose sequence grows past it: what is cached stays, rows within it are stored at their own
    positions, the others nowhere, and queries turn by the positions that the lengths say."""
    from mambo_amd.kernels.rotary import launch_rotary
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    rng = np.random.default_rng(20)
    heads, dim = 2, 64
    cache, table = new_cache(4, heads, dim, 32), prepare_rotary_table(dim)
    tables = torch.tensor([[3, 0]], dtype=torch.int32, device=gpu)
    old_k, old_v = rows_of(rng, 64, heads, dim, torch.bfloat16), rows_of(rng, 64, heads, dim, torch.bfloat16)
    ops().launch_append_kv(old_k.to(gpu), old_v.to(gpu), cache, tables, torch.tensor([64], dtype=torch.int32, device=gpu))
    before = cache.codes.clone(), cache.scales.clone()
    model = ref.Model(heads, dim)
    model.append(old_k.double().numpy(), old_v.double().numpy(), 0)
    k, v, q = (rows_of(rng, n, h, dim, torch.float32).to(gpu) for h in (heads, heads, 4))
    positions = torch.arange(start, start + n, device=gpu).int()
    got = ops().launch_append_kv(k, v, cache, tables, torch.tensor([start + n], dtype=torch.int32, device=gpu), rotary=table, q=q,
                                 offsets=torch.tensor([0, n], dtype=torch.int32, device=gpu) if ragged else None)
    assert torch.equal(got, launch_rotary(q, positions, table, out_dtype=torch.bfloat16))
    stored = (positions >= 0) & (positions < 64)
    if not stored.any():
        assert torch.equal(cache.codes, before[0]) and torch.equal(cache.scales, before[1])
        return
    turned = launch_rotary(k, positions, table)[stored].double().cpu().numpy()
    model.append(turned, v[stored].double().cpu().numpy(), max(start, 0))
    got_k, got_v = read_all(cache, tables, [64])
    same(got_k[0], model.k)
    same(got_v[0], model.v)


def test_a_captured_step_replayed_past_its_table(gpu):
    rng = np.random.default_rng(21)
    heads, dim = 1, 64
    cache = new_cache(2, heads, dim, 32)
    tables, lengths = torch.tensor([[1]], dtype=torch.int32, device=gpu), torch.tensor([29], dtype=torch.int32, device=gpu)
    old = rows_of(rng, 29, heads, dim, torch.bfloat16).to(gpu)
    ops().launch_append_kv(old, old, cache, tables, lengths)
    new = rows_of(rng, 1, heads, dim, torch.bfloat16).to(gpu)
    model = ref.Model(heads, dim)
    model.append(old.double().cpu().numpy(), old.double().cpu().numpy(), 0)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        lengths.add_(1)
        ops().launch_append_kv(new, new, cache, tables, lengths)
    torch.cuda.synchronize()
    for step in range(6):  # three tokens fit
        new.copy_(rows_of(rng, 1, heads, dim, torch.bfloat16, 1.0 + step))
        if step < 3:
            model.append(new.double().cpu().numpy(), new.double().cpu().numpy(), 29 + step)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got_k, got_v = read_all(cache, tables, [len(model.k)])
        same(got_k[0], model.k)
        same(got_v[0], model.v)
    assert int(lengths) == 35


@pytest.mark.parametrize("dim,size,interleaved", [(64, 64, False), (64, 32, True), (128, 128, False), (80, 20, False), (72, 18, True), (256, 256, True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotated_keys_are_rounded_as_the_exact_ones(gpu, dim, size, interleaved, dtype):
    """A rotated key's code is that of the rotation in 64 bits, but where that lies as close to the border between two codes as the
    rotation's last bits reach."""
    from mambo_amd.utils.rotary_table import prepare_rotary_table, rotary_frequencies
    rng = np.random.default_rng(dim + size)
    heads, n = 2, 96
    cache = new_cache(3, heads, dim, 32)
    tables, lengths = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=gpu), torch.tensor([n], dtype=torch.int32, device=gpu)
    k = rows_of(rng, n, heads, dim, dtype)
    positions = rng.integers(0, 50000, n).astype(np.int32)
    ops().launch_append_kv(k.to(gpu), k.to(gpu), cache, tables, lengths, rotary=prepare_rotary_table(size, interleaved=interleaved),
                           positions=ref.device(gpu, positions)[0])
    frequencies = rotary_frequencies(size)[0]
    turned = ref.rotate(k.double().numpy(), positions, frequencies, interleaved)
    off = ref.turn_bound(k.double().numpy(), positions, frequencies, interleaved)
    got = read_all(cache, tables, [n])[0][0]
    settled = 0
    for block in range(3):
        part = slice(32 * block, 32 * block + 32)
        for h in range(heads):
            low, high = turned[part, h] - off[part, h], turned[part, h] + off[part, h]
            e = ref.exponent(float(np.abs(turned[part, h]).max()))
            assert e == ref.exponent(float(np.maximum(np.abs(low), np.abs(high)).max()))
            low, high = ref.nearest(low, e), ref.nearest(high, e)
            assert ((low <= got[part, h]) & (got[part, h] <= high)).all()
            settled += int((low == high).sum())
    assert settled >= 0.999 * turned.size


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_arrays_of_any_values_write_nothing_elsewhere(gpu, dtype):
    """Lengths, offsets and pages of any values: what lies around the cache and the rotated queries stays, and so do pages that no
    table names, queries of no sequence, and what is read."""
    from mambo_amd.utils.kv_cache import KVCache
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    from test_gpu_attention import HOSTILE_LENGTHS, HOSTILE_OFFSETS, Guarded
    rng = np.random.default_rng(32)
    heads, dim, pages, n = 2, 64, 8, 90
    table = prepare_rotary_table(dim)
    tables = torch.tensor([[4, 99, 1], [2, -7, 2**31 - 1], [2**31 - 1, -2**31, 6]], dtype=torch.int64, device=gpu).int()
    k, v, q = (rows_of(rng, n, h, dim, dtype).to(gpu) for h in (heads, heads, 4))
    given = [t.clone() for t in (tables, k, v, q)]
    for bad in HOSTILE_LENGTHS:
        on = torch.tensor(bad, dtype=torch.int64, device=gpu).int()
        for cuts in HOSTILE_OFFSETS:
            codes, scales = Guarded(gpu, (pages, heads, 1, 2 * 32 * dim), torch.uint8, 0x51), Guarded(gpu, (pages, heads, 1, 2), torch.uint8, 0x80)
            out = Guarded(gpu, (n, 4, dim), torch.bfloat16, 7.0)
            cache = KVCache(codes.inner, scales.inner, heads, dim, 32)
            ops().launch_append_kv(k, v, cache, tables, on, offsets=None if cuts is None else torch.tensor(cuts, dtype=torch.int64, device=gpu).int(),
                                   rotary=table, q=q, out=out.inner)
            torch.cuda.synchronize()
            assert codes.untouched() and scales.untouched() and out.untouched(), (bad, cuts)
            assert (codes.inner[[0, 3, 5, 7]] == 0x51).all() and (scales.inner[[0, 3, 5, 7]] == 0x80).all(), (bad, cuts)
            if cuts == [7, 7, 7, 7]:
                assert (out.inner == 7.0).all() and (codes.inner == 0x51).all()
            if cuts == [0, 1, 2, 3]:
                assert (out.inner[3:] == 7.0).all()
    at = torch.from_numpy(rng.integers(-2**31, 2**31, (2, 500))).int().to(gpu)
    at[0, :400] %= 3
    at[1, :300] %= 96
    got = ops().launch_read_kv(cache, tables, at[0].contiguous(), at[1].contiguous())
    there = (at[0] >= 0) & (at[0] < 3) & (at[1] >= 0) & (at[1] < 96)
    named = torch.tensor([[1, 0, 1], [1, 0, 0], [0, 0, 1]], device=gpu).bool()
    there &= named[at[0].clamp(0, 2).long(), (at[1].clamp(0, 95) // 32).long()]
    assert there.sum() > 50 and not got[0][~there].any() and not got[1][~there].any() and got[0][there].any(2).all()
    assert all(torch.equal(a, b) for a, b in zip(given, (tables, k, v, q)))
