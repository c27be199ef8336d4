"""The operators between the projections together: the block of a layer against 64 bits, its command, HIP graphs that
are replayed as sequences grow, named streams, several calls at once."""

from __future__ import annotations

import json

import numpy as np
import pytest
import torch

import kv_reference as ref
from conftest import make_synthetic_iq3_s
from oracle import oracle
from test_gpu_kv_cache import new_cache, read_all, rows_of

pytestmark = pytest.mark.gpu


def prepared(gpu, n, k, seed):
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_fields
    raw = make_synthetic_iq3_s(n, k, seed=seed)
    return prepare_iq3_s_fields(torch.from_numpy(raw).to(gpu)), raw


def test_block_against_64_bits(gpu):
    """Prompts of two sequences, then two tokens each. The projections are the oracle's, on the rows that each was given;
    between them stands the definition."""
    from mambo_amd.utils.attention_layer import AttentionLayer
    from mambo_amd.utils.kv_cache import allocate_kv_cache
    from mambo_amd.utils.rotary_table import prepare_rotary_table, rotary_frequencies
    heads, group, dim, width = 2, 2, 64, 256
    q_heads = heads * group
    (q, rq), (k, rk), (v, rv), (o, ro) = (prepared(gpu, n, kk, s) for s, (n, kk) in enumerate(
        ((q_heads * dim, width), (heads * dim, width), (heads * dim, width), (width, q_heads * dim))))
    layer = AttentionLayer(q, k, v, o, prepare_rotary_table(dim))
    frequencies = rotary_frequencies(dim)[0]
    rng = np.random.default_rng(0)
    cache = allocate_kv_cache(6, heads, dim, page_size=32)
    tables = torch.tensor([[5, 1, -1], [0, 3, 4]], dtype=torch.int32, device=gpu)
    models = [ref.Model(heads, dim) for _ in range(2)]
    lengths = np.zeros(2, dtype=np.int32)
    for counts in ([33, 40], [1, 1], [2, 2]):
        starts, n = lengths.copy(), sum(counts)
        lengths += np.array(counts, dtype=np.int32)
        x = torch.from_numpy(rng.standard_normal((n, width)).astype(np.float32)).to(torch.bfloat16)
        out = layer(x.to(gpu), cache, tables, *ref.device(gpu, lengths), *ref.device(gpu, ref.offsets_of(counts)))
        rows = oracle.quantize_mxfp8(x.float().numpy())
        q64, k64, v64 = (oracle.iq3s_fp8_matmul(*rows, raw).astype(np.float64).reshape(n, -1, dim) for raw in (rq, rk, rv))
        positions = np.concatenate([np.arange(s, s + c) for s, c in zip(starts, counts)])
        q64, k64 = ref.rotate(q64, positions, frequencies, False), ref.rotate(k64, positions, frequencies, False)
        cuts, a = ref.offsets_of(counts), np.zeros((n, q_heads, dim))
        for s in range(2):
            part = slice(cuts[s], cuts[s + 1])
            models[s].append(k64[part], v64[part], int(starts[s]))
            a[part] = ref.attend(q64[part], models[s].k, models[s].v, group, dim ** -0.5, True, 0)[0]
        expected = oracle.iq3s_fp8_matmul(*oracle.quantize_mxfp8(a.reshape(n, -1).astype(np.float32)), ro).astype(np.float64)
        got = out.double().cpu().numpy()
        # Scores of a few hundred let single tokens win, so that a code that a projection's last bits move to its
        # neighbour (2^-4 of a key) can change a row: all rows together, with the 2^-4 of the codes between.
        assert np.linalg.norm(got - expected) <= 0.05 * np.linalg.norm(expected)


def test_command(gpu, capsys):
    from mambo_amd.utils import attention_layer
    for extra in ([], ["--window", "20", "--page-size", "32"]):
        assert attention_layer.main(["--users", "3", "--prompt", "45", "--steps", "5", *extra]) == 0
        line = json.loads(capsys.readouterr().out)
        assert line["graph_equals_eager"] and line["graph_us"] > 0 and line["output_rms"] > 0


@pytest.mark.parametrize("ragged", [False, True])
def test_two_graphs_with_their_own_caches(gpu, ragged):
    """Two captured steps, replayed in turn and at once on two streams, between eager calls; lengths grow on the device."""
    from mambo_amd.kernels.attention import launch_attention_kv
    from mambo_amd.kernels.kv_cache import launch_append_kv
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    rng = np.random.default_rng(1)
    heads, group, dim, page, steps = 2, 4, 64, 32, 6
    table = prepare_rotary_table(dim)
    runs = []
    for start in ([3000, 100], [40, 1500]):  # long enough to be split and joined
        host, pages = ref.tables_of(rng, [n + steps * 2 for n in start], page)
        tables, cache = ref.device(gpu, host)[0], new_cache(pages, heads, dim, page)
        k, v = rows_of(rng, sum(start), heads, dim, torch.bfloat16).to(gpu), rows_of(rng, sum(start), heads, dim, torch.bfloat16).to(gpu)
        lengths = ref.device(gpu, np.array(start, np.int32))[0]
        launch_append_kv(k, v, cache, tables, lengths, offsets=ref.device(gpu, ref.offsets_of(start))[0])
        new = [rows_of(rng, 2, h, dim, torch.float32).to(gpu) for h in (heads * group, heads, heads)]
        offsets = ref.device(gpu, np.array([0, 1, 2], np.int32))[0] if ragged else None
        runs.append((cache, tables, lengths, new, offsets))

    def step(cache, tables, lengths, new, offsets):
        lengths.add_(1)
        q = launch_append_kv(new[1], new[2], cache, tables, lengths, offsets=offsets, rotary=table, q=new[0])
        return launch_attention_kv(q, cache, tables, lengths, offsets=offsets, return_lse=True)

    def copied(run):
        from mambo_amd.utils.kv_cache import KVCache
        cache, tables, lengths, new, offsets = run
        return (KVCache(cache.codes.clone(), cache.scales.clone(), cache.heads, cache.head_dim, cache.page_size), tables,
                lengths.clone(), new, offsets)

    eager = [copied(r) for r in runs]
    expected = [[tuple(t.clone() for t in step(*r)) for _ in range(steps)] for r in eager]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for run, stream in zip(runs, streams):
        saved = run[2].clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            outs.append(step(*run))
        graphs.append(graph)
        assert torch.equal(run[2], saved)
    torch.cuda.synchronize()
    for i in range(steps):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        step(*copied(eager[0]))  # other work in between
        torch.cuda.synchronize()
        for got, want in zip(outs, expected):
            assert torch.equal(got[0], want[i][0]) and torch.equal(got[1], want[i][1]), i


def test_named_streams(gpu):
    """Every operator on a stream that is not the current one, after work of that stream: what they allocate and copy
    belongs to it, too."""
    from mambo_amd.kernels.attention import launch_attention_kv
    from mambo_amd.kernels.kv_cache import launch_append_kv, launch_read_kv
    from mambo_amd.kernels.rotary import launch_rotary
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    from test_gpu_named_streams import freed_blocks_of, made_on
    rng = np.random.default_rng(2)
    heads, group, dim, page, n = 2, 2, 64, 32, 200
    table = prepare_rotary_table(dim)
    lengths = torch.tensor([n], dtype=torch.int32, device=gpu)
    tables = torch.arange(7, dtype=torch.int32, device=gpu)[None]
    data = rows_of(rng, n, 8, 2 * dim, torch.float32).to(gpu)
    at = ref.device(gpu, np.zeros(n, np.int32), np.arange(n, dtype=np.int32))
    side = torch.cuda.Stream()

    def run(x, stream, cache):
        apart = x[..., ::2]  # values apart: copied first
        q = launch_append_kv(apart[:, 4:6], apart[:, 6:], cache, tables, lengths, rotary=table, q=apart[:, :4], stream=stream)
        turned = launch_rotary(apart, at[1], table, out_dtype=torch.bfloat16, stream=stream)
        out, lse = launch_attention_kv(q, cache, tables, lengths, return_lse=True, stream=stream)
        few = launch_attention_kv(turned[-1:, :4], cache, tables, lengths, stream=stream)
        return [q, turned, out, lse, few, *launch_read_kv(cache, tables, *at, stream=stream)]

    expected = run(data, None, new_cache(7, heads, dim, page))
    for stream in (side, side.cuda_stream):
        cache = new_cache(7, heads, dim, page)
        late = made_on(side, data, torch.zeros_like(data))
        freed_blocks_of([t.numel() * t.element_size() for t in expected])
        got = run(late, stream, cache)
        side.synchronize()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_calls_at_once_on_one_cache(gpu):
    """Attention of several streams over one cache: nothing of the calls is shared."""
    from mambo_amd.kernels.attention import launch_attention_kv
    from mambo_amd.kernels.kv_cache import launch_append_kv
    rng = np.random.default_rng(3)
    heads, group, dim, page, lengths = 2, 4, 128, 64, [5000, 3000]
    host, pages = ref.tables_of(rng, lengths, page)
    tables, cache = ref.device(gpu, host)[0], new_cache(pages, heads, dim, page)
    n = sum(lengths)
    on = ref.device(gpu, np.array(lengths, np.int32))[0]
    launch_append_kv(rows_of(rng, n, heads, dim, torch.bfloat16).to(gpu), rows_of(rng, n, heads, dim, torch.bfloat16).to(gpu), cache,
                     tables, on, offsets=ref.device(gpu, ref.offsets_of(lengths))[0])
    qs = [rows_of(rng, 2 * m, heads * group, dim, torch.bfloat16).to(gpu) for m in (1, 2, 90, 1)]
    expected = [launch_attention_kv(q, cache, tables, on) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(10):
        got = [launch_attention_kv(q, cache, tables, on, stream=s) for q, s in zip(qs, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, expected))
    keys, _ = read_all(cache, tables, [1, 1])
    assert all(np.isfinite(t).all() for t in keys)


@pytest.mark.parametrize("window", [0, 40])
def test_block_is_its_parts(gpu, window):
    """The layer bit for bit out of the operators that it is said to call, each of which has its own tests: prompts, then tokens,
    of uniform and of ragged sequences."""
    from mambo_amd.kernels.attention import launch_attention_kv
    from mambo_amd.kernels.iq3_s_fp8 import launch_iq3_s_fp8_matmul
    from mambo_amd.kernels.kv_cache import launch_append_kv
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    from mambo_amd.kernels.rotary import launch_rotary
    from mambo_amd.utils.attention_layer import AttentionLayer
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    heads, group, dim, width = 2, 4, 64, 512
    shapes = ((heads * group * dim, width), (heads * dim, width), (heads * dim, width), (width, heads * group * dim))
    (q, _), (k, _), (v, _), (o, _) = (prepared(gpu, n, kk, s) for s, (n, kk) in enumerate(shapes))
    table = prepare_rotary_table(dim)
    layer = AttentionLayer(q, k, v, o, table, window)
    rng = np.random.default_rng(5)
    caches = [new_cache(6, heads, dim, 32) for _ in range(2)]
    tables = torch.tensor([[5, 1, -1], [0, 3, 4]], dtype=torch.int32, device=gpu)
    lengths = np.zeros(2, dtype=np.int32)
    for counts, ragged in (([33, 40], True), ([2, 2], False), ([1, 1], True), ([1, 1], False)):
        starts, n = lengths.copy(), sum(counts)
        lengths += np.array(counts, dtype=np.int32)
        x = rows_of(rng, n, 1, width, torch.bfloat16).view(n, width).to(gpu)
        on = ref.device(gpu, lengths)[0]
        offsets = ref.device(gpu, ref.offsets_of(counts))[0] if ragged else None
        out = layer(x, caches[0], tables, on, offsets)
        rows = launch_quantize_fp8(x)
        q_rows, k_rows, v_rows = (launch_iq3_s_fp8_matmul(*rows, w).view(n, -1, dim) for w in (q, k, v))
        positions = ref.device(gpu, np.concatenate([np.arange(s, s + c) for s, c in zip(starts, counts)]).astype(np.int32))[0]
        launch_append_kv(k_rows, v_rows, caches[1], tables, on, offsets=offsets, rotary=table)
        turned = launch_rotary(q_rows, positions, table, out_dtype=torch.bfloat16)
        a = launch_attention_kv(turned, caches[1], tables, on, offsets=offsets, window=window)
        expected = launch_iq3_s_fp8_matmul(*launch_quantize_fp8(a.view(n, -1)), o)
        assert torch.equal(caches[0].codes, caches[1].codes) and torch.equal(caches[0].scales, caches[1].scales)
        assert torch.equal(out, expected), counts


def attended(cache, tables, lengths, q, **more):
    from mambo_amd.kernels.attention import launch_attention_kv
    return launch_attention_kv(q, cache, tables, lengths, return_lse=True, **more)


def equal(a, b):
    """Bit for bit: tokens that were never stored are NaN in these caches, and so is what sees them."""
    return all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(a, b))


@pytest.mark.parametrize("page", [32, 64])
def test_a_prefix_shared_and_a_page_copied(gpu, page):
    """Two sequences with the pages of one prefix, and the page that both go on in copied whole: as if each had its own."""
    from mambo_amd.kernels.kv_cache import launch_append_kv
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    rng = np.random.default_rng(6)
    heads, group, dim, prefix = 2, 4, 64, 2 * page + 45 % page
    table = prepare_rotary_table(dim)
    cache, alone = new_cache(9, heads, dim, page), new_cache(9, heads, dim, page)
    shared = torch.tensor([[4, 0, 7, 2], [4, 0, 5, 3]], dtype=torch.int32, device=gpu)
    own = torch.tensor([[0, 1, 2, 3], [4, 5, 6, 7]], dtype=torch.int32, device=gpu)
    old = [rows_of(rng, prefix, heads, dim, torch.bfloat16).to(gpu) for _ in range(2)]
    at = ref.device(gpu, np.array([prefix], np.int32))[0]
    launch_append_kv(*old, cache, shared[:1], at, rotary=table)
    cache.codes[5], cache.scales[5] = cache.codes[7], cache.scales[7]
    launch_append_kv(*(torch.cat([t, t]) for t in old), alone, own, at.repeat(2), rotary=table)
    counts, lengths = np.array([1, 50]), at.repeat(2)
    for _ in range(2):
        n = int(counts.sum())
        lengths = lengths + torch.from_numpy(counts).int().to(gpu)
        offsets = ref.device(gpu, ref.offsets_of(counts))[0]
        k, v, q = (rows_of(rng, n, h, dim, torch.bfloat16, 3.0).to(gpu) for h in (heads, heads, heads * group))
        got = launch_append_kv(k, v, cache, shared, lengths, offsets=offsets, rotary=table, q=q)
        want = launch_append_kv(k, v, alone, own, lengths, offsets=offsets, rotary=table, q=q)
        assert torch.equal(got, want)
        assert equal(attended(cache, shared, lengths, got, offsets=offsets), attended(alone, own, lengths, got, offsets=offsets))
        counts = counts[::-1].copy() % 20


@pytest.mark.parametrize("n,ragged", [(1, False), (1, True), (60, False), (60, True)])
def test_replays_with_any_lengths(gpu, n, ragged):
    """A call captured while its sequences are empty and replayed as they are long, short, past their tables and empty again, with
    other queries and pages; eager calls and other work between."""
    from mambo_amd.kernels.attention import launch_attention_kv
    from test_gpu_attention import filled
    rng = np.random.default_rng(7)
    heads, group, dim, page, full = 2, 4, 64, 32, [4000, 2500, 64]
    cache, tables, _, _ = filled(gpu, rng, full, heads, dim, page)
    counts = [n, 2, 3 * n] if ragged else [n] * 3
    offsets = ref.device(gpu, ref.offsets_of(counts))[0] if ragged else None
    q = rows_of(rng, sum(counts), heads * group, dim, torch.bfloat16).to(gpu)
    lengths, live = torch.zeros(3, dtype=torch.int32, device=gpu), tables.clone()
    attended(cache, live, lengths, q, offsets=offsets)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        got = attended(cache, live, lengths, q, offsets=offsets)
    torch.cuda.synchronize()
    for step, values in enumerate((full, [0, 0, 0], [4000, 0, 1], [1, 2500, 64], [33, 64, 5], [4100, 2600, 70], [2**31 - 1, 3, 2000], full)):
        lengths.copy_(torch.tensor(values, dtype=torch.int32))
        q.copy_(rows_of(rng, sum(counts), heads * group, dim, torch.bfloat16))
        live.copy_(tables if step % 2 else tables[[0, 1, 2]].roll(1, 1))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert equal(got, attended(cache, live, lengths, q, offsets=offsets)), values
    empty = launch_attention_kv(q[:0], cache, tables, lengths, return_lse=True)
    assert empty[0].shape == (0, heads * group, dim) and empty[1].shape == (0, heads * group)


@pytest.mark.parametrize("page", [1024, 65536])
def test_large_pages(gpu, page):
    from test_gpu_attention import check
    from mambo_amd.kernels.kv_cache import launch_append_kv
    rng = np.random.default_rng(8)
    heads, group, dim, lengths = 2, 3, 40, [1500, 31]
    cache = new_cache(4, heads, dim, page)
    tables = torch.tensor([[2, 0], [3, -1]], dtype=torch.int32, device=gpu)
    models = [ref.Model(heads, dim) for _ in lengths]
    for start, end in (([0, 0], [1400, 30]), ([1400, 30], lengths)):
        counts = [b - a for a, b in zip(start, end)]
        k, v = (rows_of(rng, sum(counts), heads, dim, torch.bfloat16) for _ in range(2))
        launch_append_kv(k.to(gpu), v.to(gpu), cache, tables, *ref.device(gpu, np.array(end, np.int32)),
                         offsets=ref.device(gpu, ref.offsets_of(counts))[0])
        cuts = ref.offsets_of(counts)
        for s, model in enumerate(models):
            model.append(k[cuts[s]:cuts[s + 1]].double().numpy(), v[cuts[s]:cuts[s + 1]].double().numpy(), start[s])
    for n in (1, 90):
        q = rows_of(rng, 2 * n, heads * group, dim, torch.bfloat16).to(gpu)
        out, lse = attended(cache, tables, *ref.device(gpu, np.array(lengths, np.int32)), q)
        check(out, lse, q, [m.k for m in models], [m.v for m in models], [n, n], group)


def test_appends_at_once_to_one_cache(gpu):
    """Sequences of one cache that grow on streams of their own."""
    from mambo_amd.kernels.kv_cache import launch_append_kv
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    rng = np.random.default_rng(9)
    heads, dim, page, users = 2, 64, 32, 4
    table = prepare_rotary_table(dim)
    caches = [new_cache(4 * users, heads, dim, page) for _ in range(2)]
    tables = torch.from_numpy(rng.permutation(4 * users).astype(np.int32).reshape(users, 4)).to(gpu)
    streams = [torch.cuda.Stream() for _ in range(users)]
    held = np.zeros(users, dtype=np.int32)
    for step in range(6):
        counts = [40, 1, 7, 1, 30, 2][step:] + [40, 1, 7, 1, 30, 2][:step]
        data = [[rows_of(rng, c, h, dim, torch.float32).to(gpu) for h in (heads, heads, 4)] for c in counts[:users]]
        held += np.array(counts[:users], dtype=np.int32)
        lengths = ref.device(gpu, np.minimum(held, 128).astype(np.int32))[0]
        outs = []
        torch.cuda.synchronize()
        for u, stream in enumerate(streams):
            k, v, q = data[u]
            outs.append(launch_append_kv(k, v, caches[0], tables[u:u + 1], lengths[u:u + 1], rotary=table, q=q, stream=stream))
        torch.cuda.synchronize()
        for u in range(users):
            k, v, q = data[u]
            assert torch.equal(outs[u], launch_append_kv(k, v, caches[1], tables[u:u + 1], lengths[u:u + 1], rotary=table, q=q))
        assert torch.equal(caches[0].codes, caches[1].codes) and torch.equal(caches[0].scales, caches[1].scales)
