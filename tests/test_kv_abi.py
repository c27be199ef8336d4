"""The entry points of rotary positions, the paged cache and attention without a GPU: sizes, frequencies, which kernels a
call takes, the layout of a block, and arguments that are refused before the device is touched."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

import kv_reference as ref


@pytest.fixture(scope="module")
def lib():
    from mambo_amd import _native
    return _native.lib()


def refused(lib, rc, text):
    from mambo_amd import _native
    assert rc == _native.MAMBO_ERR_VALUE and text in lib.mambo_last_error().decode(), (rc, lib.mambo_last_error())


def cache(**change):
    from mambo_amd import _native
    args = {"codes": 256, "scales": 256, "pages": 10, "heads": 2, "head_dim": 64, "page_size": 32, "reserved": 0} | change
    return _native.KVCacheArgs(*args.values())


def batch(**change):
    from mambo_amd import _native
    args = {"tables": 256, "ldt": 5, "width": 5, "lengths": 256, "offsets": None, "seqs": 2} | change
    return _native.KVBatchArgs(*args.values())


def table(**change):
    from mambo_amd import _native
    args = {"turns": 256, "size": 64, "interleaved": 0, "magnitude": 1.0} | change
    return _native.RotaryTableArgs(*args.values())


def rows(**change):
    from mambo_amd import _native
    args = dict(k=256, v=256, q=None, ldkt=128, ldkh=64, ldvt=128, ldvh=64, ldqt=0, ldqh=0, q_out=None, ldot=0, ldoh=0, q_heads=0,
                dtype=0, reserved=0) | change
    return _native.KVRowsArgs(*args.values())


BAD_CACHES = [({"head_dim": 60}, "multiple of 8"), ({"head_dim": 0}, "multiple of 8"), ({"head_dim": 264}, "multiple of 8"),
              ({"page_size": 16}, "power of two"), ({"page_size": 96}, "power of two"), ({"page_size": 131072}, "power of two"),
              ({"pages": 0}, "a cache has"), ({"pages": 2**31}, "a cache has"), ({"heads": 0}, "a cache has"), ({"heads": 16385}, "a cache has"),
              ({"pages": 2**30, "heads": 2}, "at most 2^31 - 1 blocks"), ({"codes": None}, "null pointer"), ({"scales": None}, "null pointer"),
              ({"codes": 264}, "16-byte"), ({"scales": 257}, "2-byte")]
BAD_BATCHES = [({"seqs": 0}, "sequences must number"), ({"seqs": 2**24}, "sequences must number"), ({"width": 0}, "tables must hold"),
               ({"width": 2**26, "ldt": 2**26}, "tables must hold"), ({"ldt": 4}, "tables must hold"), ({"tables": None}, "null pointer"),
               ({"lengths": None}, "null pointer")]


def calls(lib):
    return {
        "append": lambda c, b, tokens=2: lib.mambo_kv_append(rows(), tokens, c, b, None, None, None),
        "attention": lambda c, b, tokens=2: lib.mambo_kv_attention(256, tokens, 4, 64, 256, 64, c, b, 1.0, 1, 0, 256, 256, 64, None,
                                                                  256, 1 << 40, None),
        "plan": lambda c, b, tokens=2: lib.mambo_kv_attention_plan(c, b, tokens, 4, 0, (ctypes.c_int32 * 4)()),
        "workspace": lambda c, b, tokens=2: lib.mambo_kv_attention_workspace(c, b, tokens, 4, 0),
    }


@pytest.mark.parametrize("name", ["append", "attention", "plan", "workspace"])
def test_caches_and_sequences_that_are_refused(lib, name):
    call = calls(lib)[name]
    for change, text in BAD_CACHES:
        refused(lib, call(cache(**change), batch()), text)
    for change, text in BAD_BATCHES:
        refused(lib, call(cache(), batch(**change)), text)
    refused(lib, call(None, batch()), "null pointer")
    refused(lib, call(cache(), None), "null pointer")
    refused(lib, call(cache(), batch(), -1), "rows must number")
    refused(lib, call(cache(), batch(), 2**30), "rows must number")
    refused(lib, call(cache(), batch(), 3), "as many rows")


def test_read_refusals(lib):
    f = lib.mambo_kv_read
    for change, text in BAD_CACHES:
        refused(lib, f(cache(**change), batch(), 256, 256, 3, 2, 64, 256, 256, None), text)
    for change, text in BAD_BATCHES[:-1]:
        refused(lib, f(cache(), batch(**change), 256, 256, 3, 2, 64, 256, 256, None), text)
    for args, text in (((256, 256, 3, 1, 64, 256, 256), "the cache has"), ((256, 256, 3, 2, 72, 256, 256), "the cache has"),
                       ((256, 256, -1, 2, 64, 256, 256), "negative"), ((None, 256, 3, 2, 64, 256, 256), "null pointer"),
                       ((256, None, 3, 2, 64, 256, 256), "null pointer"), ((256, 256, 3, 2, 64, None, 256), "null pointer"),
                       ((256, 256, 3, 2, 64, 264, 256), "16-byte"), ((256, 256, 2**40, 2, 64, 256, 256), "too many rows")):
        refused(lib, f(cache(), batch(), *args, None), text)
    assert f(cache(), batch(lengths=None), None, None, 0, 2, 64, None, None, None) == 0


@pytest.mark.parametrize("name", ["append", "attention", "plan", "workspace"])
def test_sizes_whose_products_wrap(lib, name):
    """Widths that 64 bits do not hold the tokens of, which wrap to nothing, to few and to a negative number of them."""
    for page_size, width in ((65536, 2**48), (65536, 2**48 + 5), (32, 2**59 + 3), (32, 2**58), (65536, 2**63 - 1), (32, 2**62 + 1)):
        refused(lib, calls(lib)[name](cache(page_size=page_size), batch(width=width, ldt=2**63 - 1)), "tables must hold")


def test_rows_to_read_that_wrap(lib):
    for n in (2**63 - 1, 2**63 - 31, 2**62):
        refused(lib, lib.mambo_kv_read(cache(), batch(), 256, 256, n, 2, 64, 256, 256, None), "too many rows")
    refused(lib, lib.mambo_kv_read(cache(page_size=65536), batch(width=2**48, ldt=2**48), 256, 256, 3, 2, 64, 256, 256, None), "tables must hold")


def test_rotary_refusals(lib):
    good = dict(x=256, xd=0, tokens=2, heads=2, dim=64, ldt=128, ldh=64, positions=256, table=table(), out=256, od=1, ldot=128, ldoh=64)

    def call(**change):
        return lib.mambo_rotary(*(good | change).values(), None)

    for change, text in (({"xd": 2}, "float32 or bfloat16"), ({"od": 3}, "float32 or bfloat16"), ({"tokens": -1}, "tokens of"),
                         ({"heads": 0}, "tokens of"), ({"heads": 65536}, "tokens of"), ({"dim": 1}, "tokens of"), ({"dim": 1025}, "tokens of"),
                         ({"table": None}, "null pointer"), ({"table": table(turns=None)}, "null pointer"),
                         ({"table": table(size=3)}, "even number"), ({"table": table(size=0)}, "even number"),
                         ({"table": table(size=66)}, "even number"), ({"table": table(turns=260)}, "aligned to their type"),
                         ({"x": None}, "null pointer"), ({"positions": None}, "null pointer"), ({"out": None}, "null pointer"),
                         ({"x": 258}, "aligned to their type"), ({"out": 257}, "aligned to their type"),
                         ({"ldot": 63}, "cover a head"), ({"ldoh": 63}, "cover a head")):
        refused(lib, call(**change), text)
    assert call(tokens=0, x=None, positions=None, out=None) == 0


def test_append_refusals(lib):
    f = lib.mambo_kv_append
    for r, t, text in ((rows(dtype=2), None, "float32 or bfloat16"), (rows(k=None), None, "null pointer (keys)"),
                       (rows(v=None), None, "null pointer (values)"), (rows(k=258), None, "aligned to their type"),
                       (rows(v=257, dtype=1), None, "aligned to their type"), (rows(q=256, q_out=256, q_heads=2), None, "need a table"),
                       (rows(q=256, q_out=256, q_heads=3), table(), "no multiple"), (rows(q=256, q_out=256, q_heads=1), table(), "no multiple"),
                       (rows(q=256, q_heads=2), table(), "null pointer (rotated"), (rows(q=258, q_out=256, q_heads=2), table(), "aligned"),
                       (rows(q=256, q_out=256, q_heads=2, ldot=128, ldoh=63), table(), "cover a head"),
                       (rows(), table(size=66), "even number"), (rows(), table(size=7), "even number")):
        refused(lib, f(r, 2, cache(), batch(), t, None, None), text)
    refused(lib, f(None, 2, cache(), batch(), None, None, None), "null pointer")
    assert f(rows(k=None, v=None), 0, cache(), batch(lengths=None), None, None, None) == 0


def test_attention_refusals(lib):
    good = dict(q=256, tokens=2, heads=4, dim=64, ldqt=256, ldqh=64, cache=cache(), batch=batch(), scale=1.0, causal=1, window=0, out=256,
                ldot=256, ldoh=64, lse=None, ws=256, size=1 << 40)

    def call(**change):
        return lib.mambo_kv_attention(*(good | change).values(), None)

    for change, text in (({"heads": 3}, "no multiple"), ({"heads": 0}, "no multiple"), ({"heads": 65538}, "no multiple"), ({"dim": 72}, "heads of"),
                         ({"scale": 0.0}, "positive and finite"), ({"scale": -1.0}, "positive and finite"),
                         ({"scale": math.inf}, "positive and finite"), ({"scale": math.nan}, "positive and finite"),
                         ({"window": -1}, "a window"), ({"window": 5, "causal": 0}, "a window"), ({"q": None}, "null pointer"),
                         ({"out": None}, "null pointer"), ({"q": 264}, "16-byte"), ({"ldqt": 260}, "16-byte"), ({"ldqh": 68}, "16-byte"),
                         ({"out": 257}, "aligned to their type"), ({"lse": 258}, "aligned to their type"), ({"ldoh": 63}, "cover a head"), ({"ldot": 63}, "cover a head"),
                         ({"batch": batch(width=600, ldt=600), "size": 0}, "workspace must hold"),
                         ({"batch": batch(width=600, ldt=600), "ws": None}, "workspace must hold"), ({"ws": 264}, "16-byte")):
        refused(lib, call(**change), text)
    assert call(tokens=0, q=None, out=None, ws=None) == 0
    big = batch(seqs=2**23, width=2**20, ldt=2**20)
    refused(lib, lib.mambo_kv_attention_workspace(cache(), big, 2**23, 4, 0), "2^36 tokens")
    refused(lib, lib.mambo_kv_attention_workspace(cache(heads=2), batch(seqs=2**23), 2**23, 1024, 0), "below 2^30")


def test_cache_bytes(lib):
    f = lib.mambo_kv_cache_bytes
    assert f(3, 2, 128, 64) == 3 * 2 * 64 * 2 * 128 and f(1, 1, 8, 32) == 32 * 2 * 32 and f(1, 1, 104, 32) == 32 * 2 * 128
    for bad in ((0, 2, 64, 32), (1, 0, 64, 32), (1, 16385, 64, 32), (1, 1, 63, 32), (1, 1, 264, 32), (1, 1, 64, 48), (1, 1, 64, 16),
                (2**30, 2, 64, 32), (-1, 1, 64, 32), (2**62, 4, 64, 32)):
        assert f(*bad) == 0


def test_plans(lib):
    """Few rows take one kernel, many another, calls of both kinds both; few keys take one workgroup a sequence."""
    def plan(tokens, q_heads, window=0, dim=64, heads=2, **b):
        out = (ctypes.c_int32 * 4)()
        assert lib.mambo_kv_attention_plan(cache(head_dim=dim, heads=heads), batch(**b), tokens, q_heads, window, out) == 0
        return list(out)

    assert plan(2, 8) == [16, 0, 0, 1]                       # 160 tokens at most
    assert plan(2, 8, width=40, ldt=40) == [16, 0, 0, 1]     # 1280
    assert plan(2, 8, width=41, ldt=41) == [16, 21, 0, 1]    # a share of four blocks and more
    assert plan(2, 8, width=10000, ldt=10000) == [16, 256, 0, 1]
    assert plan(2, 8, window=500, width=10000, ldt=10000) == [16, 0, 0, 1]
    assert plan(2, 256, heads=128, seqs=2, width=64, ldt=64)[:2] == [16, 0]  # 2048 tokens of 256 workgroups
    assert plan(2, 256, heads=128, seqs=2, width=65, ldt=65)[:2] == [16, 4]
    assert plan(32, 8)[0] == 64 and plan(32, 8, dim=128)[2] == 256 and plan(32, 4, dim=128)[0] == 32
    assert plan(34, 8)[:1] == [0] and plan(34, 8)[2] == 256 and plan(34, 8, dim=192)[2] == 256 and plan(34, 8, dim=200)[2] == 128
    wide = {"width": 2000, "ldt": 2000}
    assert plan(15 * 3, 8, seqs=3, **wide)[0] == 64 and plan(15 * 4, 8, seqs=4, **wide)[:3] == [0, 0, 256]
    assert plan(8 * 4, 8, seqs=4, **wide)[0] == 32 and plan(15, 8, seqs=4, offsets=256, **wide)[0] == 64
    assert plan(40, 8, offsets=256) == [16, 0, 256, 1]
    assert plan(40, 96, offsets=256)[0] == 64 and plan(40, 160, offsets=256)[0] == 0
    assert plan(400, 8, width=2000, ldt=2000)[3] == 256 // (2 * 4 * 2)
    assert plan(400, 8, seqs=1, width=2000, ldt=2000)[3] == 256 // (7 * 2) and plan(400, 8, offsets=256, width=2000, ldt=2000)[3] == 32


def test_every_kernel_that_is_built_is_one_that_a_call_takes(lib):
    """The kernels by head size (in 32s) and row tiles (of 16): their names in the library, and what the plans of calls of all
    head sizes, rows and lengths come to."""
    import re
    from mambo_amd import _native
    held = _native.LIB_PATH.read_bytes()
    names = {(k.decode(), int(ds), int(rt or 0))
             for k, ds, rt in re.findall(rb"attend_(short|rows|tiles)_kernelILi(\d+)E(?:Li(\d+)E)?E", held)}
    taken = set()
    for ds in range(1, 9):
        for group in (1, 16, 17, 32, 33, 64, 65, 300):
            for width in (5, 2000):
                for ragged in (None, 256):
                    out = (ctypes.c_int32 * 4)()
                    assert lib.mambo_kv_attention_plan(cache(head_dim=32 * ds, heads=1), batch(width=width, ldt=width, offsets=ragged), 2,
                                                       group, 0, out) == 0
                    if out[0]:
                        taken.add(("rows" if out[1] else "short", ds, out[0] // 16))
                    if out[2]:
                        taken.add(("tiles", ds, 0))
    assert names == taken


def test_calls_of_two_to_the_24_rows_and_more(lib):
    """What is launched decides, not the rows: of large calls nothing is joined."""
    def size(tokens, q_heads, dim=128, heads=8, **b):
        return lib.mambo_kv_attention_workspace(cache(head_dim=dim, heads=heads), batch(**b), tokens, q_heads, 0)

    assert 2**17 * 128 == 2**18 * 64 == 2**19 * 32 == 2**24
    for tokens, q_heads in ((2**17, 128), (2**18, 64), (2**19, 32), (2**23, 64), (2**24, 56)):
        for more in ({"seqs": 1}, {"seqs": 2}, {"seqs": 1, "offsets": 256}, {"seqs": 1, "width": 2**20, "ldt": 2**20}):
            assert size(tokens, q_heads, **more) == 0
    assert size(2**20, 16, dim=8, heads=1, seqs=2**20) == 0        # single tokens, a workgroup each
    assert size(2**20 - 1, 1023, dim=8, heads=1, seqs=2**20 - 1) == 0
    assert size(2**20 - 1, 16, dim=8, heads=1, seqs=2**20 - 1, width=65, ldt=65) > 0  # joined, a workgroup for each of 2^24 - 16 rows
    refused(lib, size(2**20, 16, dim=8, heads=1, seqs=2**20, width=65, ldt=65), "too many rows")
    refused(lib, size(2**23, 8, seqs=2**23), "too many rows")      # 2^26 workgroups of 512
    refused(lib, size(2**22, 1023, heads=1, dim=8, seqs=2), "below 2^30")


def test_the_blocks_layout_is_a_permutation():
    """As mambo_amd/csrc/kv_cache.h states it, for every padded head size."""
    for dim in range(32, 257, 32):
        token, d = np.meshgrid(np.arange(32), np.arange(dim), indexing="ij")
        keys = (d >> 5) * 1024 + ((((d >> 3) & 3) << 4) + ((token >> 3) << 2) + (token & 3)) * 16 + ((token >> 2) & 1) * 8 + (d & 7)
        values = (d >> 5) * 1024 + (((token >> 3) << 4) + (d & 15)) * 16 + ((d >> 4) & 1) * 8 + (token & 7)
        for at in (keys, values):
            assert sorted(at.ravel().tolist()) == list(range(32 * dim))


def test_frequencies():
    from mambo_amd.utils.rotary_table import rotary_frequencies
    plain, one = rotary_frequencies(8, base=10000.0)
    assert one == 1.0 and np.allclose(plain, [1.0, 0.1, 0.01, 0.001], rtol=1e-15)
    assert np.allclose(rotary_frequencies(8, scaling={"type": "linear", "factor": 4.0})[0], np.array(plain) / 4)
    ntk, _ = rotary_frequencies(8, scaling={"type": "ntk", "factor": 2.0})
    assert ntk[0] == 1.0 and math.isclose(ntk[3], plain[3] / 2)  # the slowest pair by the factor
    llama, _ = rotary_frequencies(8, scaling={"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                              "original_length": 1000})
    # wavelengths 6.3, 63 (below 250), 628 (between), 6283 (above 1000)
    turns = 1000 * 0.01 / (2 * math.pi)
    keep = (turns - 1) / 3
    assert np.allclose(llama, [1.0, 0.1, 0.01 * (keep + (1 - keep) / 8), 0.001 / 8], rtol=1e-14)
    yarn, magnitude = rotary_frequencies(64, scaling={"type": "yarn", "factor": 16.0, "original_length": 4096})
    base, _ = rotary_frequencies(64)
    assert math.isclose(magnitude, 0.1 * math.log(16) + 1) and yarn[0] == base[0] and math.isclose(yarn[-1], base[-1] / 16)
    assert all(b / 16 <= y <= b for y, b in zip(yarn, base))
    assert rotary_frequencies(64, scaling={"type": "yarn", "factor": 16.0, "original_length": 4096, "magnitude": 1.5})[1] == 1.5


@pytest.mark.parametrize("size,more", [
    (7, {}), (0, {}), (1026, {}), (64, {"base": 1.0}), (64, {"base": math.inf}), (64, {"scaling": {"type": "other", "factor": 2.0}}),
    (64, {"scaling": {"factor": 2.0}}), (64, {"scaling": {"type": "linear"}}), (64, {"scaling": {"type": "linear", "factor": 0.0}}),
    (64, {"scaling": {"type": "linear", "factor": 2.0, "extra": 1.0}}), (2, {"scaling": {"type": "ntk", "factor": 2.0}}),
    (64, {"scaling": {"type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "high_freq_factor": 1.0, "original_length": 8192}}),
    (64, {"scaling": {"type": "yarn", "factor": 8.0, "original_length": 4096, "beta_fast": 1.0}})])
def test_frequencies_that_are_refused(size, more):
    from mambo_amd.utils.rotary_table import rotary_frequencies
    with pytest.raises(ValueError):
        rotary_frequencies(size, **more)


def test_python_refuses_without_a_gpu():
    import torch
    from mambo_amd.kernels import attention, kv_cache, rotary
    from mambo_amd.utils.kv_cache import KVCache, allocate_kv_cache
    from mambo_amd.utils.rotary_table import RotaryTable, prepare_rotary_table
    x, i = torch.zeros((2, 2, 64)), torch.zeros(2, dtype=torch.int32)
    angles = RotaryTable(torch.zeros(32, dtype=torch.int64), 64, False, 1.0)
    held = KVCache(torch.zeros((4, 2, 1, 4096), dtype=torch.uint8), torch.zeros((4, 2, 1, 2), dtype=torch.uint8), 2, 64, 32)
    tables = torch.zeros((2, 2), dtype=torch.int32)
    for call in (lambda: rotary.launch_rotary(x, i, angles), lambda: rotary.launch_rotary(x.double(), i, angles),
                 lambda: kv_cache.launch_append_kv(x, x, held, tables, i), lambda: attention.launch_attention_kv(x.bfloat16(), held, tables, i),
                 lambda: allocate_kv_cache(1, 1, 63, device="cuda:0"), lambda: allocate_kv_cache(1, 1, 64, device="cpu"),
                 lambda: prepare_rotary_table(64, device="cpu"), lambda: prepare_rotary_table(64, frequencies=[1.0], device="cpu")):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: kv_cache.launch_append_kv(x, x, None, tables, i), lambda: kv_cache.launch_read_kv(None, tables, i, i),
                 lambda: attention.launch_attention_kv(x, None, tables, i)):
        with pytest.raises(TypeError):
            call()


def test_the_models_agree_with_hand_counts():
    """The statements that the GPU tests compare with, on cases small enough to see."""
    assert [ref.exponent(a) for a in (0.0, 448.0, 448.5, 224.0, 1e-40, 3.0e38)] == [-100, 0, 1, -1, -100, 120]
    m = ref.Model(1, 8)
    m.append(np.ones((3, 1, 8)), 0.01 * np.ones((3, 1, 8)), 0)
    m.append(500.0 * np.ones((1, 1, 8)), np.full((1, 1, 8), np.nan), 3)
    assert m.k[:3, 0, 0].tolist() == [1.0] * 3 and np.isnan(m.k[3]).all() and not m.v[3].any() and m.e[0, 0, "k"] == -8
    m.append(500.0 * np.ones((1, 1, 8)), np.ones((1, 1, 8)), 4)
    assert m.k[4, 0, 0] == 512.0 and m.e[0, 0, "k"] == 1 and m.e[0, 0, "v"] == -8
    x = ref.rotate(np.array([[[1.0, 0.0, 0.0, 2.0, 5.0]]]), [1], [math.pi / 2, math.pi], False)
    assert np.allclose(x, [[[0.0, 0.0, 1.0, -2.0, 5.0]]])
    out, lse, _, _ = ref.attend(np.zeros((2, 1, 8)), np.zeros((3, 1, 8)), np.arange(3.0)[:, None, None] * np.ones((3, 1, 8)), 1, 1.0, True, 2)
    assert np.allclose(out[:, 0, 0], [0.5, 1.5]) and np.allclose(lse, math.log(2))


@pytest.mark.parametrize("length,dim", [(40011, 64), (9000, 64), (131149, 128), (20000, 128), (6000, 256)])
def test_a_lost_or_repeated_block_shows(length, dim):
    """Mistakes planted in the statement that long caches are compared with: every block left out moves the lse, and one left out
    with another taken twice, or values of another block, move an output, by more than twice what the comparison allows."""
    rng = np.random.default_rng(length)
    k, v = ref.block_rows(rng, length, 1, dim)
    block = np.arange(length) // ref.BLOCK
    blocks = int(block[-1]) + 1
    out, lse, bound, lse_bound = ref.block_attend(k, v, 1, 3, False, 0)  # rows of each kind
    counts = np.bincount(block)
    assert (lse[0, 0] - np.log(length - counts) > 2 * lse_bound[0, 0]).all()
    sums = np.stack([np.bincount(block, v[:, 0, d]) for d in range(dim)], 1)  # [blocks, D]
    for shift in (1, 2, 7, blocks // 2, blocks - 1):
        moved = np.abs(np.roll(sums, shift, 0) - sums) / length  # block b for block b - shift
        assert (moved > 2 * (bound[0, 0] + 2.0**-8 * moved)).any(1).all(), shift
    first = np.arange(blocks) * ref.BLOCK
    for kind in (1, 2):  # weights of a block that come with another one's values
        w = 2.0 ** k[first, 0, kind - 1]
        total = (w * counts).sum()
        other = np.flatnonzero(w != np.roll(w, 1))
        moved = np.abs((w - np.roll(w, 1))[other, None] * sums[other]) / total
        assert len(other) > blocks // 4 and (moved > 2 * (bound[0, kind] + 2.0**-8 * moved)).any(1).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_angles_in_32_bits_are_told_apart(interleaved):
    """The kernel's arithmetic stays within the bound of a rotation, the same with an angle of 32 bits does not."""
    rng = np.random.default_rng(40)
    f = [10000.0 ** (-2 * i / 64) for i in range(32)]
    positions = rng.integers(0, 100000, 30)
    x = rng.standard_normal((30, 4, 64)).astype(np.float32)
    exact, bound = ref.rotate(x, positions, f, interleaved, 1.1), ref.turn_bound(x, positions, f, interleaved, 1.1)
    off = []
    for bits in (np.float64, np.float32):
        got = np.array(x)
        for i in range(32):
            i0, i1 = (2 * i, 2 * i + 1) if interleaved else (i, i + 32)
            angle = np.mod(positions * f[i] / (2 * math.pi) + 0.5, 1.0) * (2 * math.pi) - math.pi
            c, s = (np.float32(1.1 * t(angle.astype(bits).astype(np.float64)))[:, None].astype(np.float64) for t in (np.cos, np.sin))
            a, b = x[..., i0].astype(np.float64), x[..., i1].astype(np.float64)
            got[..., i0] = np.float32(a * c - np.float32(b * s).astype(np.float64))
            got[..., i1] = np.float32(a * s + np.float32(b * c).astype(np.float64))
        off.append(np.abs(got.astype(np.float64) - exact) / bound)
    assert off[0].max() <= 1.0 < 1.2 < off[1].max()
