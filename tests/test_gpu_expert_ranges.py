"""The operators of a layer of experts over the ranges that they accept: long prompts, the last sizes
before an index would not fit, and what lies beyond them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import expert_reference as ref


# ------------------------------------------------------------------------------ plain statements
def chosen(logits: np.ndarray, top_k: int) -> np.ndarray:
    """The ids of ref.route for many tokens: a stable sort of falling logits, -inf and NaN out."""
    logits = np.where(np.isnan(logits), -np.inf, logits)
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :top_k].astype(np.int32)
    return np.where(np.take_along_axis(logits, ids, 1) == -np.inf, np.int32(-1), ids)


def plan_of(ids: np.ndarray, experts: int):
    """ref.plan for many choices: a stable sort by expert, choices of none last."""
    m, top_k = ids.shape
    flat = np.where(ids < 0, experts, ids).ravel()
    order = np.argsort(flat, kind="stable")
    offsets = np.searchsorted(flat[order], np.arange(experts + 1)).astype(np.int32)
    taken = flat[order] < experts
    slots = np.empty(m * top_k, dtype=np.int32)
    slots[order] = np.where(taken, np.arange(m * top_k), -1)
    return offsets, np.where(taken, order // top_k, -1).astype(np.int32), slots.reshape(m, top_k)


def some_logits(rng, m: int, experts: int, masked: float) -> np.ndarray:
    """Logits on a coarse grid, so that many are equal, a share of them masked, some tokens wholly."""
    logits = rng.integers(-6, 7, size=(m, experts)).astype(np.float32)
    logits[rng.random((m, experts)) < masked] = -np.inf
    if masked:
        logits[rng.random(m) < 0.02] = -np.inf
        logits[rng.random(m) < 0.02, 0] = np.nan
    return logits


def test_the_statements_for_many_choices_are_those_for_few():
    rng = np.random.default_rng(0)
    for m, experts, top_k, masked in ((7, 5, 2, 0.5), (40, 9, 9, 0.3), (1, 1, 1, 0.0), (30, 3, 1, 0.9)):
        logits = some_logits(rng, m, experts, masked)
        ids = chosen(logits, top_k)
        assert np.array_equal(ids, ref.route(logits.astype(np.float64), top_k, True)[0])
        for a, b in zip(plan_of(ids, experts), ref.plan(ids, experts)):
            assert np.array_equal(a, b)


# ------------------------------------------------------------------------------ router
# more than 8192 choices, so that a wave's stretch of them passes the steps of 512 that no bound guards
@pytest.mark.gpu
@pytest.mark.parametrize("masked", [0.0, 0.4])
@pytest.mark.parametrize("m,experts,top_k", [(2731, 9, 3), (8193, 2, 1), (4101, 64, 8), (8192, 256, 8), (1025, 70, 64),
                                             (20011, 5, 5), (65537, 3, 1), (3001, 513, 10)])
def test_route_of_many_choices(gpu, m, experts, top_k, masked):
    from mambo_amd.kernels.experts import launch_route_experts
    logits = some_logits(np.random.default_rng(m + experts), m, experts, masked)
    ids = chosen(logits, top_k)
    for dtype in (torch.float32, torch.bfloat16):  # the grid's values are the same in both
        got = launch_route_experts(torch.from_numpy(logits).to(gpu).to(dtype), top_k)
        assert np.array_equal(got.ids.cpu().numpy(), ids)
        for name, expected in zip(("offsets", "rows", "slots"), plan_of(ids, experts)):
            assert np.array_equal(getattr(got, name).cpu().numpy(), expected), name


@pytest.mark.gpu
def test_route_of_the_most_choices(gpu):
    """2^31 - 64 choices: every token takes all of 64 experts, in an order of its own, so expert e has
    the rows e m to (e + 1) m, a token each."""
    from mambo_amd.kernels.experts import launch_route_experts
    m, experts = 2**25 - 1, 64
    logits = torch.empty((m, experts), dtype=torch.bfloat16, device=gpu)
    expert = torch.arange(experts, dtype=torch.int32, device=gpu)
    part = 1 << 20
    tokens = [torch.arange(t, min(t + part, m), dtype=torch.int32, device=gpu) for t in range(0, m, part)]
    for t in tokens:
        logits[t[0]:t[0] + t.shape[0]] = ((expert[None] + t[:, None]) % experts).to(torch.bfloat16)
    ids, weights, offsets, rows, slots = launch_route_experts(logits, experts)
    assert offsets.tolist() == [e * m for e in range(experts + 1)]
    rows = rows.view(experts, m)
    for t in tokens:
        at = slice(int(t[0]), int(t[0]) + t.shape[0])
        # the j-th choice is the expert with the logit 63 - j
        assert torch.equal(ids[at], (experts - 1 - expert[None] - t[:, None]) % experts)
        assert torch.equal(slots[at], ids[at] * m + t[:, None])
        assert bool((rows[:, at] == t[None]).all())
        assert bool(((weights[at].sum(1) - 1.0).abs() < 64 * 2.0**-23).all())
    del ids, weights, offsets, rows, slots, logits
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route_of_more_tokens_than_a_launch(gpu, dtype):
    """2^26 + 5 tokens, one workgroup for four: token t takes expert (2 - t) mod 3."""
    from mambo_amd.kernels.experts import launch_route_experts
    m = 2**26 + 5
    t = torch.arange(m, dtype=torch.int32, device=gpu)
    logits = torch.stack([(t + e) % 3 for e in range(3)], dim=1).to(dtype)
    ids, weights, offsets, rows, slots = launch_route_experts(logits, 1)
    expected = (2 - t) % 3
    counts = [int((expected == e).sum()) for e in range(3)]
    starts = [0, counts[0], counts[0] + counts[1], m]
    assert offsets.tolist() == starts and torch.equal(ids[:, 0], expected) and bool((weights == 1.0).all())
    assert torch.equal(slots[:, 0], torch.tensor(starts[:3], dtype=torch.int32, device=gpu)[expected.long()] + t // 3)
    assert torch.equal(rows, torch.cat([t[(2 - e) % 3::3] for e in range(3)]))


# ------------------------------------------------------------------------------ launches that no grid holds
GRID_THREADS = 2**32 - 1  # of a dimension
THREADS = {(16, 16, 8): 512, (16, 32, 4): 256, (16, 64, 4): 256, (32, 64, 4): 512, (64, 64, 4): 512, (64, 128, 2): 512,
           (64, 256, 2): 512, (64, 256, 1): 256, (128, 256, 1): 256}  # tokens, weight rows, K groups: of a workgroup


def refusal(rc, text):
    from mambo_amd import _native
    assert rc == _native.MAMBO_ERR_VALUE and text in _native.lib().mambo_last_error().decode()


@pytest.mark.parametrize("experts", [0, 1, 4, 1024])
@pytest.mark.parametrize("bf16", [True, False])
def test_products_are_planned_within_a_grid(experts, bf16):
    """Whatever the sizes, the kernel that is chosen fits a grid, or none does and the call is refused."""
    import ctypes
    from mambo_amd import _native
    lib, plan = _native.lib(), (ctypes.c_int32 * 5)()
    kernels = [k for k in THREADS if bf16 or k[0] < 128]
    taken = 0
    for r in (1, 1000, 2**20 + 1, 2**25, 2**28, 2**30 + 77, 2**31 - 200, 2**31 - 1):
        for n in (1, 300, 4096, 2**17, 2**24, 0x7FFFFF00):
            def most(tokens):
                return r // tokens + min(r, experts) + 1 if experts else -(-r // tokens)

            near = 4 * (128 + r) < 2**32  # the scales of a tile within 32 bits; else the 16-token kernels alone
            fits = [k for k in kernels if (near or k[0] == 16) and
                    (most(k[0]) * -(-n // k[1]) + 255) * THREADS[k] <= GRID_THREADS]
            rc = lib.mambo_fp8_block_plan(r, r, experts, n, 128, 128,
                                          _native.DTYPE_BF16 if bf16 else _native.DTYPE_F32, plan)
            if fits:
                assert rc == 0 and tuple(plan[:3]) in fits, (r, n)
                taken += 1
            else:
                refusal(rc, "too many rows and columns")
    assert taken > 10


def test_calls_that_no_grid_holds_are_refused():
    """Before anything is launched, with the message written for it."""
    from mambo_amd import _native
    lib, r = _native.lib(), 2**31 - 1
    refusal(lib.mambo_fp8_block_matmul(16, 16, 16, 1, r, r, 16, 16, 4096, 16, 16, 0, 4096, None), "too many rows and columns")
    refusal(lib.mambo_fp8_block_matmul_experts(16, 16, 16, 1, 1, 1, 16, r, 16, 4, 16, 16, 1, 16, 16, 1, 1, None),
            "too many rows and columns")
    refusal(lib.mambo_iq3s_fp8_matmul_experts(16, 256, 16, 8, 1, 16, r, 16, 4, 16, 7040, 64, 1, 16, 0, 64, None),
            "too many rows and columns")
    refusal(lib.mambo_fp8_block_pack(16, 1, 0x7FFFFF00, 16, 0, 16, 16, None), "too large for one call")
    refusal(lib.mambo_combine_experts(16, 1, 2**36, 4, 16, 16, 2, 2, 2**36, 16, 1, 2**36, None), "rows too long")


@pytest.mark.gpu
def test_iq3s_experts_of_more_rows_than_a_launch(gpu):
    """17 experts of 2^24 rows follow each other: as one tall weight they would not fit a launch."""
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
    raws = torch.empty((17, 1 << 24, 1, 110), dtype=torch.uint8, device=gpu)
    raws.view(-1)[:110 << 24].random_(0, 256)
    for e in range(1, 17):
        raws[e] = raws[0].roll(e, 0)
    got = prepare_iq3_s_experts(raws)
    assert (got.experts, got.n, got.blocks) == (17, 1 << 24, 1)
    for e in (0, 1, 15, 16):
        assert torch.equal(got.packed[e], prepare_iq3_s_experts(raws[e:e + 1]).packed[0]), e
    del raws, got
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------ the layer
@pytest.mark.gpu
@pytest.mark.parametrize("shared", [0, 256])
@pytest.mark.parametrize("down", ["fp8", "iq3s"])
def test_layer_of_no_tokens(gpu, down, shared):
    from mambo_amd.utils.expert_layer import random_layer
    layer = random_layer(512, 256, 4, 2, down=down, shared=shared)
    out = layer(torch.empty((0, 512), dtype=torch.bfloat16, device=gpu))
    assert out.shape == (0, 512) and out.dtype == torch.bfloat16 and out.device == gpu
    assert layer(torch.ones((1, 512), dtype=torch.bfloat16, device=gpu)).shape == (1, 512)


# ------------------------------------------------------------------------------ quantizer
def encode(x: np.ndarray) -> np.ndarray:
    """e4m3_encode_bruteforce for many values: between which two codes' middles a magnitude lies, the even
    code on a middle."""
    values = ref.VALUES[:127]
    middles = (values[1:] + values[:-1]) / 2.0  # exact
    a = np.abs(x.astype(np.float64))
    code = np.searchsorted(middles, a, side="left")  # a middle: the lower code
    on = code < 126
    on[on] = middles[code[on]] == a[on]
    code[on] += code[on] & 1
    return (code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def quantized(x: np.ndarray):
    """ref.quantize_block for many rows."""
    (m, k), g = x.shape, -(-x.shape[1] // 128)
    parts = np.pad(x, ((0, 0), (0, 128 * g - k))).reshape(m, g, 128)
    amax = np.maximum(np.abs(parts).max(2, keepdims=True), np.float32(448.0 * 2.0**-100))
    codes = encode((np.float32(0.875) * parts) / (amax * np.float32(2.0**-9)))
    return codes.reshape(m, -1)[:, :k], amax[..., 0] / np.float32(448.0)


def test_the_statement_for_many_rows_is_that_for_few():
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((40, 300)) * np.exp2(rng.integers(-12, 12, size=(40, 300)))).astype(np.float32)
    x[3], x[4] = 0.0, np.arange(300) * 448.0 / 299.0
    x[5, :32] = np.concatenate([[448.0], np.arange(1, 32) * 0.5])  # middles among them
    for a, b in zip(quantized(x), ref.quantize_block(x)):
        assert a.dtype == b.dtype and np.array_equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k", [(4096, 128), (4097, 144), (5001, 16), (1367, 4112), (131073, 16)])
def test_quantizer_of_many_rows(gpu, m, k, dtype, aligned):
    """Sizes that take two rows at a time: an odd last row, a last group that is not whole, more pairs than
    a grid's second dimension, rows that vectors do not reach."""
    from mambo_amd.kernels.fp8_block import launch_quantize_fp8_block
    assert m * -(-k // 2048) >= 4096  # rows times workgroups of a row
    rng = np.random.default_rng(m + k)
    x = rng.standard_normal((m, k)).astype(np.float32) * np.exp2(rng.integers(-20, 20, size=(m, 1))).astype(np.float32)
    x[rng.random(m) < 0.05] = 0.0
    x = torch.from_numpy(x).to(dtype)
    expected = quantized(x.float().numpy())
    rows = x.to(gpu)
    if not aligned:
        wide = torch.zeros((m, k + 5), dtype=dtype, device=gpu)
        wide[:, 1:k + 1] = rows
        rows = wide[:, 1:k + 1]
    codes, scales = launch_quantize_fp8_block(rows)
    assert np.array_equal(codes.cpu().numpy(), expected[0]) and np.array_equal(scales.cpu().numpy(), expected[1])
    buffer = torch.full((m + 1, k + 19), 9, dtype=torch.uint8, device=gpu)
    left = 16 if aligned else 3
    by_row = torch.full((m + 1, scales.shape[1] + 2), 7.0, device=gpu)
    launch_quantize_fp8_block(rows, out=(buffer[:m, left:left + k], by_row[:m, 1:-1]))
    assert torch.equal(buffer[:m, left:left + k], codes) and torch.equal(by_row[:m, 1:-1], scales)
    assert (buffer[m] == 9).all() and (buffer[:, :left] == 9).all() and (buffer[:, left + k:] == 9).all()
    assert (by_row[m] == 7).all() and (by_row[:, 0] == 7).all() and (by_row[:, -1] == 7).all()


# ------------------------------------------------------------------------------ many rows
@pytest.mark.gpu
@pytest.mark.parametrize("m,top_k,n", [(65536, 3, 5), (70001, 2, 520), (131073, 1, 64)])
def test_combine_of_many_tokens(gpu, m, top_k, n):
    """More tokens than a grid's second dimension; weights of powers of two and small integers: exact."""
    from mambo_amd.kernels.experts import launch_combine_experts
    gen = torch.Generator(device=gpu).manual_seed(m)
    y = torch.randint(-64, 65, (m * top_k, n), generator=gen, device=gpu).to(torch.bfloat16)
    slots = torch.randperm(m * top_k, generator=gen, device=gpu).to(torch.int32).view(m, top_k)
    slots = slots.masked_fill(torch.rand((m, top_k), generator=gen, device=gpu) < 0.2, -1)
    weights = torch.exp2(torch.randint(-2, 3, (m, top_k), generator=gen, device=gpu).float())
    expected = torch.zeros((m, n), device=gpu)
    for j in range(top_k):
        some = slots[:, j] >= 0
        expected[some] += weights[some, j, None] * y[slots[some, j].long()].float()
    assert torch.equal(launch_combine_experts(y, slots, weights, out_dtype=torch.float32), expected)
    assert torch.equal(launch_combine_experts(y, slots, weights), expected.to(torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("weight", ["fp8", "iq3s"])
def test_products_of_many_rows(gpu, weight, out_dtype):
    """4.2 million rows of 700 tokens, more tiles of 64 than a grid's second dimension: each is the product of its token
    with its expert, as those 700 rows give it alone."""
    from mambo_amd.kernels.experts import launch_fp8_block_matmul_experts, launch_iq3_s_fp8_matmul_experts
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
    rng = np.random.default_rng(3)
    r, m, n, k, experts = 64 * 65535 + 77, 700, 70, 256, 3
    offsets = torch.tensor([0, 1, r // 2, r - 1000], dtype=torch.int32, device=gpu)
    rows = torch.from_numpy(rng.integers(0, m, size=r).astype(np.int32)).to(gpu)
    if weight == "fp8":  # integers: the same in any order
        call = launch_fp8_block_matmul_experts
        values, wv = (torch.from_numpy(ref.integer_codes(rng, s)).to(gpu) for s in ((m, k), (experts, n, k)))
        scales = torch.ones((m, 2), device=gpu)
        w = prepare_fp8_block_weight(wv, torch.ones((experts, 1, 2), device=gpu))
        tolerance = 0.0
    else:  # float32 sums in another order: as test_gpu_experts.test_iq3s_experts
        call = launch_iq3_s_fp8_matmul_experts
        raw = rng.integers(0, 256, size=(experts, n, 1, 110), dtype=np.uint8)
        raw[..., :2] = np.array([0.01], dtype=np.float16).view(np.uint8)
        w = prepare_iq3_s_experts(torch.from_numpy(raw).to(gpu))
        values, scales = launch_quantize_fp8(torch.randn((m, k), device=gpu))
        tolerance = 1e-4 if out_dtype == torch.float32 else 2.0**-8
    out = call(values, scales, w, offsets, rows=rows, out_dtype=out_dtype)
    assert not bool(out[r - 1000:].any())
    starts = offsets.tolist()
    for e in range(experts):
        alone = torch.zeros(experts + 1, dtype=torch.int32, device=gpu)
        alone[e + 1:] = m
        expected = call(values, scales, w, alone, out_dtype=out_dtype).float()
        a, b = starts[e], starts[e + 1]
        off = (out[a:b].float() - expected[rows[a:b].long()]).norm(dim=1)
        assert bool((off <= tolerance * expected.norm(dim=1)[rows[a:b].long()]).all()), e
