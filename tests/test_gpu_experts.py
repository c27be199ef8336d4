"""The operators of a layer of experts on the GPU: the router's plan exactly, the grouped products
against a product per expert, the join against 64 bits, all of it together in a HIP graph."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import expert_reference as ref
from conftest import make_synthetic_iq3_s
from oracle import oracle

pytestmark = pytest.mark.gpu


def ops():
    from mambo_amd.kernels import experts
    return experts


def device(gpu, *arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).to(gpu) for a in arrays]


# ------------------------------------------------------------------------------ router
def check_plan(got, logits, top_k, renormalize):
    ids, weights = ref.route(logits.double().cpu().numpy(), top_k, renormalize)
    offsets, rows, slots = ref.plan(ids, logits.shape[1])
    assert np.array_equal(got.ids.cpu().numpy(), ids)
    for name, a in (("offsets", offsets), ("rows", rows), ("slots", slots)):
        t = getattr(got, name)
        assert t.dtype == torch.int32 and np.array_equal(t.cpu().numpy(), a), name
    # exp and a sum of up to E terms in float32, each a few units off
    assert np.abs(got.weights.double().cpu().numpy() - weights).max(initial=0.0) <= (logits.shape[1] + 8) * 2.0**-23


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("m,experts,top_k", [(1, 1, 1), (1, 8, 2), (16, 64, 8), (5, 65, 3), (33, 128, 1), (100, 130, 7),
                                             (70, 256, 8), (9, 300, 10), (12, 512, 6), (3, 1000, 64), (700, 6, 6)])
def test_route(gpu, m, experts, top_k, renormalize):
    rng = np.random.default_rng(m + experts)
    logits = torch.from_numpy(rng.standard_normal((m, experts)).astype(np.float32) * 3).to(gpu)
    check_plan(ops().launch_route_experts(logits, top_k, renormalize=renormalize), logits, top_k, renormalize)
    half = logits.to(torch.bfloat16)  # ties
    check_plan(ops().launch_route_experts(half, top_k, renormalize=renormalize), half, top_k, renormalize)


@pytest.mark.parametrize("renormalize", [True, False])
def test_route_masks_ties_and_extremes(gpu, renormalize):
    inf, nan = float("inf"), float("nan")
    rows = [[0.0] * 70, [-inf] * 70, [nan] * 70, [inf] * 2 + [1.0] * 68, [-3.4e38] * 70, [0.0, -0.0] * 35,
            [-inf] * 69 + [2.0], [nan, 5.0] + [-inf] * 68, [3.4e38, -3.4e38] * 35, [1e-45, -1e-45, 0.0] + [-1.0] * 67,
            [float(i % 7) for i in range(70)], [-inf, nan, inf, 1.0, 3.0] * 14]
    logits = torch.tensor(rows, dtype=torch.float32, device=gpu)
    for top_k in (1, 3, 64):
        check_plan(ops().launch_route_experts(logits, top_k, renormalize=renormalize), logits, top_k, renormalize)
    tiny = logits[:, :3].contiguous()
    check_plan(ops().launch_route_experts(tiny, 3, renormalize=renormalize), tiny, 3, renormalize)


def test_route_no_tokens_and_strides(gpu):
    plan = ops().launch_route_experts(torch.empty((0, 9), device=gpu), 2)
    assert plan.ids.shape == (0, 2) and plan.rows.shape == (0,) and plan.offsets.tolist() == [0] * 10
    rng = np.random.default_rng(1)
    wide = torch.from_numpy(rng.standard_normal((40, 50)).astype(np.float32)).to(gpu)
    for logits in (wide[:, 3:20], wide[::2, 1:30], wide.t()[:40, :7], wide[:1].expand(6, 50)):
        check_plan(ops().launch_route_experts(logits, 4), logits, 4, True)


# ------------------------------------------------------------------------------ products
# (rows, experts, rows of no expert, N, K)
GROUPED = [(1, 1, 0, 33, 144), (1, 7, 0, 64, 128), (16, 64, 0, 96, 256), (37, 3, 5, 130, 272), (40, 3, 0, 64, 1040),
           (128, 64, 3, 257, 400), (150, 2, 0, 160, 128), (300, 5, 40, 300, 384), (200, 130, 1, 40, 144),
           (700, 3, 10, 192, 528), (64, 65, 64, 32, 128), (900, 4, 0, 257, 272), (520, 1, 20, 130, 256)]


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("r,experts,unrouted,n,k", GROUPED)
def test_fp8_experts(gpu, r, experts, unrouted, n, k, gather, out_dtype):
    """Integer sums, exact in any order (test_gpu_fp8_block); rows of no expert are zeros."""
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    rng = np.random.default_rng(r + experts + n + k)
    g, m = -(-k // 128), max(1, r // 3) if gather else r
    xv, wv = ref.integer_codes(rng, (m, k)), ref.integer_codes(rng, (experts, n, k))
    xs = np.exp2(rng.integers(-1, 2, size=(m, g))).astype(np.float32)
    ws = np.exp2(rng.integers(-1, 2, size=(experts, -(-n // 128), g))).astype(np.float32)
    offsets = ref.some_offsets(rng, r, experts, unrouted)
    rows = rng.integers(0, m, size=r).astype(np.int32) if gather else np.arange(r, dtype=np.int32)
    rows[offsets[-1]:] = -1
    expected = np.zeros((r, n))
    for e in range(experts):
        at = rows[offsets[e]:offsets[e + 1]]
        if at.size:
            expected[offsets[e]:offsets[e + 1]] = ref.product(xv[at], xs[at], wv[e], ws[e])[0]
    xv, xs, wv, ws, offsets, rows = device(gpu, xv, xs, wv, ws, offsets, rows)
    w = prepare_fp8_block_weight(wv, ws)
    out = ops().launch_fp8_block_matmul_experts(xv, xs, w, offsets, rows=rows if gather else None, out_dtype=out_dtype)
    assert torch.equal(out.cpu(), torch.from_numpy(expected).float().to(out_dtype))


@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("r,experts,unrouted,n,k", [(1, 1, 0, 33, 256), (1, 9, 0, 16, 512), (16, 64, 0, 48, 256),
                                                    (37, 3, 5, 130, 768), (128, 64, 3, 100, 256), (300, 5, 40, 300, 1280),
                                                    (200, 130, 1, 40, 256), (700, 3, 10, 192, 2304), (64, 65, 64, 32, 256),
                                                    (900, 4, 0, 257, 1024)])
def test_iq3s_experts(gpu, r, experts, unrouted, n, k, gather):
    """Against the oracle's product per expert: its sums and these are float32 in different orders
    over K terms, each off by K units of the last place of the sum of magnitudes at most, which a
    relative 2-norm of 1e-4 holds (as the projections' tests do with 1e-3)."""
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
    rng = np.random.default_rng(r + experts + n + k)
    m = max(1, r // 3) if gather else r
    raws = np.stack([make_synthetic_iq3_s(n, k, seed=100 * r + e) for e in range(experts)])
    x = rng.standard_normal((m, k)).astype(np.float32)
    offsets = ref.some_offsets(rng, r, experts, unrouted)
    rows = rng.integers(0, m, size=r).astype(np.int32) if gather else np.arange(r, dtype=np.int32)
    rows[offsets[-1]:] = -1
    eq, es = oracle.quantize_mxfp8(x)
    expected = np.zeros((r, n))
    for e in range(experts):
        at = rows[offsets[e]:offsets[e + 1]]
        if at.size:
            expected[offsets[e]:offsets[e + 1]] = oracle.iq3s_fp8_matmul(eq[at], es[at], raws[e])
    x, raws, offsets, rows = device(gpu, x, raws, offsets, rows)
    w = prepare_iq3_s_experts(raws)
    values, scales = launch_quantize_fp8(x)
    for dtype, tolerance in ((torch.float32, 1e-4), (torch.bfloat16, 2.0**-8)):
        out = ops().launch_iq3_s_fp8_matmul_experts(values, scales, w, offsets, rows=rows if gather else None,
                                                    out_dtype=dtype).double().cpu().numpy()
        taken = int(offsets[-1])
        assert not out[taken:].any()
        for i in range(taken):  # row by row, so that one wrong row shows
            assert np.linalg.norm(out[i] - expected[i]) <= tolerance * np.linalg.norm(expected[i]), i


@pytest.mark.parametrize("n,k", [(32, 256), (33, 512), (16, 768), (130, 256)])
def test_iq3s_experts_of_any_strides(gpu, n, k):
    """Packed alike from contiguous weights, rows apart, experts apart, and one weight at a time."""
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
    raws = device(gpu, np.stack([make_synthetic_iq3_s(n, k, seed=50 + e) for e in range(5)]))[0]
    expected = torch.cat([prepare_iq3_s_experts(raws[e:e + 1]).packed for e in range(5)])
    apart = torch.zeros((5, n + 3, k // 256, 110), dtype=torch.uint8, device=gpu)
    apart[:, :n] = raws
    wide = torch.zeros((5, 2 * n, k // 256, 112), dtype=torch.uint8, device=gpu)
    wide[:, ::2, :, 1:111] = raws
    for source in (raws, apart[:, :n], wide[:, ::2, :, 1:111], raws.flip(0).flip(0), raws.transpose(0, 1).contiguous().transpose(0, 1)):
        got = prepare_iq3_s_experts(source)
        assert (got.experts, got.n, got.blocks) == (5, n, k // 256) and torch.equal(got.packed, expected)


def test_experts_equal_the_projection(gpu):
    """One expert is the dense product (bit for bit where the rows take the same kernel)."""
    from mambo_amd.kernels.fp8_block import launch_fp8_block_matmul
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    rng = np.random.default_rng(4)
    for m in (1, 16, 60, 300):
        xv, xs, wv, ws = device(gpu, ref.random_codes(rng, (m, 640)), rng.random((m, 5)).astype(np.float32),
                                ref.random_codes(rng, (200, 640)), rng.random((2, 5)).astype(np.float32))
        dense = launch_fp8_block_matmul(xv, xs, prepare_fp8_block_weight(wv, ws))
        one = ops().launch_fp8_block_matmul_experts(xv, xs, prepare_fp8_block_weight(wv[None], ws[None]),
                                                    torch.tensor([0, m], dtype=torch.int32, device=gpu))
        assert torch.equal(dense, one), m


def test_plan_of_other_values_stays_inside(gpu):
    """Offsets that fall or leave [0, R] and rows outside [0, M) read and write nothing outside the
    tensors: the kernels hold every value within its range."""
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    rng = np.random.default_rng(8)
    wv, ws = device(gpu, ref.integer_codes(rng, (3, 70, 144)), np.ones((3, 1, 2), dtype=np.float32))
    w = prepare_fp8_block_weight(wv, ws)
    xv, xs = device(gpu, ref.integer_codes(rng, (20, 144)), np.ones((20, 2), dtype=np.float32))
    for offsets in ([0, 50, 7, 90], [-5, 3, 2, 1], [0, 2**31 - 1, -2**31, 40]):
        rows = torch.tensor(rng.integers(-2**31, 2**31, size=40), dtype=torch.int32, device=gpu)
        buf = torch.full((44, 70), 77.0, device=gpu)
        ops().launch_fp8_block_matmul_experts(xv, xs, w, torch.tensor(offsets, dtype=torch.int32, device=gpu), rows=rows,
                                              out=buf[2:42])
        assert (buf[:2] == 77).all() and (buf[42:] == 77).all() and torch.isfinite(buf).all()


def test_nan_of_other_experts_stays_there(gpu):
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    rng = np.random.default_rng(9)
    for counts in ((3, 0, 20), (70, 1, 150)):
        r = sum(counts)
        wv = ref.integer_codes(rng, (3, 40, 400))
        wv[1] = 0x7F
        xv = ref.integer_codes(rng, (r, 400))
        offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        xv[offsets[1]:offsets[2]] = 0x7F
        xv, wv, offsets_t = device(gpu, xv, wv, offsets)
        w = prepare_fp8_block_weight(wv, torch.ones((3, 1, 4), device=gpu))
        out = ops().launch_fp8_block_matmul_experts(xv, torch.ones((r, 4), device=gpu), w, offsets_t).cpu()
        nan = torch.isnan(out).all(1)
        assert nan[offsets[1]:offsets[2]].all() and torch.isfinite(out[~nan]).all() and int(nan.sum()) == counts[1]


# ------------------------------------------------------------------------------ join
@pytest.mark.parametrize("y_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, None])
@pytest.mark.parametrize("m,top_k,n", [(1, 1, 1), (1, 8, 4096), (5, 2, 33), (40, 3, 130), (70, 64, 16), (300, 8, 1028)])
def test_combine(gpu, m, top_k, n, y_dtype, out_dtype):
    rng = np.random.default_rng(m + top_k + n)
    r = m * top_k
    y = torch.from_numpy(rng.standard_normal((r, n)).astype(np.float32)).to(y_dtype)
    slots = rng.permutation(r).reshape(m, top_k).astype(np.int32)
    slots[rng.random((m, top_k)) < 0.2] = -1
    slots[m // 2] = -1
    weights = rng.standard_normal((m, top_k)).astype(np.float32)
    terms = np.where(slots[..., None] < 0, 0.0, weights[..., None].astype(np.float64) * y.double().numpy()[slots])
    expected, magnitudes = terms.sum(1), np.abs(terms).sum(1)
    s, w = device(gpu, slots, weights)
    out = ops().launch_combine_experts(y.to(gpu), s, w, out_dtype=out_dtype)
    assert out.dtype == (out_dtype or y_dtype)
    off = np.abs(out.double().cpu().numpy() - expected)
    assert (off <= ref.bound(magnitudes, top_k, expected, out.dtype)).all()
    assert not out[m // 2].any()


def test_combine_leaves_masked_rows_unread(gpu):
    """A row that no slot names may hold anything; slots outside the rows add nothing."""
    y = torch.full((4, 70), float("nan"), device=gpu)
    y[1] = 2.0
    slots = torch.tensor([[1, -1, 4], [-1, 2**31 - 1, -2**31]], dtype=torch.int32, device=gpu)
    out = ops().launch_combine_experts(y, slots, torch.full((2, 3), 0.5, device=gpu))
    assert (out[0] == 1.0).all() and (out[1] == 0.0).all()
    assert ops().launch_combine_experts(y, slots[:0], torch.empty((0, 3), device=gpu)).shape == (0, 70)


def test_combine_strides(gpu):
    rng = np.random.default_rng(6)
    wide = torch.from_numpy(rng.standard_normal((12, 300)).astype(np.float32)).to(gpu)
    slots = torch.tensor([[0, 5], [3, 2]], dtype=torch.int32, device=gpu)
    weights = torch.tensor([[1.0, 2.0], [4.0, 8.0]], device=gpu)
    for y in (wide[:, 4:204], wide[:, 1:200], wide[::2, 8:40], wide.t()[:9, :7]):
        expected = torch.stack([y[0] + 2 * y[5], 4 * y[3] + 8 * y[2]])
        buf = torch.full((2, y.shape[1] + 5), 77.0, device=gpu)
        ops().launch_combine_experts(y, slots, weights, out=buf[:, 2:2 + y.shape[1]])
        assert torch.allclose(buf[:, 2:2 + y.shape[1]], expected, rtol=1e-6, atol=1e-6)
        assert (buf[:, :2] == 77).all() and (buf[:, 2 + y.shape[1]:] == 77).all()


# ------------------------------------------------------------------------------ together
def test_layer_in_a_graph(gpu):
    """Route, quantize, both products and the join captured once; each replay follows the inputs."""
    from mambo_amd.kernels.fp8_block import launch_quantize_fp8_block
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
    ex = ops()
    rng = np.random.default_rng(12)
    codes, scales = device(gpu, ref.random_codes(rng, (5, 256, 320)), rng.random((5, 2, 3)).astype(np.float32) * 1e-3)
    up = prepare_fp8_block_weight(codes, scales)
    down = prepare_iq3_s_experts(device(gpu, np.stack([make_synthetic_iq3_s(96, 256, seed=e) for e in range(5)]))[0])
    x, logits = torch.zeros((70, 320), device=gpu), torch.zeros((70, 5), device=gpu)

    def layer():
        plan = ex.launch_route_experts(logits, 2)
        h = ex.launch_fp8_block_matmul_experts(*launch_quantize_fp8_block(x), up, plan.offsets, rows=plan.rows)
        y = ex.launch_iq3_s_fp8_matmul_experts(*launch_quantize_fp8(h), down, plan.offsets)
        return ex.launch_combine_experts(y, plan.slots, plan.weights)

    layer()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = layer()
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(4):
        gen = torch.Generator(device=gpu).manual_seed(seed)
        x.copy_(torch.randn(x.shape, generator=gen, device=gpu))
        logits.copy_(torch.randn(logits.shape, generator=gen, device=gpu))
        logits[3] = float("-inf")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer()) and not out[3].any() and bool(out.any())


def test_refusals(gpu):
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
    ex = ops()
    logits = torch.zeros((3, 4), device=gpu)
    w = prepare_fp8_block_weight(torch.zeros((4, 8, 32), dtype=torch.uint8, device=gpu), torch.ones((4, 1, 1), device=gpu))
    raw = torch.zeros((4, 8, 1, 110), dtype=torch.uint8, device=gpu)
    iq = prepare_iq3_s_experts(raw)
    xv, xs = torch.zeros((3, 32), dtype=torch.uint8, device=gpu), torch.ones((3, 1), device=gpu)
    mv, ms = torch.zeros((3, 256), dtype=torch.uint8, device=gpu), torch.zeros((3, 8), dtype=torch.uint8, device=gpu)
    offsets = torch.tensor([0, 1, 1, 2, 3], dtype=torch.int32, device=gpu)
    rows = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
    slots, weights = torch.zeros((3, 2), dtype=torch.int32, device=gpu), torch.zeros((3, 2), device=gpu)
    y = torch.zeros((6, 8), device=gpu)
    value = [
        lambda: ex.launch_route_experts(logits, 0),
        lambda: ex.launch_route_experts(logits, 5),
        lambda: ex.launch_route_experts(logits.half(), 2),
        lambda: ex.launch_route_experts(logits.cpu(), 2),
        lambda: ex.launch_route_experts(logits[0], 2),
        lambda: ex.launch_route_experts(torch.zeros((1, 1025), device=gpu), 2),
        lambda: ex.launch_fp8_block_matmul_experts(xv, xs, w, offsets[:4]),
        lambda: ex.launch_fp8_block_matmul_experts(xv, xs, w, offsets.long()),
        lambda: ex.launch_fp8_block_matmul_experts(xv, xs, w, offsets.cpu()),
        lambda: ex.launch_fp8_block_matmul_experts(xv, xs, w, offsets, rows=rows.long()),
        lambda: ex.launch_fp8_block_matmul_experts(xv, xs, w, offsets, rows=rows[:, None]),
        lambda: ex.launch_fp8_block_matmul_experts(xv[:0], xs[:0], w, offsets, rows=rows),
        lambda: ex.launch_fp8_block_matmul_experts(xv, xs, w, offsets, rows=rows, out=torch.empty((2, 8), device=gpu)),
        lambda: ex.launch_iq3_s_fp8_matmul_experts(mv[:, :128], ms, iq, offsets),
        lambda: ex.launch_iq3_s_fp8_matmul_experts(mv, ms.int(), iq, offsets),
        lambda: ex.launch_iq3_s_fp8_matmul_experts(mv, ms, iq, offsets, out_dtype=torch.float16),
        lambda: prepare_iq3_s_experts(raw[0]),
        lambda: prepare_iq3_s_experts(raw.cpu()),
        lambda: ex.launch_combine_experts(y.half(), slots, weights),
        lambda: ex.launch_combine_experts(y, slots.long(), weights),
        lambda: ex.launch_combine_experts(y, slots, weights[:2]),
        lambda: ex.launch_combine_experts(y, slots, weights.double()),
        lambda: ex.launch_combine_experts(y, slots, weights, out=torch.empty((3, 9), device=gpu)),
    ]
    for call in value:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ex.launch_fp8_block_matmul_experts(xv, xs, iq, offsets)
    with pytest.raises(TypeError):
        ex.launch_iq3_s_fp8_matmul_experts(mv, ms, w, offsets)
