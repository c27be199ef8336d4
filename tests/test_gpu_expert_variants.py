"""Every kernel of the 8-bit block products, dense and grouped by expert, both orders of the rows'
scales, and operands whose offsets do not fit 32 bits."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import expert_reference as ref
from conftest import make_synthetic_iq3_s

F32, BF16 = torch.float32, torch.bfloat16

# (dtype, tokens, experts (0: dense), N, K)
VARIANTS = [
    (F32, 1, 0, 33, 4112), (F32, 1500, 0, 33, 2064), (F32, 2050, 0, 33, 2064), (F32, 2050, 0, 33, 4112),
    (F32, 3001, 0, 130, 2064), (F32, 67, 0, 8200, 1040), (F32, 203, 0, 8200, 528), (F32, 203, 0, 8200, 1040),
    (F32, 1, 2, 33, 4112), (F32, 1500, 2, 33, 2064), (F32, 2050, 2, 33, 2064), (F32, 2050, 2, 33, 4112),
    (F32, 3001, 2, 130, 2064), (F32, 33, 2, 8200, 1040), (F32, 67, 4, 8200, 528), (F32, 67, 4, 8200, 1040),
    (BF16, 1, 0, 33, 4112), (BF16, 1500, 0, 33, 2064), (BF16, 2050, 0, 33, 2064), (BF16, 2050, 0, 33, 4112),
    (BF16, 17, 0, 8200, 2064), (BF16, 1030, 0, 650, 1040), (BF16, 203, 0, 8200, 528),
    (BF16, 203, 0, 8200, 1552), (BF16, 523, 0, 15000, 528), (BF16, 1, 2, 33, 4112), (BF16, 1500, 2, 33, 2064),
    (BF16, 2050, 2, 33, 2064), (BF16, 2050, 2, 33, 4112), (BF16, 1500, 40, 130, 2064), (BF16, 5, 2, 8200, 1040),
    (BF16, 17, 4, 8200, 528), (BF16, 131, 2, 8200, 1040), (BF16, 131, 4, 15000, 1040), (F32, 1, 0, 8200, 2064),
    (F32, 1500, 0, 650, 1040), (F32, 3001, 0, 650, 1552), (F32, 523, 40, 130, 2064), (F32, 131, 2, 8200, 528),
    (F32, 67, 2, 8200, 1040), (F32, 17, 4, 15000, 1040), (BF16, 1, 0, 8200, 2064), (BF16, 1030, 0, 33, 2064),
    (BF16, 3001, 0, 130, 2064), (BF16, 67, 0, 8200, 1040), (BF16, 203, 0, 8200, 2064),
    (BF16, 1030, 0, 8200, 528), (BF16, 17, 4, 1100, 2064), (BF16, 96, 40, 1100, 2064),
    (BF16, 1030, 2, 33, 2064), (BF16, 1030, 40, 300, 2064), (BF16, 5, 2, 15000, 528), (BF16, 17, 4, 8200, 1552),
    (BF16, 401, 4, 15000, 656), (BF16, 6000, 2, 4100, 272), (BF16, 801, 2, 1100, 2064),
    (F32, 801, 2, 1100, 2064), (F32, 8200, 2, 1300, 272),
]
IDS = [f"{str(d)[6:]}-{m}x{e}x{n}x{k}" for d, m, e, n, k in VARIANTS]


def plan(m, r, experts, n, k, dtype, ldxv=None):
    from mambo_amd import _native
    out = (ctypes.c_int32 * 5)()
    _native.check(_native.lib().mambo_fp8_block_plan(m, r, experts, n, k, ldxv or k,
                                                     _native.DTYPE_BF16 if dtype == BF16 else _native.DTYPE_F32, out))
    return tuple(out)


def test_each_kernel_is_tested():
    """Every kernel of a dtype, dense and by expert, and every order of the workgroups: in turn, an eighth
    to each XCD (one column at a time, or four), 32 at a time."""
    for dtype, kernels in ((F32, 8), (BF16, 9)):
        for grouped in (False, True):
            plans = {plan(m, m, e, n, k, d) for d, m, e, n, k in VARIANTS if d == dtype and (e > 0) == grouped}
            assert len({p[:3] for p in plans}) == kernels, (dtype, grouped)
            assert any(p[4] not in (1, 32) and p[3] == 1 for p in plans)
            if grouped:
                assert {1, 32} <= {p[4] for p in plans}
            else:
                assert any(p[3] == 4 for p in plans)


def test_far_rows_take_the_streaming_kernels():
    for m, experts, ld in ((3, 0, 1 << 25), (300, 0, 1 << 25), (1 << 20, 4, 4096), (600, 4, 1 << 25)):
        assert plan(m, 500 if experts else m, experts, 8200, 1040, BF16, ld)[:3] in ((16, 16, 8), (16, 32, 4), (16, 64, 4))


def test_plan_refuses_what_the_call_refuses():
    from mambo_amd import _native
    lib, tile = _native.lib(), (ctypes.c_int32 * 5)()
    good = dict(m=5, r=5, experts=2, n=64, k=128, ldxv=128, out_dtype=_native.DTYPE_F32)
    assert lib.mambo_fp8_block_plan(*good.values(), tile) == 0
    for bad in (dict(k=120), dict(n=0), dict(out_dtype=7), dict(experts=1025), dict(experts=-1), dict(r=0), dict(r=-1),
                dict(m=0), dict(ldxv=112)):
        assert lib.mambo_fp8_block_plan(*{**good, **bad}.values(), tile) == _native.MAMBO_ERR_VALUE, bad
    assert lib.mambo_fp8_block_plan(*good.values(), None) == _native.MAMBO_ERR_VALUE


# ------------------------------------------------------------------------------ on the GPU
def values_of(codes: torch.Tensor) -> torch.Tensor:
    return torch.from_numpy(ref.VALUES).to(codes.device)[codes.long()]


def exact(xv, xs, wv, ws):
    """Sums and sums of magnitudes of codes [M,K] and [N,K] on the GPU, float64."""
    k = xv.shape[1]
    x = values_of(xv) * xs.double().repeat_interleave(128, 1)[:, :k]
    w = values_of(wv) * ws.double().repeat_interleave(128, 0)[:wv.shape[0]].repeat_interleave(128, 1)[:, :k]
    return x @ w.t().contiguous(), x.abs() @ w.abs().t().contiguous()


def grouped(xv, xs, wv, ws, offsets):
    parts = [exact(xv[a:b], xs[a:b], wv[e], ws[e]) for e, (a, b) in enumerate(zip(offsets[:-1], offsets[1:]))]
    return tuple(torch.cat(p) for p in zip(*parts))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,m,experts,n,k", VARIANTS, ids=IDS)
def test_integers_add_up_exactly(gpu, dtype, m, experts, n, k):
    """Codes of small integers and scales of powers of two: every order of the sum gives the same
    float32. Scales group by group and row by row give the same."""
    from mambo_amd.kernels.experts import launch_fp8_block_matmul_experts
    from mambo_amd.kernels.fp8_block import launch_fp8_block_matmul
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    gen = torch.Generator(device=gpu).manual_seed(m + n + k)
    integers = torch.from_numpy(ref.e4m3_encode_bruteforce(np.arange(-8.0, 9.0))).to(gpu)
    g, e = -(-k // 128), max(experts, 1)

    def rand(*shape, scale=False):
        if scale:
            return torch.exp2(torch.randint(-1, 2, shape, generator=gen, device=gpu).float())
        return integers[torch.randint(0, 17, shape, generator=gen, device=gpu)]

    xv, xs, wv, ws = rand(m, k), rand(m, g, scale=True), rand(e, n, k), rand(e, -(-n // 128), g, scale=True)
    rng = np.random.default_rng(m)
    offsets = ref.some_offsets(rng, m, experts) if experts else np.array([0, m], dtype=np.int32)
    offsets[-1] = m
    expected = grouped(xv, xs, wv, ws, offsets.tolist())[0]
    assert expected.abs().max() < 2**22  # a multiple of 1/4 in 24 bits
    expected = expected.float().to(dtype)
    for scales in (xs, xs.t().contiguous().t(), torch.nn.functional.pad(xs, (0, 3))[:, :g]):
        if experts:
            w = prepare_fp8_block_weight(wv, ws)
            order = torch.randperm(m, generator=gen, device=gpu)
            back = torch.argsort(order).to(torch.int32)  # row i of the product is row back[i] of the shuffled ones
            offs = torch.from_numpy(offsets).to(gpu)
            out = launch_fp8_block_matmul_experts(xv, scales, w, offs, out_dtype=dtype)
            moved = scales[order] if scales.stride(1) == 1 else scales.t()[:, order].contiguous().t()
            again = launch_fp8_block_matmul_experts(xv[order], moved, w, offs, rows=back, out_dtype=dtype)
            assert torch.equal(again, out)
        else:
            out = launch_fp8_block_matmul(xv, scales, prepare_fp8_block_weight(wv[0], ws[0]), out_dtype=dtype)
        assert torch.equal(out, expected)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,m,experts,n,k", [v for v in VARIANTS if v[0] == F32 and not v[2]])
def test_real_values_within_the_bound_of_float32_sums(gpu, dtype, m, experts, n, k):
    from mambo_amd.kernels.fp8_block import launch_fp8_block_matmul
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    gen = torch.Generator(device=gpu).manual_seed(m + n + k)
    g = -(-k // 128)
    xv, wv = (torch.randint(0, 256, s, generator=gen, device=gpu, dtype=torch.uint8) for s in ((m, k), (n, k)))
    xv, wv = (torch.where((c & 127) == 127, 0, c) for c in (xv, wv))
    xs, ws = (torch.rand(s, generator=gen, device=gpu) + 0.01 for s in ((m, g), (-(-n // 128), g)))
    expected, magnitudes = exact(xv, xs, wv, ws)
    out = launch_fp8_block_matmul(xv, xs, prepare_fp8_block_weight(wv, ws))
    off = (out.double() - expected).abs().cpu().numpy()
    assert (off <= ref.bound(magnitudes.cpu().numpy(), k, expected.cpu().numpy(), dtype)).all()


# ------------------------------------------------------------------------------ offsets past 32 bits
@pytest.mark.gpu
def test_rows_far_apart(gpu):
    """Rows 2^25 elements apart, then rows gathered from more than 4 GiB; the outputs far apart too."""
    from mambo_amd.kernels.experts import launch_fp8_block_matmul_experts, launch_iq3_s_fp8_matmul_experts
    from mambo_amd.kernels.fp8_block import launch_fp8_block_matmul, launch_quantize_fp8_block
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
    rng = np.random.default_rng(1)
    n, k, m = 200, 1024, 140  # 140 rows of 2^25 bytes: 4.7 GB
    x = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).to(gpu)
    values, scales = launch_quantize_fp8_block(x)
    w = prepare_fp8_block_weight(torch.from_numpy(ref.random_codes(rng, (3, n, k))).to(gpu),
                                 torch.rand((3, 2, 8), device=gpu))
    one = prepare_fp8_block_weight(torch.from_numpy(ref.random_codes(rng, (n, k))).to(gpu), torch.rand((2, 8), device=gpu))
    far = torch.empty((m, 1 << 25), dtype=torch.uint8, device=gpu)[:, :k]
    far.copy_(values)
    outs = torch.empty((m, 1 << 24), device=gpu)[:, :n]  # 64 MiB apart: 9.4 GB
    launch_fp8_block_matmul(far, scales, one, out=outs)
    close = launch_fp8_block_matmul(values, scales, one)
    # other kernels, other orders of the sum: each within k units of the last place
    assert torch.allclose(outs, close, rtol=0.0, atol=2 * k * 2.0**-23 * float(close.abs().max()) * 8)
    offsets = torch.tensor([0, 50, 51, m - 3], dtype=torch.int32, device=gpu)
    rows = torch.from_numpy(rng.permutation(m).astype(np.int32)).to(gpu)
    a = launch_fp8_block_matmul_experts(far, scales, w, offsets, rows=rows, out=outs)
    b = launch_fp8_block_matmul_experts(values, scales, w, offsets, rows=rows)
    assert torch.allclose(a, b, rtol=0.0, atol=2 * k * 2.0**-23 * float(b.abs().max()) * 8) and not a[m - 3:].any()
    # the quantizers' rows, read and written far apart
    wide = torch.empty((m, 1 << 24), device=gpu)[:, :k]
    wide.copy_(x)
    v, s = launch_quantize_fp8_block(wide, out=(far, torch.empty((m, 8), device=gpu)))
    assert torch.equal(v, values) and torch.equal(s, scales)
    raws = torch.from_numpy(np.stack([make_synthetic_iq3_s(n, k, seed=e) for e in range(3)])).to(gpu)
    iq = prepare_iq3_s_experts(raws)
    values, scales = launch_quantize_fp8(x)
    far.copy_(values)
    a = launch_iq3_s_fp8_matmul_experts(far, scales, iq, offsets, rows=rows, out=outs)
    b = launch_iq3_s_fp8_matmul_experts(values, scales, iq, offsets, rows=rows)
    assert torch.allclose(a, b, rtol=0.0, atol=2 * k * 2.0**-23 * float(b.abs().max()) * 8) and not a[m - 3:].any()


@pytest.mark.gpu
def test_many_gathered_rows(gpu):
    """Rows past 4 GiB of a buffer of many (2^20 + 9 rows of 4096)."""
    from mambo_amd.kernels.experts import launch_fp8_block_matmul_experts
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    rng = np.random.default_rng(2)
    m, n, k, r = (1 << 20) + 9, 40, 4096, 60
    xv = torch.zeros((m, k), dtype=torch.uint8, device=gpu)
    xs = torch.ones((k // 128, m), device=gpu).t()
    rows = torch.cat([torch.arange(r // 2), torch.arange(m - r // 2, m)]).to(torch.int32).to(gpu)
    part = torch.from_numpy(ref.integer_codes(rng, (r, k))).to(gpu)
    xv[rows.long()] = part
    wv = torch.from_numpy(ref.integer_codes(rng, (2, n, k))).to(gpu)
    ws = torch.ones((2, 1, k // 128), device=gpu)
    out = launch_fp8_block_matmul_experts(xv, xs, prepare_fp8_block_weight(wv, ws),
                                          torch.tensor([0, 11, r], dtype=torch.int32, device=gpu), rows=rows)
    assert torch.equal(out.double(), grouped(part, torch.ones((r, k // 128), device=gpu), wv, ws, [0, 11, r])[0])


@pytest.mark.gpu
def test_weights_past_32_bits(gpu):
    """40 experts of 8192 x 14336, 4.7 GB: rows of the last, by the streaming and the tile kernels."""
    from mambo_amd.kernels.experts import launch_fp8_block_matmul_experts
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    experts, n, k = 40, 8192, 14336
    gen = torch.Generator(device=gpu).manual_seed(5)
    integers = torch.from_numpy(ref.e4m3_encode_bruteforce(np.arange(-4.0, 5.0))).to(gpu)
    wv = torch.zeros((experts, n, k), dtype=torch.uint8, device=gpu)
    wv[-1] = integers[torch.randint(0, 9, (n, k), generator=gen, device=gpu)]
    ws = torch.ones((experts, n // 128, k // 128), device=gpu)
    w = prepare_fp8_block_weight(wv, ws)
    wv = wv[-1:].clone()
    for r in (3, 90):
        xv = integers[torch.randint(0, 9, (r, k), generator=gen, device=gpu)]
        xs = torch.ones((r, k // 128), device=gpu)
        offsets = torch.zeros(experts + 1, dtype=torch.int32, device=gpu)
        offsets[-1] = r
        out = launch_fp8_block_matmul_experts(xv, xs, w, offsets)
        assert torch.equal(out.double(), exact(xv, xs, wv[0], ws[0])[0])


@pytest.mark.gpu
def test_join_and_router_far_apart(gpu):
    from mambo_amd.kernels.experts import launch_combine_experts, launch_route_experts
    rng = np.random.default_rng(3)
    y = torch.empty((40, 1 << 26), dtype=torch.bfloat16, device=gpu)[:, :130]  # 5.4 GB
    y.copy_(torch.from_numpy(rng.standard_normal((40, 130)).astype(np.float32)))
    slots = torch.from_numpy(rng.permutation(40).reshape(20, 2).astype(np.int32)).to(gpu)
    weights = torch.rand((20, 2), device=gpu)
    out = torch.empty((20, 1 << 26), device=gpu)[:, :130]
    launch_combine_experts(y, slots, weights, out_dtype=torch.float32, out=out)
    assert torch.equal(out, launch_combine_experts(y.contiguous(), slots, weights, out_dtype=torch.float32))
    logits = torch.empty((40, 1 << 26), dtype=torch.bfloat16, device=gpu)[:, :70]
    logits.copy_(torch.from_numpy(rng.standard_normal((40, 70)).astype(np.float32)))
    for a, b in zip(launch_route_experts(logits, 3), launch_route_experts(logits.contiguous(), 3)):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------ IQ3_S by expert
@pytest.mark.gpu
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("r,experts,n,k", [
    (3, 4, 70, 2304), (6, 4, 9000, 2304), (150, 120, 1000, 2304),  # 4 tokens a tile: four waves, two, one
    (20, 4, 70, 2304), (60, 6, 6000, 2304), (200, 20, 4000, 2048),  # 16 tokens a tile: four, two, one
    (300, 4, 2211, 1024),  # the 32 x 32 MFMAs, 64 x 128 tiles
    (130, 8, 4090, 2048), (500, 8, 4090, 2304),  # of two K groups: 64 tokens, 128
    (900, 2, 1500, 1280), (1100, 64, 600, 768), (1300, 3, 3000, 1024),
])
def test_iq3s_kernels(gpu, r, experts, n, k, gather):
    """As test_gpu_experts.test_iq3s_experts, at sizes that each of the kernels takes; an expert may have
    more rows than the tile of the kernel that the average chose."""
    from mambo_amd.kernels.experts import launch_iq3_s_fp8_matmul_experts
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
    from oracle import oracle
    rng = np.random.default_rng(r + experts + n + k)
    m = max(1, r // 3) if gather else r
    raws = rng.integers(0, 256, size=(experts, n, k // 256, 110), dtype=np.uint8)
    raws[..., :2] = (0.01 + 0.02 * rng.random((experts, n, k // 256, 1))).astype(np.float16).view(np.uint8)
    x = rng.standard_normal((m, k)).astype(np.float32)
    offsets = ref.some_offsets(rng, r, experts, 1)
    rows = rng.integers(0, m, size=r).astype(np.int32) if gather else np.arange(r, dtype=np.int32)
    eq, es = oracle.quantize_mxfp8(x)
    expected = np.zeros((r, n))
    for e in range(experts):
        at = rows[offsets[e]:offsets[e + 1]]
        if at.size:
            expected[offsets[e]:offsets[e + 1]] = oracle.iq3s_fp8_matmul(eq[at], es[at], raws[e])
    x, raws, offsets, rows = (torch.from_numpy(a).to(gpu) for a in (x, raws, offsets, rows))
    w = prepare_iq3_s_experts(raws)
    values, scales = launch_quantize_fp8(x)
    taken = int(offsets[-1])
    for dtype, tolerance in ((F32, 1e-4), (BF16, 2.0**-8)):
        out = launch_iq3_s_fp8_matmul_experts(values, scales, w, offsets, rows=rows if gather else None,
                                              out_dtype=dtype).double().cpu().numpy()
        assert not out[taken:].any()
        for i in range(taken):  # row by row, so that one wrong row shows
            assert np.linalg.norm(out[i] - expected[i]) <= tolerance * np.linalg.norm(expected[i]), i
