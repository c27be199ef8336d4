"""Every kernel of the IQ3_S product by expert, each at sizes that are held to it: six that stream the weights (4 or
16 tokens a tile, one, two or four waves that share K) and six shapes of the 32 x 32 MFMA kernel. Many rows
of no expert, experts without rows and with more than a tile, K of one block and fewer blocks than K groups."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import expert_reference as ref
from conftest import make_synthetic_iq3_s

F32, BF16 = torch.float32, torch.bfloat16

# kernel (tokens, weight rows, parts of K): (rows, experts, rows of none, N, K blocks)
CASES = [
    ((4, 32, 1), (1, 1, 0, 17, 1)), ((4, 32, 1), (150, 120, 30, 1000, 9)), ((4, 32, 2), (1, 1, 0, 17, 4)),
    ((4, 32, 2), (6, 4, 1, 9000, 9)), ((4, 32, 4), (3, 4, 1, 70, 9)), ((4, 32, 4), (2, 1, 0, 33, 8)),
    ((16, 32, 1), (3, 1, 0, 17, 1)), ((16, 32, 1), (200, 20, 40, 4000, 8)), ((16, 32, 2), (3, 1, 0, 17, 4)),
    ((16, 32, 2), (60, 6, 9, 6000, 9)), ((16, 32, 4), (20, 4, 5, 70, 9)), ((16, 32, 4), (4, 1, 0, 17, 8)),
    ((64, 64, 4), (300, 4, 77, 2211, 4)), ((64, 64, 4), (8047, 29, 1300, 42, 3)),
    ((64, 128, 1), (5495, 1, 600, 66, 1)), ((64, 128, 1), (1100, 64, 140, 600, 3)), ((64, 128, 1), (1300, 3, 1, 3000, 4)),
    ((64, 128, 2), (130, 8, 35, 4090, 8)), ((64, 128, 2), (7894, 22, 1000, 71, 4)),
    ((128, 128, 1), (3120, 44, 500, 1297, 2)), ((128, 128, 1), (2600, 8, 333, 4090, 9)),
    ((128, 128, 2), (500, 8, 140, 4090, 9)), ((128, 128, 2), (6728, 79, 900, 135, 4)),
    ((128, 256, 1), (8059, 9, 1111, 651, 1)), ((128, 256, 1), (2442, 1, 300, 12787, 10)),
]


def plan(r, experts, n, blocks, m=None, ldxv=None):
    from mambo_amd import _native
    out = (ctypes.c_int32 * 3)()
    _native.check(_native.lib().mambo_iq3s_experts_plan(r if m is None else m, r, experts, n, blocks, ldxv or 256 * blocks,
                                                        8 * blocks, out))
    return tuple(out)


def test_each_size_takes_its_kernel():
    for kernel, (r, experts, _, n, blocks) in CASES:
        assert plan(r, experts, n, blocks) == plan(r, experts, n, blocks, m=max(1, r // 3)) == kernel, (r, experts, n, blocks)
    assert len({kernel for kernel, _ in CASES}) == 12


def test_rows_that_32_bit_offsets_do_not_reach_take_16_tokens_a_tile():
    """Gathered from 4 GiB and more, or 2^24 bytes apart, and more row tiles than a grid's second dimension."""
    assert plan(4096, 8, 4096, 56, m=299592)[0] == plan(4096, 8, 4096, 56)[0] == 128
    assert plan(4096, 8, 4096, 56, m=299593)[:2] == plan(4096, 8, 4096, 56, ldxv=1 << 24)[:2] == (16, 32)
    assert plan(64 * 65535, 8, 64, 1)[:2] == (16, 32)


def test_plan_refuses_what_the_call_refuses():
    from mambo_amd import _native
    lib, out = _native.lib(), (ctypes.c_int32 * 3)()
    good = dict(m=5, r=5, experts=2, n=64, blocks=1, ldxv=256, ldxs=8)
    assert lib.mambo_iq3s_experts_plan(*good.values(), out) == 0
    for bad in (dict(n=0), dict(blocks=0), dict(experts=0), dict(experts=1025), dict(r=0), dict(r=-1), dict(m=0), dict(ldxv=255),
                dict(ldxs=7), dict(r=2**31 - 1)):
        assert lib.mambo_iq3s_experts_plan(*{**good, **bad}.values(), out) == _native.MAMBO_ERR_VALUE, bad
    assert lib.mambo_iq3s_experts_plan(*good.values(), None) == _native.MAMBO_ERR_VALUE


@pytest.mark.gpu
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("kernel,size", CASES, ids=["-".join(map(str, (*k, *s))) for k, s in CASES])
def test_kernel(gpu, kernel, size, gather):
    """Against products in 64 bits of the decoded rows and weights (exact in float32), within the relative 2-norm of a
    row that test_gpu_experts.test_iq3s_experts derives, over all of the rows; rows of no expert are zeros."""
    from mambo_amd.kernels.experts import launch_iq3_s_fp8_matmul_experts
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
    from oracle import oracle
    r, experts, unrouted, n, blocks = size
    rng = np.random.default_rng(r + experts + n + blocks)
    m = max(1, r // 3) if gather else r
    raws = np.stack([make_synthetic_iq3_s(n, 256 * blocks, seed=7 * r + e) for e in range(experts)])
    x = rng.standard_normal((m, 256 * blocks)).astype(np.float32)
    offsets = ref.some_offsets(rng, r, experts, unrouted)
    rows = rng.integers(0, m, size=r).astype(np.int32) if gather else np.arange(r, dtype=np.int32)
    rows[offsets[-1]:] = -1
    values, scales = oracle.quantize_mxfp8(x)
    decoded = torch.from_numpy(oracle.mxfp8_decode(values, scales)).to(gpu).double()
    expected = torch.zeros((r, n), dtype=torch.float64, device=gpu)
    for e in range(experts):
        a, b = int(offsets[e]), int(offsets[e + 1])
        if a < b:
            w = torch.from_numpy(oracle.dequant_iq3s(raws[e])).to(gpu).double()
            expected[a:b] = decoded[torch.from_numpy(rows[a:b]).to(gpu).long()] @ w.t().contiguous()
    taken = int(offsets[-1])
    assert taken == r - unrouted
    weight = prepare_iq3_s_experts(torch.from_numpy(raws).to(gpu))
    values, scales = launch_quantize_fp8(torch.from_numpy(x).to(gpu))
    offsets, rows = torch.from_numpy(offsets).to(gpu), torch.from_numpy(rows).to(gpu)
    for dtype, tolerance in ((F32, 1e-4), (BF16, 2.0**-8)):
        buffer = torch.full((r + 2, n + 7), 77.0, dtype=dtype, device=gpu)
        out = launch_iq3_s_fp8_matmul_experts(values, scales, weight, offsets, rows=rows if gather else None, out_dtype=dtype,
                                              out=buffer[1:r + 1, 4:n + 4])
        assert bool((buffer[0] == 77).all()) and bool((buffer[r + 1] == 77).all())
        assert bool((buffer[:, :4] == 77).all()) and bool((buffer[:, n + 4:] == 77).all())
        assert not bool(out[taken:].any())
        off, size_of = (out.double() - expected)[:taken].norm(dim=1), expected[:taken].norm(dim=1)
        assert bool((off <= tolerance * size_of).all()), (off / size_of).max()
        again = launch_iq3_s_fp8_matmul_experts(values, scales, weight, offsets, rows=rows if gather else None, out_dtype=dtype)
        assert torch.equal(again, out)  # other strides, the same sums in the same order
