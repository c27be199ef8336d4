"""Launchers on a stream that is not the current one, whose inputs that stream alone has made: the
copies that a launcher makes of them come after them, and the memory that it allocates is not the current
stream's, which may still have work to do in it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import make_synthetic_iq3_s

pytestmark = pytest.mark.gpu


@pytest.fixture
def side(gpu):
    stream = torch.cuda.Stream()
    yield stream
    torch.cuda.synchronize()


def keep_busy(stream) -> None:
    """Some tens of milliseconds of work on the stream."""
    with torch.cuda.stream(stream):
        a = torch.full((4096, 4096), 1e-3, device="cuda")
        for _ in range(40):
            a = a @ a
            a *= 1e-3


def made_on(stream, data: torch.Tensor, late: torch.Tensor) -> torch.Tensor:
    """`late` (zeros until then) holding `data` once the stream has got through other work."""
    torch.cuda.synchronize()
    keep_busy(stream)
    with torch.cuda.stream(stream):
        late.copy_(data)
    return late


def freed_blocks_of(sizes) -> None:
    """Blocks of these sizes back in the current stream's pool, which is still to overwrite them."""
    blocks = [torch.empty(s, dtype=torch.uint8, device="cuda") for s in sizes]
    torch.cuda.synchronize()
    keep_busy(torch.cuda.current_stream())
    for b in blocks:
        b.fill_(0xA5)


def test_quantizer_copies_its_rows_on_the_stream(gpu, side):
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    rng = np.random.default_rng(1)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.from_numpy(rng.standard_normal((256, 70)).astype(np.float32)).to(gpu).to(dtype)
        expected = launch_quantize_fp8(x.t().contiguous())
        for stream in (side, side.cuda_stream):
            late = made_on(side, x, torch.zeros_like(x))
            got = launch_quantize_fp8(late.t(), stream=stream)  # columns apart: copied first
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_quantizer_allocates_on_the_stream(gpu, side):
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    x = torch.randn((1000, 8192), device=gpu)
    expected = launch_quantize_fp8(x)
    freed_blocks_of([1000 * 8192, 1000 * 256])
    got = launch_quantize_fp8(x, stream=side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


# ------------------------------------------------------------------------------ IQ3_S projections
M, N, K = 4, 96, 512


def weights(gpu, count: int = 1, n: int = N):
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_fields
    made = [prepare_iq3_s_fields(torch.from_numpy(make_synthetic_iq3_s(n, K, seed=e)).to(gpu), pack=True)
            for e in range(count)]
    torch.cuda.synchronize()
    return made


def late_rows(side, m: int):
    """MXFP8 rows (values, scales), and the same in buffers whose rows no kernel reads in place, made on the
    side stream late."""
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    values, scales = launch_quantize_fp8(torch.randn((m, K), device="cuda"))
    wide = torch.zeros((m, K + 3), dtype=torch.uint8, device="cuda")[:, 1:K + 1]
    wide_scales = torch.zeros((m, K // 32 + 3), dtype=torch.uint8, device="cuda")[:, 1:K // 32 + 1]
    made_on(side, values, wide)
    with torch.cuda.stream(side):
        wide_scales.copy_(scales)
    return (values, scales), (wide, wide_scales)


def test_projections_copy_their_rows_on_the_stream(gpu, side):
    from mambo_amd.kernels import iq3_s_fp8 as ops
    w = weights(gpu, 2)
    rows, late = late_rows(side, M)
    got = ops.launch_iq3_s_fp8_matmul(*late, w[0], stream=side)
    side.synchronize()
    assert torch.equal(got, ops.launch_iq3_s_fp8_matmul(*rows, w[0]))
    rows, late = late_rows(side, M)
    got = ops.launch_iq3_s_fp8_matmul_grouped(*late, w, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ops.launch_iq3_s_fp8_matmul_grouped(*rows, w)))
    x = torch.randn((K, M), device=gpu)
    expected = ops.launch_iq3_s_matmul_quantize(x.t().contiguous(), w)
    late = made_on(side, x, torch.zeros_like(x))
    got = ops.launch_iq3_s_matmul_quantize(late.t(), w, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_chain_copies_and_clears_on_the_stream(gpu, side):
    from mambo_amd.kernels import iq3_s_fp8 as ops
    w = weights(gpu, 2)
    x = torch.randn((M, K), device=gpu)
    rows, late = late_rows(side, M)
    expected = ops.launch_iq3_s_fp8_matmul_chain([ops.ChainLaunch(x, w), ops.ChainLaunch(rows[0], w, rows[1])])
    late_x = torch.zeros((M, K + 1), device=gpu)[:, 1:]
    made_on(side, x, late_x)
    freed_blocks_of([4 * 4224])  # the sync words': all ones, were they the current stream's
    got = ops.launch_iq3_s_fp8_matmul_chain([ops.ChainLaunch(late_x, w), ops.ChainLaunch(late[0], w, late[1])],
                                            stream=side)
    torch.cuda.synchronize()
    for a, b in zip(got, expected):
        assert all(torch.equal(i, j) for i, j in zip(a, b))


def test_projections_allocate_on_the_stream(gpu, side):
    from mambo_amd.kernels import iq3_s_fp8 as ops
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    w = weights(gpu, 1, 4096)
    m = 300
    x = torch.randn((m, K), device=gpu)
    values, scales = launch_quantize_fp8(x)
    expected = ops.launch_iq3_s_fp8_matmul(values, scales, w[0])
    for call in (lambda: ops.launch_iq3_s_fp8_matmul(values, scales, w[0], stream=side),
                 lambda: ops.launch_iq3_s_fp8_matmul_grouped(values, scales, w, stream=side)[0],
                 lambda: ops.launch_iq3_s_matmul_quantize(x, w[0], stream=side)):
        freed_blocks_of([4 * m * 4096, m * K, m * K // 32])
        got = call()
        torch.cuda.synchronize()
        assert torch.equal(got, expected)


def test_weights_allocate_on_the_stream(gpu, side):
    from mambo_amd.kernels.iq3_s_fp8 import launch_dequant_iq3_s
    from mambo_amd.utils.iq3_s_weight import ensure_packed, packed_bytes, prepare_iq3_s_fields
    n, blocks = 5000, 8
    raw = torch.from_numpy(make_synthetic_iq3_s(n, 256 * blocks, seed=3)).to(gpu)
    expected = prepare_iq3_s_fields(raw, pack=True)
    decoded = launch_dequant_iq3_s(expected)
    names = ("d", "qs", "qh", "signs", "scales")
    sizes = [getattr(expected, name).numel() * getattr(expected, name).element_size() for name in names]
    freed_blocks_of([*sizes, packed_bytes(n, blocks)])
    got = prepare_iq3_s_fields(raw, pack=True, stream=side)
    torch.cuda.synchronize()
    for name in (*names, "packed"):
        assert torch.equal(getattr(got, name).view(torch.uint8), getattr(expected, name).view(torch.uint8)), name
    unpacked = prepare_iq3_s_fields(raw)
    freed_blocks_of([packed_bytes(n, blocks)])
    packed = ensure_packed(unpacked, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(packed, expected.packed)
    freed_blocks_of([n * blocks * 256, n * blocks * 32])
    values, scales = launch_dequant_iq3_s(expected, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(values, decoded[0]) and torch.equal(scales, decoded[1])
