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
