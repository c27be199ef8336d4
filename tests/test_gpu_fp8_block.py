"""E4M3 products with a scale for each block of 128, on the GPU: the quantizer bit for bit, the
products exactly where the sums are integers and within the bound of float32 sums otherwise."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import expert_reference as ref

pytestmark = pytest.mark.gpu


def ops():
    from mambo_amd.kernels import fp8_block
    from mambo_amd.utils import fp8_block_weight
    return fp8_block, fp8_block_weight


def device(gpu, *arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).to(gpu) for a in arrays]


# ------------------------------------------------------------------------------ quantizer
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k", [(1, 16), (1, 4096), (3, 112), (2, 128), (5, 144), (70, 2832), (7, 4112)])
def test_quantizer_matches_the_division(gpu, m, k, dtype):
    fp8, _ = ops()
    rng = np.random.default_rng(m * 10000 + k)
    x = rng.standard_normal((m, k)) * np.exp2(rng.integers(-30, 30, size=(m, k // 16)).repeat(16, 1))
    x[rng.random((m, k)) < 0.1] = 0.0
    x = torch.from_numpy(x).to(dtype)
    codes, scales = fp8.launch_quantize_fp8_block(x.to(gpu))
    expected = ref.quantize_block(x.float().numpy())
    assert np.array_equal(codes.cpu().numpy(), expected[0])
    assert np.array_equal(scales.cpu().numpy(), expected[1])


def test_quantizer_keeps_halves_of_bf16_rows(gpu):
    """Values half way between two codes go to the even one, whatever amax is."""
    fp8, _ = ops()
    for mantissa in range(128):
        amax = (1.0 + mantissa / 128.0)
        steps = np.concatenate([np.arange(16, 32) + 0.5, np.arange(16, 32)]) / 32.0  # of E4M3's top binades
        x = torch.tensor(np.concatenate([[amax], amax * steps * 448 / 480]), dtype=torch.float64)
        x = torch.nn.functional.pad(x, (0, 48 - x.numel()))[None].to(torch.bfloat16)
        codes, _ = fp8.launch_quantize_fp8_block(x.to(gpu))
        peak = x.double().abs().max()
        q = ref.e4m3_encode_bruteforce((448.0 * x.double() / peak).numpy()).reshape(1, -1)
        assert np.array_equal(codes.cpu().numpy(), q), mantissa


def test_quantizer_extremes(gpu):
    fp8, _ = ops()
    x = torch.zeros((9, 256), dtype=torch.float32)
    x[1, 3] = -0.0
    x[2, :4] = torch.tensor([3.4e38, -3.4e38, 1e30, 1.0])
    x[3, :4] = torch.tensor([1e-45, -1e-40, 1e-38, 0.0])
    x[4, 5] = float("inf")
    x[5, 130] = float("nan")
    x[6, 200] = float("-inf")
    x[7, :3] = torch.tensor([448.0 * 2.0**-100, 2.0**-101, -(2.0**-100)])
    x[8] = 1.0
    codes, scales = (t.cpu() for t in fp8.launch_quantize_fp8_block(x.to(gpu)))
    for row in (0, 1, 2, 3, 7, 8):
        expected = ref.quantize_block(x[row:row + 1].numpy())
        assert np.array_equal(codes[row].numpy(), expected[0][0]), row
        assert np.array_equal(scales[row].numpy(), expected[1][0]), row
    for row, group in ((4, 0), (5, 1), (6, 1)):  # the group is NaN, the other one is not
        assert torch.isnan(scales[row, group]) and (codes[row].view(2, 128)[group] & 127 == 127).all()
        assert scales[row, 1 - group] == 2.0**-100 and (codes[row].view(2, 128)[1 - group] == 0).all()


def test_quantizer_strides_and_out(gpu):
    fp8, _ = ops()
    rng = np.random.default_rng(7)
    base = torch.from_numpy(rng.standard_normal((12, 400)).astype(np.float32)).to(gpu)
    for x in (base[:, 16:160], base[::3, 1:145], base.t()[:, :].contiguous().t()[:, :144], base[:1].expand(5, 400)):
        expected = ref.quantize_block(x.cpu().numpy())
        codes, scales = fp8.launch_quantize_fp8_block(x)
        assert np.array_equal(codes.cpu().numpy(), expected[0]) and np.array_equal(scales.cpu().numpy(), expected[1])
    big = torch.full((12, 403), 9, dtype=torch.uint8, device=gpu)
    out = (big[:, 1:401], torch.empty((12, 9), dtype=torch.float32, device=gpu)[:, 2:6])
    assert fp8.launch_quantize_fp8_block(base, out=out)[0].data_ptr() == out[0].data_ptr()
    expected = ref.quantize_block(base.cpu().numpy())
    assert np.array_equal(out[0].cpu().numpy(), expected[0]) and np.array_equal(out[1].cpu().numpy(), expected[1])
    assert (big[:, 0] == 9).all() and (big[:, 401:] == 9).all()


# ------------------------------------------------------------------------------ products
SHAPES = [(1, 1, 16), (1, 1024, 4096), (2, 33, 112), (3, 130, 144), (15, 64, 128), (16, 96, 256), (17, 257, 272),
          (31, 31, 1024), (33, 160, 640), (64, 128, 512), (65, 300, 1040), (97, 129, 384), (128, 256, 2048),
          (130, 500, 656), (203, 1003, 2832), (256, 320, 1024), (300, 257, 128), (513, 640, 768), (1000, 384, 400)]


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_integers_add_up_exactly(gpu, m, n, k, out_dtype):
    """Codes of small integers and scales of powers of two: every order of the sum gives the same
    float32, so a term that is missing, doubled or misplaced shows."""
    fp8, weight = ops()
    rng = np.random.default_rng(m + 7 * n + 13 * k)
    g = -(-k // 128)
    xv, wv = ref.integer_codes(rng, (m, k)), ref.integer_codes(rng, (n, k))
    xs = np.exp2(rng.integers(-1, 2, size=(m, g))).astype(np.float32)
    ws = np.exp2(rng.integers(-1, 2, size=(-(-n // 128), g))).astype(np.float32)
    expected = ref.product(xv, xs, wv, ws)[0]
    assert np.abs(expected).max() < 2**22  # a multiple of 1/4 in 24 bits
    xv, xs, wv, ws = device(gpu, xv, xs, wv, ws)
    out = fp8.launch_fp8_block_matmul(xv, xs, weight.prepare_fp8_block_weight(wv, ws), out_dtype=out_dtype)
    assert out.dtype == out_dtype
    assert torch.equal(out.cpu(), torch.from_numpy(expected).to(torch.float32).to(out_dtype))


@pytest.mark.parametrize("m,n,k", [(1, 200, 4096), (9, 72, 1040), (40, 129, 2048), (128, 256, 1024), (301, 200, 7152)])
def test_real_scales(gpu, m, n, k):
    fp8, weight = ops()
    rng = np.random.default_rng(m * n + k)
    g = -(-k // 128)
    xv, wv = ref.random_codes(rng, (m, k)), ref.random_codes(rng, (n, k))
    xs = rng.uniform(1e-3, 1.0, size=(m, g)).astype(np.float32) * np.float32(10.0) ** rng.integers(-3, 3, size=(m, g))
    xs = xs.astype(np.float32)
    ws = rng.uniform(-2.0, 2.0, size=(-(-n // 128), g)).astype(np.float32)
    expected, magnitudes = ref.product(xv, xs, wv, ws)
    tensors = device(gpu, xv, xs, wv, ws)
    w = weight.prepare_fp8_block_weight(tensors[2], tensors[3])
    for dtype in (torch.float32, torch.bfloat16):
        out = fp8.launch_fp8_block_matmul(tensors[0], tensors[1], w, out_dtype=dtype).double().cpu().numpy()
        assert (np.abs(out - expected) <= ref.bound(magnitudes, k, expected, dtype)).all()


def test_rows_are_the_same_alone(gpu):
    """A row's result does not depend on the rows beside it where the kernel is the same, and is
    repeatable."""
    fp8, weight = ops()
    rng = np.random.default_rng(3)
    xv, xs, wv, ws = device(gpu, ref.random_codes(rng, (40, 1040)), rng.random((40, 9)).astype(np.float32),
                            ref.random_codes(rng, (100, 1040)), rng.random((1, 9)).astype(np.float32))
    w = weight.prepare_fp8_block_weight(wv, ws)
    out = fp8.launch_fp8_block_matmul(xv, xs, w)
    for _ in range(3):
        assert torch.equal(out, fp8.launch_fp8_block_matmul(xv, xs, w))
    assert torch.equal(out[8:], fp8.launch_fp8_block_matmul(xv[8:], xs[8:], w))


def test_nan_stays_in_its_row_and_column(gpu):
    fp8, weight = ops()
    rng = np.random.default_rng(5)
    for m, k in ((5, 144), (70, 400), (300, 1040)):
        xv, wv = ref.integer_codes(rng, (m, k)), ref.integer_codes(rng, (75, k))
        g = -(-k // 128)
        xs, ws = np.ones((m, g), dtype=np.float32), np.ones((1, g), dtype=np.float32)
        clean = ref.product(xv, xs, wv, ws)[0].astype(np.float32)
        xv[2, k - 3], wv[70, 5] = 0x7F, 0xFF
        xs[m - 1, g - 1] = np.inf
        xv, xs, wv, ws = device(gpu, xv, xs, wv, ws)
        out = fp8.launch_fp8_block_matmul(xv, xs, weight.prepare_fp8_block_weight(wv, ws)).cpu().numpy()
        assert np.isnan(out[2]).all() and np.isnan(out[:, 70]).all()
        assert not np.isfinite(out[m - 1]).any()
        keep = np.ones(out.shape, dtype=bool)
        keep[[2, m - 1]] = False
        keep[:, 70] = False
        assert np.array_equal(out[keep], clean[keep])


def test_strided_rows_and_outputs(gpu):
    """Rows of a wider buffer are read in place, unaligned ones copied; outputs of a wider buffer get
    their columns and nothing beside them."""
    fp8, weight = ops()
    rng = np.random.default_rng(11)
    for m, n, k in ((5, 70, 144), (150, 131, 272)):
        g = -(-k // 128)
        xv, wv = ref.integer_codes(rng, (m, k)), ref.integer_codes(rng, (n, k))
        xs = np.exp2(rng.integers(-1, 2, size=(m, g))).astype(np.float32)
        ws = np.exp2(rng.integers(-1, 2, size=(-(-n // 128), g))).astype(np.float32)
        expected = torch.from_numpy(ref.product(xv, xs, wv, ws)[0]).float()
        xv, xs, wv, ws = device(gpu, xv, xs, wv, ws)
        wide_w = torch.zeros((n, k + 37), dtype=torch.uint8, device=gpu)
        wide_w[:, 5:5 + k] = wv
        w = weight.prepare_fp8_block_weight(wide_w[:, 5:5 + k].view(torch.float8_e4m3fn), ws)
        for pad, shift in ((48, 16), (3, 1)):
            wide = torch.full((m, k + pad), 0x7F, dtype=torch.uint8, device=gpu)
            wide[:, shift:shift + k] = xv
            scales = torch.full((m, g + 3), float("nan"), device=gpu)
            scales[:, 1:1 + g] = xs
            for dtype in (torch.float32, torch.bfloat16):
                for left, right in ((4, 8), (3, 2)):
                    buf = torch.full((m, left + n + right), 77.0, dtype=dtype, device=gpu)
                    view = buf[:, left:left + n]
                    got = fp8.launch_fp8_block_matmul(wide[:, shift:shift + k], scales[:, 1:1 + g], w, out_dtype=dtype,
                                                      out=view)
                    assert got.data_ptr() == view.data_ptr()
                    assert torch.equal(view.cpu(), expected.to(dtype))
                    assert (buf[:, :left] == 77).all() and (buf[:, left + n:] == 77).all()


def test_no_rows(gpu):
    fp8, weight = ops()
    w = weight.prepare_fp8_block_weight(torch.zeros((8, 32), dtype=torch.uint8, device=gpu), torch.ones((1, 1), device=gpu))
    values, scales = fp8.launch_quantize_fp8_block(torch.empty((0, 32), device=gpu))
    assert values.shape == (0, 32) and scales.shape == (0, 1)
    assert fp8.launch_fp8_block_matmul(values, scales, w).shape == (0, 8)


def test_side_stream(gpu):
    """On a stream of its own, copies of unaligned rows and the output included."""
    fp8, weight = ops()
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.standard_normal((130, 1041)).astype(np.float32)).to(gpu)[:, 1:]
    codes, scales = device(gpu, ref.random_codes(rng, (300, 1040)), rng.random((3, 9)).astype(np.float32))
    w = weight.prepare_fp8_block_weight(codes, scales)
    expected = fp8.launch_fp8_block_matmul(*fp8.launch_quantize_fp8_block(x), w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        w2 = weight.prepare_fp8_block_weight(codes, scales, stream=stream)
        values, s = fp8.launch_quantize_fp8_block(x, stream=stream)
        out = fp8.launch_fp8_block_matmul(values, s, w2, stream=stream)
        side.synchronize()
        assert torch.equal(out, expected)


def test_refusals(gpu):
    fp8, weight = ops()
    codes, scales = torch.zeros((8, 32), dtype=torch.uint8, device=gpu), torch.ones((1, 1), device=gpu)
    w = weight.prepare_fp8_block_weight(codes, scales)
    xv, xs = torch.zeros((2, 32), dtype=torch.uint8, device=gpu), torch.ones((2, 1), device=gpu)
    value = [
        lambda: fp8.launch_quantize_fp8_block(torch.zeros((2, 24), device=gpu)),
        lambda: fp8.launch_quantize_fp8_block(torch.zeros((2, 32), dtype=torch.float16, device=gpu)),
        lambda: fp8.launch_quantize_fp8_block(torch.zeros((2, 32))),
        lambda: fp8.launch_quantize_fp8_block(torch.zeros((2, 32), device=gpu), out=(xv[:1], xs)),
        lambda: fp8.launch_quantize_fp8_block(torch.zeros((2, 32), device=gpu), out=(xv[:1].expand(2, 32), xs)),
        lambda: weight.prepare_fp8_block_weight(codes.int(), scales),
        lambda: weight.prepare_fp8_block_weight(codes.cpu(), scales),
        lambda: weight.prepare_fp8_block_weight(codes, scales.cpu()),
        lambda: weight.prepare_fp8_block_weight(codes, scales.double()),
        lambda: weight.prepare_fp8_block_weight(codes, torch.ones((1, 2), device=gpu)),
        lambda: weight.prepare_fp8_block_weight(codes[:, :24], scales),
        lambda: fp8.launch_fp8_block_matmul(xv[:, :16], xs, w),
        lambda: fp8.launch_fp8_block_matmul(xv.view(torch.int8), xs, w),
        lambda: fp8.launch_fp8_block_matmul(xv, xs[:1], w),
        lambda: fp8.launch_fp8_block_matmul(xv, xs.double(), w),
        lambda: fp8.launch_fp8_block_matmul(xv, xs.cpu(), w),
        lambda: fp8.launch_fp8_block_matmul(xv, xs, w, out_dtype=torch.float16),
        lambda: fp8.launch_fp8_block_matmul(xv, xs, w, out=torch.empty((2, 9), device=gpu)),
        lambda: fp8.launch_fp8_block_matmul(xv, xs, w, out=torch.empty((8, 2), device=gpu).t()),
        lambda: fp8.launch_fp8_block_matmul(xv, xs, w, out_dtype=torch.bfloat16, out=torch.empty((2, 8), device=gpu)),
        lambda: fp8.launch_fp8_block_matmul(xv, xs, weight.prepare_fp8_block_weight(codes[None].expand(2, 8, 32),
                                                                                   scales[None].expand(2, 1, 1))),
    ]
    for call in value:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        fp8.launch_fp8_block_matmul(xv, xs, codes)
