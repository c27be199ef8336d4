"""Rotary positions on the GPU against rotations in 64 bits: layouts, parts of the head, scalings, far
positions, strides, in place."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu

LLAMA3 = {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_length": 8192}
YARN = {"type": "yarn", "factor": 16.0, "original_length": 4096}


def rotary():
    from mambo_amd.kernels.rotary import launch_rotary
    return launch_rotary


def check(got, x, positions, frequencies, interleaved, magnitude, size):
    x64 = x.double().cpu().numpy()
    expected = ref.rotate(x64, positions, frequencies, interleaved, magnitude)
    bound = ref.rotation_bound(x64, size, interleaved, magnitude)
    bound += (np.abs(expected) + bound) * torch.finfo(got.dtype).eps / 2
    assert (np.abs(got.double().cpu().numpy() - expected) <= bound).all()
    if got.dtype == x.dtype:
        assert torch.equal(got[..., size:], x[..., size:])


# tokens, heads, head size, rotated values
SHAPES = [(1, 1, 2, 2), (1, 40, 128, 128), (3, 5, 80, 40), (9, 2, 64, 64), (7, 3, 96, 96), (2, 9, 20, 6), (33, 4, 256, 256),
          (5, 1, 1024, 1024), (1030, 3, 64, 32), (2100, 2, 32, 32), (6, 17, 72, 48), (4, 3, 600, 400)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,size", SHAPES)
@pytest.mark.parametrize("dtype,out_dtype", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
                                             (torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
def test_rotation(gpu, tokens, heads, dim, size, interleaved, dtype, out_dtype):
    from mambo_amd.utils.rotary_table import prepare_rotary_table, rotary_frequencies
    rng = np.random.default_rng(dim + size)
    x = torch.from_numpy(rng.standard_normal((tokens, heads, dim)).astype(np.float32)).to(gpu).to(dtype)
    positions = rng.integers(0, 100000, tokens).astype(np.int32)
    table = prepare_rotary_table(size, interleaved=interleaved)
    got = rotary()(x, *ref.device(gpu, positions), table, out_dtype=out_dtype)
    assert got.dtype == out_dtype
    check(got, x, positions, rotary_frequencies(size)[0], interleaved, 1.0, size)


@pytest.mark.parametrize("scaling", [LLAMA3, YARN, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 2.0}])
def test_scalings_and_far_positions(gpu, scaling):
    from mambo_amd.utils.rotary_table import prepare_rotary_table, rotary_frequencies
    rng = np.random.default_rng(1)
    positions = np.array([0, 1, -1, -77, 2**20 + 3, 2**31 - 1, -2**31, 99999], dtype=np.int32)
    x = torch.from_numpy(rng.standard_normal((8, 2, 64)).astype(np.float32)).to(gpu)
    frequencies, magnitude = rotary_frequencies(64, base=500000.0, scaling=scaling)
    got = rotary()(x, *ref.device(gpu, positions), prepare_rotary_table(64, base=500000.0, scaling=scaling))
    # the frequencies' own 2^-53, times positions of 2^31, are 2^-22 of a radian
    x64 = x.double().cpu().numpy()
    expected = ref.rotate(x64, positions, frequencies, False, magnitude)
    bound = ref.rotation_bound(x64, 64, False, magnitude)
    far = np.abs(positions.astype(np.float64)) * 2.0**-51
    bound = bound * (1 + far[:, None, None] / (12 * 2.0**-24)) + np.abs(expected) * 2.0**-24
    assert (np.abs(got.double().cpu().numpy() - expected) <= bound).all()


def test_given_frequencies(gpu):
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    rng = np.random.default_rng(2)
    frequencies = [1.0, 0.25, -0.5, 7.0]
    x = torch.from_numpy(rng.standard_normal((5, 3, 8)).astype(np.float32)).to(gpu)
    positions = np.arange(5, dtype=np.int32)
    got = rotary()(x, *ref.device(gpu, positions), prepare_rotary_table(8, frequencies=frequencies))
    check(got, x, positions, frequencies, False, 1.0, 8)


def test_strides_alignment_and_place(gpu):
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    rng = np.random.default_rng(3)
    positions = ref.device(gpu, rng.integers(0, 9999, 50).astype(np.int32))[0]
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.from_numpy(rng.standard_normal((50, 6, 70)).astype(np.float32)).to(gpu).to(dtype)
        for interleaved in (False, True):
            table = prepare_rotary_table(32, interleaved=interleaved)
            for view in (wide[:, 1:5, :64], wide[:, :, 3:67], wide[:, ::2, :64], wide.transpose(0, 1).contiguous().transpose(0, 1)[..., :64],
                         wide[..., 0:64].flip(2), wide[:1, :1, :64].expand(50, 6, 64)):
                expected = rotary()(view.contiguous(), positions, table)
                assert torch.equal(rotary()(view, positions, table), expected)
                whole = torch.full((52, 8, 70), 7.0, dtype=dtype, device=gpu)
                out = whole[1:51, 1:1 + view.shape[1], 3:67]
                assert rotary()(view, positions, table, out=out) is out
                assert torch.equal(out, expected)
                whole[1:51, 1:1 + view.shape[1], 3:67] = 7.0
                assert (whole == 7.0).all()
            for place in (wide[:, :, 3:67].clone(), wide[:, :4, :64].clone()):
                expected = rotary()(place, positions, table)
                assert rotary()(place, positions, table, out=place) is place
                assert torch.equal(place, expected)
    assert rotary()(wide[:0, :, :64], positions[:0], table).shape == (0, 6, 64)


def test_values_that_are_not_finite_stay_with_their_pair(gpu):
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    for interleaved in (False, True):
        x = torch.ones((2, 1, 48), device=gpu)
        x[0, 0, 3], x[0, 0, 40], x[1, 0, 47] = float("nan"), float("inf"), float("-inf")
        got = rotary()(x, torch.tensor([5, 6], dtype=torch.int32, device=gpu), prepare_rotary_table(32, interleaved=interleaved))
        wrong = (~torch.isfinite(got)).nonzero().tolist()
        assert wrong == [[0, 0, i] for i in ((2, 3, 40) if interleaved else (3, 19, 40))] + [[1, 0, 47]]


def test_refusals(gpu):
    from mambo_amd.utils.rotary_table import prepare_rotary_table
    x, at, table = torch.zeros((3, 2, 64), device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu), prepare_rotary_table(64)
    rotary()(x, at, table)
    for args, more in (((x.half(), at, table), {}), ((x[0], at, table), {}), ((x.cpu(), at, table), {}), ((x, at.long(), table), {}),
                       ((x, at[:2], table), {}), ((x, at.cpu(), table), {}), ((x, at, prepare_rotary_table(66)), {}),
                       ((torch.zeros((3, 1, 1026), device=gpu), at, table), {}), ((x, at, table), {"out_dtype": torch.float16}),
                       ((x, at, table), {"out": x.bfloat16()}), ((x, at, table), {"out": x[:2]}),
                       ((x, at, table), {"out": x[:1].expand(3, 2, 64)}), ((x[:, :0], at, table), {})):
        with pytest.raises(ValueError):
            rotary()(*args, **more)
    with pytest.raises(TypeError):
        rotary()(x, at, None)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,size", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotation_to_its_last_bits(gpu, tokens, heads, dim, size, interleaved, dtype):
    """Cosines and sines are rounded once from 64 bits: angles of 32 bits, which the bound of test_rotation allows, are further off."""
    from mambo_amd.utils.rotary_table import prepare_rotary_table, rotary_frequencies
    rng = np.random.default_rng(dim + size + 1)
    scaling = {"type": "yarn", "factor": 4.0, "original_length": 4096}
    x = torch.from_numpy(rng.standard_normal((tokens, heads, dim)).astype(np.float32)).to(gpu).to(dtype)
    positions = rng.integers(-1000, 100000, tokens).astype(np.int32)
    frequencies, magnitude = rotary_frequencies(size, scaling=scaling)
    got = rotary()(x, *ref.device(gpu, positions), prepare_rotary_table(size, scaling=scaling, interleaved=interleaved), out_dtype=torch.float32)
    x64 = x.double().cpu().numpy()
    off = np.abs(got.double().cpu().numpy() - ref.rotate(x64, positions, frequencies, interleaved, magnitude))
    assert (off <= ref.turn_bound(x64, positions, frequencies, interleaved, magnitude)).all()
