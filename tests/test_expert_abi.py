"""The expert-layer entry points of the C ABI without a GPU: sizes, and arguments that are refused
before the device is touched."""

from __future__ import annotations

import numpy as np
import pytest

import expert_reference as ref


@pytest.fixture(scope="module")
def lib():
    from mambo_amd import _native
    return _native.lib()


def refused(lib, rc, text):
    from mambo_amd import _native
    assert rc == _native.MAMBO_ERR_VALUE and text in lib.mambo_last_error().decode(), lib.mambo_last_error()


def test_packed_bytes(lib):
    assert lib.mambo_fp8_block_packed_bytes(1, 32, 128) == 4096
    assert lib.mambo_fp8_block_packed_bytes(3, 33, 144) == 3 * 2 * 2 * 4096
    for bad in ((0, 32, 128), (1, 0, 128), (1, 32, 0), (1025, 32, 128), (1, 32, 2**26 + 16), (1, 2**31, 16), (-1, 32, 128)):
        assert lib.mambo_fp8_block_packed_bytes(*bad) == 0


def test_quantizer_refusals(lib):
    f = lib.mambo_quantize_fp8_block
    refused(lib, f(16, 2, 1, 128, 128, 16, 128, 16, 1, 1, None), "float32 or bfloat16")
    refused(lib, f(16, 0, 1, 24, 24, 16, 24, 16, 1, 1, None), "multiple of 16")
    refused(lib, f(16, 0, -1, 32, 32, 16, 32, 16, 1, 1, None), "multiple of 16")
    refused(lib, f(16, 0, 2, 144, 144, 16, 144, 16, 1, 1, None), "strides must cover K")
    refused(lib, f(16, 0, 2, 144, 128, 16, 144, 16, 2, 1, None), "strides must cover K")
    refused(lib, f(None, 0, 1, 32, 32, 16, 32, 16, 1, 1, None), "null pointer")
    refused(lib, f(18, 0, 1, 32, 32, 16, 32, 16, 1, 1, None), "aligned to their type")
    assert f(None, 0, 0, 32, 32, None, 32, None, 1, 1, None) == 0


def test_pack_refusals(lib):
    f = lib.mambo_fp8_block_pack
    refused(lib, f(16, 1, 8, 24, 192, 24, 16, None), "multiple of 16")
    refused(lib, f(16, 1025, 8, 32, 256, 32, 16, None), "E in [1, 1024]")
    refused(lib, f(16, 1, 8, 2**26 + 16, 8 * (2**26 + 16), 2**26 + 16, 16, None), "up to 2^26")
    refused(lib, f(None, 1, 8, 32, 256, 32, 16, None), "null pointer")
    refused(lib, f(16, 1, 8, 32, 256, 32, 8, None), "16-byte aligned")


def test_product_refusals(lib):
    #      xv  ldxv xs ldxs gsxs m packed ws n k out dtype ldo stream
    good = [16, 32, 16, 1, 1, 2, 16, 16, 8, 32, 16, 0, 8, None]

    def call(**change):
        names = ["xv", "ldxv", "xs", "ldxs", "gsxs", "m", "packed", "ws", "n", "k", "out", "dtype", "ldo", "stream"]
        args = list(good)
        for name, value in change.items():
            args[names.index(name)] = value
        return lib.mambo_fp8_block_matmul(*args)

    for change, text in (({"dtype": 2}, "float32 or bfloat16"), ({"m": -1}, "negative"), ({"k": 40, "ldxv": 48}, "multiple of 16"),
                         ({"n": 0}, "multiple of 16"), ({"k": 2**26 + 16, "ldxv": 2**26 + 16}, "up to 2^26"), ({"ldxv": 16}, "must cover"), ({"ldxs": 0}, "must cover"), ({"gsxs": 0}, "must cover"),
                         ({"ldo": 7}, "must cover"), ({"xv": None}, "null pointer"), ({"out": None}, "null pointer"),
                         ({"xv": 8}, "16-byte aligned"), ({"ldxv": 40}, "16-byte aligned"), ({"packed": 24}, "16-byte aligned"),
                         ({"xs": 18}, "aligned to their type"), ({"out": 18}, "aligned to their type")):
        refused(lib, call(**change), text)
    assert call(m=0, xv=None, out=None) == 0


def test_expert_product_refusals(lib):
    f, q = lib.mambo_fp8_block_matmul_experts, lib.mambo_iq3s_fp8_matmul_experts
    for rows, r, offsets, experts, m, text in ((None, 3, 16, 2, 2, "a row of its own"), (16, -1, 16, 2, 2, "0 to 2^31"),
                                               (16, 2**31, 16, 2, 2, "0 to 2^31"), (16, 2, 16, 0, 2, "experts must be"),
                                               (16, 2, 16, 1025, 2, "experts must be"), (16, 2, None, 2, 2, "null pointer"),
                                               (16, 2, 16, 2, 0, "a row of its own")):
        text = text.replace("a row of its own", "an input row of its own")
        refused(lib, f(16, 32, 16, 1, 1, m, rows, r, offsets, experts, 16, 16, 8, 32, 16, 0, 8, None), text)
        refused(lib, q(16, 256, 16, 8, m, rows, r, offsets, experts, 16, 1760, 8, 1, 16, 0, 8, None), text)
    assert f(None, 32, None, 1, 1, 0, None, 0, None, 2, None, None, 8, 32, None, 0, 8, None) == 0
    assert q(None, 256, None, 8, 0, None, 0, None, 2, None, 1760, 8, 1, None, 0, 8, None) == 0
    for stride, xs, ldxs, text in ((1744, 16, 8, "expert_stride"), (1768, 16, 8, "expert_stride"), (1760, 12, 8, "aligned"),
                                   (1760, 16, 12, "aligned"), (1760, 16, 7, "must cover")):
        refused(lib, q(16, 256, xs, ldxs, 2, None, 2, 16, 2, 16, stride, 8, 1, 16, 0, 8, None), text)


def test_route_and_combine_refusals(lib):
    f, c = lib.mambo_route_experts, lib.mambo_combine_experts
    for dtype, ld, m, experts, top_k, logits, text in ((2, 8, 1, 8, 2, 16, "float32 or bfloat16"), (0, 7, 1, 8, 2, 16, "cover"),
                                                       (0, 8, -1, 8, 2, 16, "below 2^31"), (0, 8, 2**31, 8, 1, 16, "below 2^31"),
                                                       (0, 8, 2**30, 8, 2, 16, "below 2^31"), (0, 8, 1, 0, 1, 16, "experts must be"),
                                                       (0, 2000, 1, 1025, 2, 16, "experts must be"), (0, 8, 1, 8, 9, 16, "top_k"),
                                                       (0, 100, 1, 100, 65, 16, "top_k"), (0, 8, 1, 8, 0, 16, "top_k"),
                                                       (0, 8, 1, 8, 2, None, "null pointer")):
        refused(lib, f(logits, dtype, ld, m, experts, top_k, 1, 16, 16, 16, 16, 16, None), text)
    for y, yd, ldy, r, m, top_k, n, od, ldo, text in ((16, 2, 8, 4, 2, 2, 8, 0, 8, "float32 or bfloat16"),
                                                     (16, 0, 8, 4, 2, 2, 8, 3, 8, "float32 or bfloat16"),
                                                     (16, 0, 7, 4, 2, 2, 8, 0, 8, "must cover"), (16, 0, 8, 4, 2, 2, 8, 0, 7, "must cover"),
                                                     (16, 0, 8, 4, 2, 65, 8, 0, 8, "choices"), (16, 0, 8, -1, 2, 2, 8, 0, 8, "choices"),
                                                     (None, 0, 8, 4, 2, 2, 8, 0, 8, "null pointer"), (17, 1, 8, 4, 2, 2, 8, 0, 8, "aligned")):
        refused(lib, c(y, yd, ldy, r, 16, 16, m, top_k, n, 16, od, ldo, None), text)
    assert c(None, 0, 8, 0, None, None, 0, 2, 8, None, 0, 8, None) == 0


def test_python_refuses_without_a_gpu():
    import torch
    from mambo_amd.kernels import experts, fp8_block
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
    for call in (lambda: fp8_block.launch_quantize_fp8_block(torch.zeros((2, 32))),
                 lambda: prepare_fp8_block_weight(torch.zeros((2, 32), dtype=torch.uint8), torch.ones((1, 1))),
                 lambda: prepare_iq3_s_experts(torch.zeros((2, 2, 1, 110), dtype=torch.uint8)),
                 lambda: experts.launch_route_experts(torch.zeros((2, 4)), 2),
                 lambda: experts.launch_combine_experts(torch.zeros((2, 4)), torch.zeros((1, 1), dtype=torch.int32),
                                                        torch.zeros((1, 1)))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        fp8_block.launch_fp8_block_matmul(None, None, None)


def test_reference_plan_and_route_agree_with_hand_counts():
    """The statements that the GPU tests compare with, on cases small enough to see."""
    ids, weights = ref.route(np.array([[1.0, 3.0, 3.0, -np.inf], [-np.inf, np.nan, -np.inf, 2.0]]), 2, False)
    assert ids.tolist() == [[1, 2], [3, -1]]
    assert np.allclose(weights, [[1 / (2 + np.exp(-2))] * 2, [1.0, 0.0]])
    offsets, rows, slots = ref.plan(ids, 4)
    assert offsets.tolist() == [0, 0, 1, 2, 3] and rows.tolist() == [0, 0, 1, -1] and slots.tolist() == [[0, 1], [2, -1]]
    codes, scales = ref.quantize_block(np.array([[448.0, 1.0] + [0.0] * 14], dtype=np.float32))
    assert codes[0, :3].tolist() == [0x7E, 0x38, 0] and scales[0, 0] == 1.0
