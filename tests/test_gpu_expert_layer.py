"""The layer of experts (mambo_amd.utils.expert_layer) against the same layer in 64 bits, and its
command."""

from __future__ import annotations

import json

import numpy as np
import pytest
import torch

import expert_reference as ref
from conftest import make_synthetic_iq3_s
from oracle import oracle

pytestmark = pytest.mark.gpu


def bf16(a: np.ndarray) -> np.ndarray:
    return torch.from_numpy(a).to(torch.bfloat16).double().numpy()


def quantized(x: np.ndarray) -> np.ndarray:
    """Rows as their 8-bit codes hold them, float64."""
    return ref.dequantize(*ref.quantize_block(x.astype(np.float32)), 1)


def gated(h: np.ndarray, width: int) -> np.ndarray:
    gate, up = bf16(h)[:, :width], bf16(h)[:, width:]
    return bf16(bf16(gate / (1.0 + np.exp(-gate))) * up)


@pytest.mark.parametrize("down", ["fp8", "iq3s"])
@pytest.mark.parametrize("m,experts,top_k,hidden,ffn,shared", [(1, 4, 2, 256, 256, 0), (7, 9, 3, 400, 256, 144),
                                                               (50, 6, 2, 272, 512, 272)])
def test_layer(gpu, m, experts, top_k, hidden, ffn, shared, down):
    """Both sides round the rows to 8 bits alike and the sums to bf16; a sum that lies near the middle
    of two bf16 values may round to either, one part in 2^8 of it, and a code of a row that follows
    it then too, one part in 2^3. Fewer than one sum in ten can differ (their error is below 2^-4 of
    the distance of two values), of which one in 2^4 moves a code: a row's 2-norm is off by less than
    sqrt(0.1 / 16) / 8 = 1% of the experts' terms, and by 2^-8 for the last rounding."""
    from mambo_amd.utils.expert_layer import ExpertLayer
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
    rng = np.random.default_rng(m)

    def weight(*shape):
        *e, n, k = shape
        scales = (0.5 + rng.random((*e, -(-n // 128), -(-k // 128)))).astype(np.float32) / np.float32(110 * k**0.5)
        codes = ref.random_codes(rng, shape)
        packed = prepare_fp8_block_weight(torch.from_numpy(codes).to(gpu), torch.from_numpy(scales).to(gpu))
        flat = [ref.dequantize(c, s, 128) for c, s in zip(codes.reshape(-1, n, k), scales.reshape(-1, *scales.shape[-2:]))]
        return packed, flat

    # logits that are whole numbers: the bf16 product of the router is exact, ties included
    router = torch.zeros((experts, hidden), dtype=torch.bfloat16)
    router[torch.arange(experts), torch.arange(experts)] = 1.0
    x = torch.from_numpy(rng.standard_normal((m, hidden)).astype(np.float32)).to(torch.bfloat16)
    gate_up, gate_up64 = weight(experts, 2 * ffn, hidden)
    if down == "iq3s":
        raws = np.stack([make_synthetic_iq3_s(hidden, ffn, seed=e) for e in range(experts)])
        packed = prepare_iq3_s_experts(torch.from_numpy(raws).to(gpu))
    else:
        packed, down64 = weight(experts, hidden, ffn)
    more, shared64 = {}, None
    if shared:
        (a, a64), (b, b64) = weight(2 * shared, hidden), weight(hidden, shared)
        more, shared64 = {"shared_gate_up": a, "shared_down": b}, (a64[0], b64[0])
    layer = ExpertLayer(router.to(gpu), top_k, gate_up, packed, **more)
    out = layer(x.to(gpu)).double().cpu().numpy()

    x64 = x.double().numpy()
    ids, weights = ref.route(x64[:, :experts], top_k, True)
    rows = quantized(x64)
    expected = np.zeros((m, hidden))
    for t in range(m):
        for e, w in zip(ids[t], weights[t]):
            act = gated(rows[t:t + 1] @ gate_up64[e].T, ffn)
            if down == "iq3s":
                y = oracle.iq3s_fp8_matmul(*oracle.quantize_mxfp8(act.astype(np.float32)), raws[e])[0].astype(np.float64)
            else:
                y = (quantized(act) @ down64[e].T)[0]
            expected[t] += w * bf16(y)
    if shared:
        expected += quantized(gated(rows @ shared64[0].T, shared)) @ shared64[1].T
    for t in range(m):
        assert np.linalg.norm(out[t] - expected[t]) <= 0.02 * np.linalg.norm(expected[t]), t


def test_command(gpu, capsys):
    from mambo_amd.utils import expert_layer
    for extra in ([], ["--down", "iq3s", "--shared", "0"]):
        assert expert_layer.main(["--tokens", "5", "--experts", "6", "--top-k", "2", "--hidden", "512", "--ffn", "256",
                                  "--steps", "2", "--shared", "256", *extra]) == 0
        line = json.loads(capsys.readouterr().out)
        assert line["graph_equals_eager"] and line["graph_us"] > 0 and 0.01 < line["output_rms"] < 100


def test_named_stream(gpu):
    """Every operator on a stream that is not the current one, after work of that stream: what they
    allocate and copy (strided rows, scales) belongs to it."""
    from mambo_amd.kernels.experts import (launch_combine_experts, launch_fp8_block_matmul_experts,
                                           launch_iq3_s_fp8_matmul_experts, launch_route_experts)
    from mambo_amd.kernels.fp8_block import launch_quantize_fp8_block
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
    rng = np.random.default_rng(21)
    side = torch.cuda.Stream()
    codes = torch.from_numpy(ref.random_codes(rng, (4, 512, 256))).to(gpu)
    scales = torch.rand((4, 4, 2), device=gpu) * 1e-3
    raws = torch.from_numpy(np.stack([make_synthetic_iq3_s(96, 512, seed=e) for e in range(4)])).to(gpu)

    def layer(x, logits, stream):
        with torch.cuda.stream(stream):  # the inputs are ready on the stream alone
            x, logits = x * 2.0, logits * 2.0
        s = None if stream == torch.cuda.current_stream() else stream
        up, down = prepare_fp8_block_weight(codes, scales, stream=s), prepare_iq3_s_experts(raws, stream=s)
        plan = launch_route_experts(logits, 2, stream=s)
        values, row_scales = launch_quantize_fp8_block(x, stream=s)
        h = launch_fp8_block_matmul_experts(values, row_scales, up, plan.offsets, rows=plan.rows, stream=s)
        mx = launch_quantize_fp8(h, stream=s)
        y = launch_iq3_s_fp8_matmul_experts(*mx, down, plan.offsets, stream=s)
        return launch_combine_experts(y, plan.slots, plan.weights, stream=s)

    for seed in range(3):
        gen = torch.Generator(device=gpu).manual_seed(seed)
        x, logits = torch.randn((90, 256), generator=gen, device=gpu), torch.randn((90, 4), generator=gen, device=gpu)
        expected = layer(x, logits, torch.cuda.current_stream())
        side.wait_stream(torch.cuda.current_stream())
        out = layer(x, logits, side)
        side.synchronize()
        assert torch.equal(out, expected) and bool(out.any())
