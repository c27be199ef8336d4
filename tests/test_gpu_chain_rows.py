"""A chained call whose rows all have to be copied first: every copy stays until the kernel has read it."""

from __future__ import annotations

import pytest
import torch

from conftest import make_synthetic_iq3_s

pytestmark = pytest.mark.gpu


def test_copied_rows_and_scales_stay(gpu):
    from mambo_amd.kernels import iq3_s_fp8 as ops
    from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
    from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_fields
    m, k, n = 2, 256, 300  # outputs larger than the copies, which would take their place
    w = prepare_iq3_s_fields(torch.from_numpy(make_synthetic_iq3_s(n, k, seed=1)).to(gpu), pack=True)
    launches, plain = [], []
    for i in range(8):
        values, scales = launch_quantize_fp8(torch.randn((m, k), device=gpu) * 4.0**i)
        wide = torch.zeros((m, k + 3), dtype=torch.uint8, device=gpu)[:, 1:k + 1]
        wide_scales = torch.zeros((m, k // 32 + 3), dtype=torch.uint8, device=gpu)[:, 1:k // 32 + 1]
        wide.copy_(values)
        wide_scales.copy_(scales)
        plain.append(ops.ChainLaunch(values, [w], scales))
        launches.append(ops.ChainLaunch(wide, [w], wide_scales))
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    for got, expected in zip(ops.launch_iq3_s_fp8_matmul_chain(launches), ops.launch_iq3_s_fp8_matmul_chain(plain)):
        assert torch.equal(got[0], expected[0])
