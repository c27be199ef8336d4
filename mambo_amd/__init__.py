"""mambo_amd: MI355X (gfx950) fused IQ3_S x MXFP8 projection path.

Operator API (mirrors the reference's mambo.kernels / mambo.utils modules):
    mambo_amd.kernels.quantize_fp8.launch_quantize_fp8
    mambo_amd.utils.iq3_s_weight.prepare_iq3_s_fields / IQ3SFields
    mambo_amd.kernels.iq3_s_fp8.launch_dequant_iq3_s / launch_iq3_s_fp8_matmul
    mambo_amd.utils.kernel_benchmark (autotuner / benchmark CLI)
Beyond the reference, a layer of experts (mambo_amd.utils.expert_layer puts them together):
    mambo_amd.kernels.fp8_block.launch_quantize_fp8_block / launch_fp8_block_matmul
    mambo_amd.kernels.experts.launch_route_experts / launch_fp8_block_matmul_experts /
        launch_iq3_s_fp8_matmul_experts / launch_combine_experts
    mambo_amd.utils.fp8_block_weight.prepare_fp8_block_weight, mambo_amd.utils.iq3_s_weight.prepare_iq3_s_experts
The kernels live in libmambo_hip.so (gfx950 HIP, C ABI in include/mambo_hip.h).
"""

__version__ = "0.1.0"
