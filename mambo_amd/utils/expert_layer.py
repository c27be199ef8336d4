"""A layer of experts out of the package's operators, for inference: the router, a gated MLP per
expert and the shared one, joined per token.

    logits = x @ router.T                           top-k experts of each token and their weights
    h = rows by expert of x @ gate_up[e].T          8-bit weights with a scale for each block of 128
    a = silu(h[:, :F]) * h[:, F:]
    y = a @ down[e].T                               8-bit weights, or IQ3_S
    out[t] = sum_j weight[t, j] * y[row of choice j] (+ the shared MLP of x[t])

Nothing is read back to the host between the router and the join, so a layer can be recorded into a
HIP graph. The command builds one with random weights, runs it eagerly and from a graph and prints
one JSON line:

    python -m mambo_amd.utils.expert_layer --tokens 16 --experts 64 --top-k 8 --hidden 4096 --ffn 2048
    python -m mambo_amd.utils.expert_layer --tokens 4 --experts 8 --top-k 2 --down iq3s
"""

from __future__ import annotations

import argparse
import json
from dataclasses import dataclass

import torch

from mambo_amd.kernels.experts import (launch_combine_experts, launch_fp8_block_matmul_experts,
                                       launch_iq3_s_fp8_matmul_experts, launch_route_experts)
from mambo_amd.kernels.fp8_block import launch_fp8_block_matmul, launch_quantize_fp8_block
from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
from mambo_amd.utils.fp8_block_weight import Fp8BlockWeight, prepare_fp8_block_weight
from mambo_amd.utils.iq3_s_weight import IQ3SExperts, prepare_iq3_s_experts


def silu_mul(h: torch.Tensor) -> torch.Tensor:
    """silu of the first half of each row times the second, each rounded to the rows' type: of bfloat16
    2^-8, beside the 2^-4 of the 8-bit codes that the next product makes of it."""
    gate, up = h.chunk(2, dim=1)
    return torch.nn.functional.silu(gate) * up


@dataclass(frozen=True)
class ExpertLayer:
    """Prepared weights of a layer: ``router`` [E, H] of the activations' type, ``gate_up`` [E, 2F, H],
    ``down`` [E, H, F] (8-bit or IQ3_S), and the shared MLP's ``shared_gate_up`` [2S, H] and
    ``shared_down`` [H, S], or None."""

    router: torch.Tensor
    top_k: int
    gate_up: Fp8BlockWeight
    down: Fp8BlockWeight | IQ3SExperts
    shared_gate_up: Fp8BlockWeight | None = None
    shared_down: Fp8BlockWeight | None = None
    renormalize: bool = True

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        """The layer's output [M, H] of bfloat16 rows x [M, H]. The joined rows and the shared MLP's are rounded to
        bfloat16 each and then added (2^-8 of either; float32 ones would be read and written at twice
        the bytes)."""
        dtype = torch.bfloat16
        if x.shape[0] == 0:  # launch_quantize_fp8 takes one row and more
            return torch.empty((0, self.down.n), dtype=dtype, device=x.device)
        plan = launch_route_experts(x @ self.router.t(), self.top_k, renormalize=self.renormalize)
        values, scales = launch_quantize_fp8_block(x)  # a token's row once, however many experts read it
        h = launch_fp8_block_matmul_experts(values, scales, self.gate_up, plan.offsets, rows=plan.rows, out_dtype=dtype)
        a = silu_mul(h)
        if isinstance(self.down, IQ3SExperts):
            y = launch_iq3_s_fp8_matmul_experts(*launch_quantize_fp8(a), self.down, plan.offsets, out_dtype=dtype)
        else:
            y = launch_fp8_block_matmul_experts(*launch_quantize_fp8_block(a), self.down, plan.offsets, out_dtype=dtype)
        out = launch_combine_experts(y, plan.slots, plan.weights)
        if self.shared_gate_up is not None:
            h = launch_fp8_block_matmul(values, scales, self.shared_gate_up, out_dtype=dtype)
            out += launch_fp8_block_matmul(*launch_quantize_fp8_block(silu_mul(h)), self.shared_down, out_dtype=dtype)
        return out


def random_fp8_weight(shape: tuple[int, ...], generator: torch.Generator):
    """E4M3 codes of all values but NaN, uint8 [.., N, K], and block scales float32 [.., ceil(N/128),
    ceil(K/128)] that keep the spread of a row's sums near that of a row of N(0, 1)."""
    *experts, n, k = shape
    codes = torch.randint(0, 256, shape, generator=generator, dtype=torch.uint8, device=generator.device)
    codes = torch.where((codes & 127) == 127, 0, codes)
    scales = torch.rand((*experts, -(-n // 128), -(-k // 128)), generator=generator, device=generator.device)
    return codes, (0.5 + scales) / (110.0 * k**0.5)  # 110: root mean square of the codes' values


def random_layer(hidden: int, ffn: int, experts: int, top_k: int, *, down: str = "fp8", shared: int = 0,
                 seed: int = 0) -> ExpertLayer:
    """A layer of random weights on the current GPU."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    router = (torch.randn((experts, hidden), generator=gen, device="cuda") / hidden**0.5).to(torch.bfloat16)
    gate_up = prepare_fp8_block_weight(*random_fp8_weight((experts, 2 * ffn, hidden), gen))
    if down == "iq3s":
        if ffn % 256:
            raise ValueError("IQ3_S weights need --ffn to be a multiple of 256")
        raw = torch.randint(0, 256, (experts, hidden, ffn // 256, 110), generator=gen, dtype=torch.uint8, device="cuda")
        # the block's fp16 d: the codes reach 15 times a scale of up to 31
        raw[..., :2] = torch.tensor([1.0 / (140.0 * ffn**0.5)], dtype=torch.float16, device="cuda").view(torch.uint8)
        prepared = prepare_iq3_s_experts(raw)
    else:
        prepared = prepare_fp8_block_weight(*random_fp8_weight((experts, hidden, ffn), gen))
    more = {}
    if shared:
        more = {"shared_gate_up": prepare_fp8_block_weight(*random_fp8_weight((2 * shared, hidden), gen)),
                "shared_down": prepare_fp8_block_weight(*random_fp8_weight((hidden, shared), gen))}
    return ExpertLayer(router, top_k, gate_up, prepared, **more)


def main(argv: list[str] | None = None) -> int:
    parser = argparse.ArgumentParser(description="Run one layer of experts with random weights.")
    parser.add_argument("--tokens", type=int, default=16)
    parser.add_argument("--experts", type=int, default=64)
    parser.add_argument("--top-k", type=int, default=8)
    parser.add_argument("--hidden", type=int, default=4096)
    parser.add_argument("--ffn", type=int, default=2048)
    parser.add_argument("--shared", type=int, default=2048, help="width of the shared MLP, 0: none")
    parser.add_argument("--down", choices=("fp8", "iq3s"), default="fp8")
    parser.add_argument("--steps", type=int, default=20)
    args = parser.parse_args(argv)
    layer = random_layer(args.hidden, args.ffn, args.experts, args.top_k, down=args.down, shared=args.shared)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((args.tokens, args.hidden), generator=gen, device="cuda").to(torch.bfloat16)
    eager = layer(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = layer(x)
    torch.cuda.current_stream().wait_stream(side)
    graph.replay()
    same = torch.equal(out, eager)
    times = {}
    for name, step in (("eager", lambda: layer(x)), ("graph", graph.replay)):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(args.steps):
            step()
        end.record()
        torch.cuda.synchronize()
        times[name] = round(1e3 * start.elapsed_time(end) / args.steps, 2)
    print(json.dumps({"layer": {"tokens": args.tokens, "experts": args.experts, "top_k": args.top_k,
                                "hidden": args.hidden, "ffn": args.ffn, "shared": args.shared, "down": args.down},
                      "eager_us": times["eager"], "graph_us": times["graph"], "graph_equals_eager": same,
                      "output_rms": round(float(out.float().square().mean().sqrt()), 4)}))
    return 0 if same else 1


if __name__ == "__main__":
    raise SystemExit(main())
