"""The attention block of a decoder layer out of the package's operators, for inference: IQ3_S projections,
rotary positions, the paged 8-bit cache and attention over it.

    q, k, v = x @ q.T, x @ k.T, x @ v.T          IQ3_S x MXFP8, one grouped launch
    cache <- k rotated, v; q rotated             one launch
    a = attention of q over the cached tokens
    out = a @ o.T                                IQ3_S x MXFP8

Nothing is read back to the host, so a decoding step can be recorded into a HIP graph, its lengths
counted on in it, and replayed token after token. The command builds a block of one of the sweep's models
with synthetic weights, takes a prompt for each user and then decodes, eagerly and from a graph, and prints one
JSON line:

    python -m mambo_amd.utils.attention_layer --model llama8b --users 4 --prompt 1000 --steps 20
"""

from __future__ import annotations

import argparse
import json
from dataclasses import dataclass

import torch

from mambo_amd.kernels.attention import launch_attention_kv
from mambo_amd.kernels.iq3_s_fp8 import launch_iq3_s_fp8_matmul, launch_iq3_s_fp8_matmul_grouped
from mambo_amd.kernels.kv_cache import launch_append_kv
from mambo_amd.kernels.quantize_fp8 import launch_quantize_fp8
from mambo_amd.utils.iq3_s_weight import IQ3SFields
from mambo_amd.utils.kv_cache import KVCache, allocate_kv_cache
from mambo_amd.utils.rotary_table import RotaryTable, prepare_rotary_table
from mambo_amd.utils.sweep import MODELS, layer_shapes, synth_weight

HEAD_DIM = 128  # of the sweep's models


@dataclass(frozen=True)
class AttentionLayer:
    """Prepared weights of a block: ``q`` [Hq D, K], ``k`` and ``v`` [H D, K], ``o`` [K, Hq D], the rotary
    angles and the window of the attention (0: none)."""

    q: IQ3SFields
    k: IQ3SFields
    v: IQ3SFields
    o: IQ3SFields
    rotary: RotaryTable
    window: int = 0

    def __call__(self, x: torch.Tensor, cache: KVCache, tables: torch.Tensor, lengths: torch.Tensor,
                 offsets: torch.Tensor | None = None) -> torch.Tensor:
        """The block's float32 output [T, K] of bfloat16 or float32 rows x [T, K], T of one and more, which are the last
        tokens of their sequences (launch_append_kv). Rows of no sequence come out as anything."""
        tokens, dim = x.shape[0], cache.head_dim
        q, k, v = launch_iq3_s_fp8_matmul_grouped(*launch_quantize_fp8(x), [self.q, self.k, self.v])
        heads = [t.view(tokens, -1, dim) for t in (q, k, v)]
        rotated = launch_append_kv(heads[1], heads[2], cache, tables, lengths, offsets=offsets, rotary=self.rotary, q=heads[0])
        a = launch_attention_kv(rotated, cache, tables, lengths, offsets=offsets, window=self.window)
        return launch_iq3_s_fp8_matmul(*launch_quantize_fp8(a.view(tokens, -1)), self.o)


def synthetic_layer(model: str, *, seed: int = 0, window: int = 0) -> tuple[AttentionLayer, int, int]:
    """A block of one of the sweep's models with synthetic weights on the current GPU, its key/value heads and its width."""
    shapes = {name: (n, k) for name, n, k, _ in layer_shapes(model)}
    weights = [synth_weight(*shapes[name], seed=1000 * seed + i) for i, name in enumerate(("q", "k", "v", "o"))]
    return AttentionLayer(*weights, prepare_rotary_table(HEAD_DIM, base=500000.0), window), shapes["k"][0] // HEAD_DIM, shapes["q"][1]


def main(argv: list[str] | None = None) -> int:
    parser = argparse.ArgumentParser(description="Run the attention block of a layer with synthetic weights.")
    parser.add_argument("--model", choices=sorted(MODELS), default="llama8b")
    parser.add_argument("--users", type=int, default=4)
    parser.add_argument("--prompt", type=int, default=1000, help="tokens of each user's prompt")
    parser.add_argument("--page-size", type=int, default=64)
    parser.add_argument("--window", type=int, default=0, help="last tokens that a token sees, 0: all")
    parser.add_argument("--steps", type=int, default=20, help="tokens decoded after the prompts")
    args = parser.parse_args(argv)
    if args.users < 1 or args.prompt < 1 or args.steps < 1:
        parser.error("--users, --prompt and --steps must be positive")
    layer, heads, width = synthetic_layer(args.model, window=args.window)
    columns = -(-(args.prompt + args.steps) // args.page_size)
    gen = torch.Generator(device="cuda").manual_seed(1)
    order = torch.randperm(args.users * columns, generator=gen, device="cuda").int()
    tables = order.view(args.users, columns)
    prompts = torch.randn((args.users * args.prompt, width), generator=gen, device="cuda").to(torch.bfloat16)
    tokens = torch.randn((args.steps, args.users, width), generator=gen, device="cuda").to(torch.bfloat16)

    def timed(run) -> float:
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        run()
        end.record()
        torch.cuda.synchronize()
        return 1e3 * start.elapsed_time(end)

    def fresh():
        cache = allocate_kv_cache(args.users * columns, heads, HEAD_DIM, page_size=args.page_size)
        return cache, torch.full((args.users,), args.prompt, dtype=torch.int32, device="cuda")

    def decode(cache, lengths):
        outs = []
        for i in range(args.steps):
            lengths.add_(1)
            outs.append(layer(tokens[i], cache, tables, lengths))
        return outs

    cache, lengths = fresh()
    layer(prompts, cache, tables, lengths)
    prompt_us = timed(lambda: layer(prompts, cache, tables, lengths))
    eager = decode(cache, lengths)
    lengths.fill_(args.prompt)  # the same tokens once more: what they overwrite is what they were
    eager_us = timed(lambda: decode(cache, lengths)) / args.steps

    cache, lengths = fresh()
    layer(prompts, cache, tables, lengths)
    row = torch.empty_like(tokens[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        lengths.add_(1)
        out = layer(row, cache, tables, lengths)
    torch.cuda.current_stream().wait_stream(side)
    replayed = []

    def replay():
        for i in range(args.steps):
            row.copy_(tokens[i])
            graph.replay()
            replayed.append(out.clone())

    graph_us = timed(replay) / args.steps
    same = all(torch.equal(a, b) for a, b in zip(eager, replayed))
    print(json.dumps({"block": {"model": args.model, "users": args.users, "prompt": args.prompt, "page_size": args.page_size,
                                "window": args.window, "steps": args.steps},
                      "prompt_us": round(prompt_us, 2), "eager_us": round(eager_us, 2), "graph_us": round(graph_us, 2),
                      "graph_equals_eager": same,
                      "output_rms": round(float(out.square().mean().sqrt()), 4)}))
    return 0 if same else 1


if __name__ == "__main__":
    raise SystemExit(main())
