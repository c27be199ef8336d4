"""Performance cases of the expert-layer operators: the router's plan, the products of 8-bit
floating-point weights with a scale for each block of 128, dense and grouped by expert, the IQ3_S
products grouped by expert, and the join of the experts' rows.

Kinds of case:

  dense    rows of bf16 or f32 are quantized in groups of 128 and multiplied by one weight
  experts  the tokens' rows (``gather``) or rows already in the experts' order are quantized and
           multiplied by the weight of the expert that each belongs to; ``weight`` is fp8 or iq3s
  route    router logits to the chosen experts, their weights and the plan of the products
  combine  the experts' rows weighted and added per token

``own`` false: the operators in elementary torch operations; true: the framework's kernels.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

# The 512 four-weight codes of the IQ3_S codebook, three hex digits each: level l of weight j
# in bits 3j..3j+2, magnitude 2l + 1.
GRID = (
    "00000100200500700800900a00c00e01001101501b02002202502702902b03003203903c03f04004104204404804904d"
    "05005305705905d06407107507a08008108508708808b08e09109509809c0a20a50a70a90ab0b80bb0c30c90cd0d00d2"
    "0d90db0de0e40e80ea0f70f90fd10010b10f11111411a12012312913814214415015215615b16116516717617b186189"
    "18b1991aa1b91c01c21c41d01d21d61db1e81ec20020120220420820920b20d20f21021221921c21e22c22e23123a240"
    "24124324624824c25125825b26126826a27827e28028a28d28f29029429a2a02a32ad2b02ba2c12c42c72c82cb2d12d7"
    "2d82dc2e12f22f830330530a30c31931b32232632832c34134834b35135835a3693903943973a43a63c13c33c83ca3d1"
    "3dd3e13f23f840040140340540740840a40c40e41141341741841a42142342542842a43743843b43d44044244844b44f"
    "45245545945c46246948148448749149349849f4a14ab4af4b94bc4c04c24c54c94d24d44d94db4e24e84f6501507510"
    "51351a51d52153a53d54454955255f56056b5785805825875915ad5b15c55c95d65d85e35e860260960b60d60f612619"
    "61b61d62262462762963363964164364564c65165366067067a67e68068a69069a69c6a86c16c86cc6d16d36d76d86e1"
    "6e36e76ed6fb70370970e71271972a73073474174874a75575a76476e77b78e7a17c17c37d07d27dd80080480a810814"
    "81781a82182883884284784984b85285885d86386986d88188388888d89189b8a08af8b28b88c48c98cb8d08d28d98dd"
    "90090291491f92093994594795197298b99c9b09c89cd9d89e39e9a02a08a0ca12a20a24a27a2aa36a3ca41a43a45a4a"
    "a51a5aa7aa80a89a93a98a9eaabac2ac7ac8ad7ae4ae9af5afbb01b04b10b1ab26b4ab56b69b6bba2bc2bc4bd2c09c0b"
    "c0dc19c1bc30c40c50c57c74c8ac9cca2cadcb2cb8cc0ccccd1ce0d15d23d32d40d43d5cd70d85da0dc9dcbe00e04e07"
    "e10e12e1ee20e2ce32e42e49e54e63e65e81e84e88e8ee91e98ea9ec2edaeddeebf01f05f0bf10f28f52f62f82f99fc0"
)


def listed() -> list[dict]:
    return [
        # one token through the smallest projection of a layer (k or v of the 8B model): latency
        {"name": "dense_m1", "kind": "dense", "m": 1, "n": 1024, "k": 4096, "dtype": "bf16"},
        # a prompt chunk of a size that divides nothing, rows that the caller holds in f32
        {"name": "dense_ragged", "kind": "dense", "m": 203, "n": 5003, "k": 2832, "dtype": "f32"},
        # a long prompt through the 8B model's gate projection
        {"name": "dense_m8192", "kind": "dense", "m": 8192, "n": 14336, "k": 4096, "dtype": "bf16"},
        # a serving batch of 16 tokens, 8 of 64 experts each: every weight is read for a row or two
        {"name": "experts_fp8_decode", "kind": "experts", "weight": "fp8", "m": 16, "experts": 64, "top_k": 8,
         "n": 2048, "k": 4096, "gather": True, "skew": 0.0},
        # prompt chunks through a few large experts, some of which get most of the tokens; the second product
        {"name": "experts_fp8_ragged", "kind": "experts", "weight": "fp8", "m": 301, "experts": 8, "top_k": 2,
         "n": 4096, "k": 7152, "gather": False, "skew": 1.0},
        # a long prompt over many experts
        {"name": "experts_fp8_m8192", "kind": "experts", "weight": "fp8", "m": 8192, "experts": 64, "top_k": 8,
         "n": 2048, "k": 4096, "gather": True, "skew": 0.5},
        # four users decode with experts of the 8B model's MLP shape
        {"name": "experts_iq3s_decode", "kind": "experts", "weight": "iq3s", "m": 4, "experts": 8, "top_k": 2,
         "n": 14336, "k": 4096, "gather": True, "skew": 0.0},
        # a prompt through the same experts' second product
        {"name": "experts_iq3s_m2048", "kind": "experts", "weight": "iq3s", "m": 2048, "experts": 8, "top_k": 2,
         "n": 4096, "k": 14336, "gather": False, "skew": 0.5},
        # the router of a decoding step and of a long prompt
        {"name": "route_m16", "kind": "route", "m": 16, "experts": 64, "top_k": 8, "dtype": "f32",
         "renormalize": True, "masked": 0.0},
        {"name": "route_m8192", "kind": "route", "m": 8192, "experts": 256, "top_k": 8, "dtype": "bf16",
         "renormalize": True, "masked": 0.1},
        # the join of the same
        {"name": "combine_m16", "kind": "combine", "m": 16, "top_k": 8, "n": 4096, "masked": 0.0},
        {"name": "combine_m8192", "kind": "combine", "m": 8192, "top_k": 8, "n": 4096, "masked": 0.1},
    ]


# What no drawn case exceeds: the largest listed multiply-adds, and weights that fit the card.
MOST_MNK = 8192 * 8 * 2048 * 4096
MOST_WEIGHTS = 64 * 2048 * 4096


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["dense", "dense", "experts", "experts", "experts", "experts", "route", "combine"])
    while True:
        if kind == "dense":
            case = {"kind": kind, "m": _log_int(rng, 1, 8192), "n": _log_int(rng, 64, 28672),
                    "k": 16 * _log_int(rng, 8, 1792), "dtype": rng.choice(["bf16", "f32"])}
            rows, weights = case["m"], case["n"] * case["k"]
        elif kind == "experts":
            experts = _log_int(rng, 2, 128)
            case = {"kind": kind, "weight": rng.choice(["fp8", "fp8", "iq3s"]), "m": _log_int(rng, 1, 8192),
                    "experts": experts, "top_k": rng.randint(1, min(8, experts)), "n": _log_int(rng, 64, 14336),
                    "gather": rng.random() < 0.5, "skew": rng.choice([0.0, 0.5, 1.0])}
            case["k"] = 256 * _log_int(rng, 1, 56) if case["weight"] == "iq3s" else 16 * _log_int(rng, 8, 896)
            rows, weights = case["m"] * case["top_k"], experts * case["n"] * case["k"]
            if rows > 65536 or rows * max(case["n"], case["k"]) > 65536 * 4096:
                continue
        elif kind == "route":
            experts = _log_int(rng, 2, 512)
            return {"kind": kind, "m": _log_int(rng, 1, 16384), "experts": experts,
                    "top_k": rng.randint(1, min(10, experts)), "dtype": rng.choice(["bf16", "f32"]),
                    "renormalize": rng.random() < 0.5, "masked": rng.choice([0.0, 0.1, 0.6])}
        else:
            case = {"kind": kind, "m": _log_int(rng, 1, 8192), "top_k": rng.randint(1, 8),
                    "n": _log_int(rng, 64, 8192), "masked": rng.choice([0.0, 0.1])}
            if case["m"] * case["top_k"] * case["n"] <= 8192 * 8 * 4096:
                return case
            continue
        if weights <= MOST_WEIGHTS and rows * case["n"] * case["k"] <= MOST_MNK:
            return case


# ------------------------------------------------------------------------------ inputs
def _generator(seed: int) -> torch.Generator:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    return gen


def _rows(m: int, k: int, dtype: torch.dtype, gen: torch.Generator) -> torch.Tensor:
    """Activations as a transformer has them: N(0, 1) with one value in a thousand 20 times as
    large."""
    x = torch.randn((m, k), generator=gen, device="cuda")
    big = torch.rand((m, k), generator=gen, device="cuda") < 1e-3
    return torch.where(big, 20.0 * x, x).to(dtype)


def _fp8_weight(experts: int, n: int, k: int, gen: torch.Generator):
    """E4M3 codes uint8 [E, N, K] and scales f32 [E, ceil(N/128), ceil(K/128)]."""
    codes = torch.empty((experts, n, k), dtype=torch.uint8, device="cuda")
    for e in range(experts):
        w = (100.0 * torch.randn((n, k), generator=gen, device="cuda")).clamp(-448.0, 448.0)
        codes[e] = w.to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.rand((experts, -(-n // 128), -(-k // 128)), generator=gen, device="cuda")
    return codes, (0.5 + scales) * 2e-4


def _raw(experts: int, n: int, k: int, gen: torch.Generator) -> torch.Tensor:
    """GGUF blocks uint8 [E, N, K/256, 110]: uniform codes, signs and scale nibbles, block scales
    in [0.002, 0.04]."""
    raw = torch.randint(0, 256, (experts, n, k // 256, 110), dtype=torch.uint8, generator=gen, device="cuda")
    d = 0.002 + 0.038 * torch.rand((experts, n, k // 256, 1), generator=gen, device="cuda")
    raw[..., :2] = d.to(torch.float16).view(torch.uint8)
    return raw


def _logits(case: dict, gen: torch.Generator) -> torch.Tensor:
    """Router logits; ``skew`` lets the first experts take more, ``masked`` is the share of experts
    that a token may not take (one token in 97, from the tenth on, may take none)."""
    m, experts = case["m"], case["experts"]
    rank = torch.arange(1, experts + 1, device="cuda", dtype=torch.float32)
    logits = 1.5 * torch.randn((m, experts), generator=gen, device="cuda") - 1.5 * case.get("skew", 0.0) * rank.log()
    if case.get("masked", 0.0):
        gone = torch.rand((m, experts), generator=gen, device="cuda") < case["masked"]
        gone |= (torch.arange(m, device="cuda") % 97 == 10)[:, None]
        logits = logits.masked_fill(gone, float("-inf"))
    return logits.to(DTYPES[case.get("dtype", "f32")])


def _make(case: dict, seed: int) -> dict:
    """A case's data, the same for every form of the operators."""
    gen, kind = _generator(seed), case["kind"]
    if kind == "route":
        return {"logits": _logits(case, gen)}
    m, n = case["m"], case["n"]
    if kind == "combine":
        made = {"y": torch.randn((m * case["top_k"], n), generator=gen, device="cuda").to(torch.bfloat16)}
        slots = torch.randperm(m * case["top_k"], generator=gen, device="cuda").to(torch.int32).view(m, -1)
        gone = torch.rand((m, case["top_k"]), generator=gen, device="cuda") < case["masked"]
        made["slots"] = slots.masked_fill(gone, -1)
        made["weights"] = torch.rand((m, case["top_k"]), generator=gen, device="cuda")
        return made
    k = case["k"]
    if kind == "dense":
        codes, scales = _fp8_weight(1, n, k, gen)
        return {"x": _rows(m, k, DTYPES[case["dtype"]], gen), "codes": codes[0], "scales": scales[0]}
    plan = _plan_of(_logits(case, gen).topk(case["top_k"]).indices, case["experts"])
    made = {"x": _rows(m if case["gather"] else m * case["top_k"], k, torch.bfloat16, gen), "offsets": plan[0],
            "rows": plan[1] if case["gather"] else None}
    if case["weight"] == "fp8":
        made["codes"], made["scales"] = _fp8_weight(case["experts"], n, k, gen)
    else:
        made["raw"] = _raw(case["experts"], n, k, gen)
    return made


def prepare(case: dict, seed: int) -> dict:
    state = {"case": dict(case), **_make(case, seed)}
    if case["kind"] == "experts":  # the plain form's slices of the rows
        state["counts"] = (state["offsets"][1:] - state["offsets"][:-1]).tolist()
    if own and case["kind"] in ("dense", "experts"):  # weights laid out once, as at a model's load
        if "raw" in state:
            from mambo_amd.utils.iq3_s_weight import prepare_iq3_s_experts
            state["prepared"] = prepare_iq3_s_experts(state.pop("raw"))
        else:
            from mambo_amd.utils.fp8_block_weight import prepare_fp8_block_weight
            state["prepared"] = prepare_fp8_block_weight(state.pop("codes"), state.pop("scales"))
    return state


# ------------------------------------------------------------------------------- a pass
def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state: dict):
    from mambo_amd.kernels import experts, fp8_block, quantize_fp8
    case = state["case"]
    kind = case["kind"]
    if kind == "route":
        plan = experts.launch_route_experts(state["logits"], case["top_k"], renormalize=case["renormalize"])
        return [plan.ids, plan.weights, plan.offsets, plan.rows, plan.slots]
    if kind == "combine":
        return experts.launch_combine_experts(state["y"], state["slots"], state["weights"], out_dtype=torch.bfloat16)
    if kind == "dense":
        values, scales = fp8_block.launch_quantize_fp8_block(state["x"])
        return fp8_block.launch_fp8_block_matmul(values, scales, state["prepared"], out_dtype=torch.bfloat16)
    if case["weight"] == "iq3s":
        values, scales = quantize_fp8.launch_quantize_fp8(state["x"])
        product = experts.launch_iq3_s_fp8_matmul_experts
    else:
        values, scales = fp8_block.launch_quantize_fp8_block(state["x"])
        product = experts.launch_fp8_block_matmul_experts
    return product(values, scales, state["prepared"], state["offsets"], rows=state["rows"], out_dtype=torch.bfloat16)


# ------------------------------------------------------------ the plain form, in 32 bits
def _groups(x: torch.Tensor, size: int) -> torch.Tensor:
    """[M, K] as [M, ceil(K/size), size], the last group filled with zeros."""
    m, k = x.shape
    return torch.nn.functional.pad(x, (0, -k % size)).view(m, -1, size)


def _dequantized_rows(x: torch.Tensor) -> torch.Tensor:
    """Groups of 128 with the scale amax / 448; x / scale as one division by amax, so that a value
    half way between two codes of a bf16 row stays there."""
    g = _groups(x.float(), 128)
    amax = g.abs().amax(-1, keepdim=True).clamp(min=448.0 * 2.0**-100)
    codes = (0.875 * g / (amax * 2.0**-9)).to(torch.float8_e4m3fn)
    return (codes.float() * (amax / 448.0)).flatten(1)[:, :x.shape[1]]


def _dequantized_mx_rows(x: torch.Tensor) -> torch.Tensor:
    """Groups of 32 with the scale 2^ceil(log2(amax / 448))."""
    g = _groups(x.float(), 32)
    mant, exp = torch.frexp(g.abs().amax(-1, keepdim=True))
    e = torch.where(mant <= 0.875, exp - 9, exp - 8)
    codes = torch.ldexp(g, -e).to(torch.float8_e4m3fn)
    return torch.ldexp(codes.float(), e).flatten(1)


def _dequantized_fp8(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    n, k = codes.shape
    s = scales.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return codes.view(torch.float8_e4m3fn).float() * s


_LEVELS: list[torch.Tensor] = []


def _levels() -> torch.Tensor:
    if not _LEVELS:
        codes = torch.tensor([int(GRID[i:i + 3], 16) for i in range(0, 1536, 3)], device="cuda")
        _LEVELS.append(2.0 * ((codes[:, None] >> torch.tensor([0, 3, 6, 9], device="cuda")) & 7).float() + 1.0)
    return _LEVELS[0]


def _dequantized_iq3s(raw: torch.Tensor) -> torch.Tensor:
    n, blocks, _ = raw.shape
    bits = torch.arange(8, device="cuda", dtype=torch.uint8)
    qh = (raw[..., 66:74, None] >> bits) & 1
    index = raw[..., 2:66].int() + 256 * qh.view(n, blocks, 64).int()
    sign = 1.0 - 2.0 * ((raw[..., 74:106, None] >> bits) & 1).float()
    d = raw[..., :2].contiguous().view(torch.float16).float()
    nibbles = torch.stack((raw[..., 106:110] & 15, raw[..., 106:110] >> 4), -1).view(n, blocks, 8)
    scale = d * (1.0 + 2.0 * nibbles.float())
    w = _levels()[index].view(n, blocks, 8, 32) * sign.view(n, blocks, 8, 32)
    return (w * scale[..., None]).view(n, -1)


def _plan_of(ids: torch.Tensor, experts: int):
    """Offsets of the experts' rows, the token of each row (-1: none) and the row of each choice."""
    m, top_k = ids.shape
    flat = torch.where(ids < 0, experts, ids).flatten().int()
    keys, order = torch.sort(flat, stable=True)
    offsets = torch.searchsorted(keys, torch.arange(experts + 1, device="cuda", dtype=torch.int32)).int()
    taken = keys < experts
    rows = torch.where(taken, torch.div(order, top_k, rounding_mode="floor"), -1).int()
    slots = torch.empty_like(flat)
    slots[order] = torch.where(taken, torch.arange(m * top_k, device="cuda"), -1).int()
    return offsets, rows, slots.view(m, top_k)


def _run_plain(state: dict):
    case = state["case"]
    kind = case["kind"]
    if kind == "route":
        logits = state["logits"].float()
        best, ids = torch.sort(logits, dim=1, descending=True, stable=True)
        best, ids = best[:, :case["top_k"]], ids[:, :case["top_k"]]
        p = torch.exp(best - best[:, :1])
        p = torch.where(best == float("-inf"), 0.0, p)
        total = p if case["renormalize"] else torch.exp(logits - best[:, :1])
        weights = torch.where(p > 0.0, p / total.sum(1, keepdim=True), 0.0)
        ids = torch.where(best == float("-inf"), -1, ids).int()
        return [ids, weights, *_plan_of(ids, case["experts"])]
    if kind == "combine":
        y = state["y"][state["slots"].clamp(min=0).long()].float()
        w = torch.where(state["slots"] < 0, 0.0, state["weights"])
        return (y * w[..., None]).sum(1).to(torch.bfloat16)
    if kind == "dense":
        w = _dequantized_fp8(state["codes"], state["scales"])
        return (_dequantized_rows(state["x"]) @ w.t()).to(torch.bfloat16)
    iq3s = case["weight"] == "iq3s"
    x = _dequantized_mx_rows(state["x"]) if iq3s else _dequantized_rows(state["x"])
    if state["rows"] is not None:
        x = x[state["rows"].long()]
    parts = []
    for e, part in enumerate(x.split(state["counts"])):  # each expert's rows; those without are left out
        if part.shape[0]:
            w = _dequantized_iq3s(state["raw"][e]) if iq3s else _dequantized_fp8(state["codes"][e], state["scales"][e])
            parts.append((part @ w.t()).to(torch.bfloat16))
    return torch.cat(parts)


# ------------------------------------------------------------------- what a pass has to do
def work(case: dict) -> dict:
    kind, m = case["kind"], case["m"]
    if kind == "route":
        size = DTYPES[case["dtype"]].itemsize
        return {"bytes": m * case["experts"] * size + m * case["top_k"] * 16 + 4 * case["experts"] + 4, "flops": 0}
    n = case["n"]
    if kind == "combine":
        return {"bytes": m * case["top_k"] * (2 * n + 8) + 2 * m * n, "flops": 2 * m * case["top_k"] * n}
    k = case["k"]
    if kind == "dense":
        size = DTYPES[case["dtype"]].itemsize
        return {"bytes": m * k * size + n * k * (1 + 4 / 128**2) + 2 * m * n, "flops": 2 * m * n * k}
    # experts that some row goes to, as the choices fall on average
    share = [r ** (-1.5 * case["skew"]) for r in range(1, case["experts"] + 1)]
    taken = sum(1.0 - (1.0 - min(1.0, case["top_k"] * s / sum(share))) ** m for s in share)
    per = 110 / 256 if case["weight"] == "iq3s" else 1 + 4 / 128**2
    rows = m * case["top_k"]
    return {"bytes": (m if case["gather"] else rows) * k * 2 + taken * n * k * per + rows * (2 * n + 4),
            "flops": 2 * rows * n * k}


# -------------------------------------------------- the definition in 64 bits, written apart
def _fp8_values() -> torch.Tensor:
    """The value of each E4M3 code."""
    code = torch.arange(256, device="cuda")
    e, f = ((code >> 3) & 15).double(), (code & 7).double()
    v = torch.where(e == 0, f / 512.0, (8.0 + f) * torch.exp2(e - 10.0))
    v = torch.where((code & 127) == 127, torch.nan, v)
    return torch.where(code >= 128, -v, v)


def _nearest_fp8(v: torch.Tensor) -> torch.Tensor:
    """Double values within +-448 (or less than half a step beyond) to the nearest E4M3 value, ties to even."""
    a = v.abs().clamp(min=2.0**-300)
    step = torch.exp2(torch.floor(torch.log2(a)).clamp(min=-6.0) - 3.0)
    return (v / step).round() * step


def _exact_rows(x: torch.Tensor, mx: bool) -> torch.Tensor:
    x = x.double()
    m, k = x.shape
    size = 32 if mx else 128
    padded = torch.zeros((m, -(-k // size) * size), dtype=torch.float64, device="cuda")
    padded[:, :k] = x
    g = padded.view(m, -1, size)
    amax = g.abs().amax(2).clamp(min=448.0 * 2.0**-100)[:, :, None]
    if mx:
        amax = 448.0 * torch.exp2(torch.ceil(torch.log2(amax / 448.0)))
    return (_nearest_fp8(448.0 * g / amax).clamp(-448.0, 448.0) * (amax / 448.0)).view(m, -1)[:, :k].contiguous()


def _exact_weight(made: dict, e: int) -> torch.Tensor:
    if "codes" in made:
        codes, scales = (made["codes"][e], made["scales"][e]) if made["codes"].ndim == 3 else (made["codes"], made["scales"])
        i = torch.arange(codes.shape[0], device="cuda") // 128
        j = torch.arange(codes.shape[1], device="cuda") // 128
        return _fp8_values()[codes.long()] * scales.double()[i][:, j]
    raw = made["raw"][e].long()
    n, blocks, _ = raw.shape
    at = torch.arange(256, device="cuda")  # of a block's weights
    code = raw[:, :, 2 + at // 4] + (((raw[:, :, 66 + at // 32] >> (at // 4 % 8)) & 1) << 8)
    words = torch.tensor([int(GRID[i:i + 3], 16) for i in range(0, 1536, 3)], device="cuda")
    w = 2.0 * ((words[code] >> (3 * (at % 4))) & 7).double() + 1.0
    w = torch.where(((raw[:, :, 74 + at // 8] >> (at % 8)) & 1) == 1, -w, w)
    nibble = (raw[:, :, 106 + at // 64] >> (4 * (at // 32 % 2))) & 15
    d = made["raw"][e][..., :2].contiguous().view(torch.float16).double()
    return (d * (2.0 * nibble.double() + 1.0) * w).view(n, -1)


def exact(case: dict, seed: int):
    made, kind = _make(case, seed), case["kind"]
    if kind == "route":
        logits = made["logits"].double()
        top = logits.topk(case["top_k"]).values
        some = torch.isfinite(top)
        e = torch.where(some, torch.exp(top - logits.amax(1, keepdim=True)), 0.0)
        all_e = torch.where(torch.isfinite(logits), torch.exp(logits - logits.amax(1, keepdim=True)), 0.0)
        total = (e if case["renormalize"] else all_e).sum(1, keepdim=True)
        return [None, torch.where(some, e / total, 0.0), None, None, None]
    if kind == "combine":
        out = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        for j in range(case["top_k"]):
            slot = made["slots"][:, j].long()
            w = torch.where(slot < 0, 0.0, made["weights"][:, j].double())
            out += w[:, None] * made["y"][slot.clamp(min=0)].double()
        return out
    x = _exact_rows(made["x"], mx="raw" in made)
    if kind == "dense":
        return x @ _exact_weight(made, 0).t().contiguous()
    out = torch.empty((case["m"] * case["top_k"], case["n"]), dtype=torch.float64, device="cuda")
    offsets = made["offsets"].tolist()
    for e in range(case["experts"]):
        lo, hi = offsets[e], offsets[e + 1]
        if hi > lo:
            rows = x[lo:hi] if made["rows"] is None else x[made["rows"][lo:hi].long()]
            out[lo:hi] = rows @ _exact_weight(made, e).t().contiguous()
    return out
