"""Performance cases of the operators between a layer's q/k/v and o projections: rotary positions,
appending keys and values to a paged 8-bit cache with the rotation on the way, and attention over
that cache for prompts and for single tokens.

Kinds of case:

  rotary  queries or keys [T, H, D] rotated by their positions
  append  new tokens of ``seqs`` sequences go to the cache, rotated, and their queries are rotated
          with them; then the blocks that were written are read back as the values they stand for
  attend  queries of the last ``new`` tokens of each sequence over its cached keys and values

The cache holds E4M3 codes in blocks of 32 tokens of one head, keys and values each with a power of
two 2^e: e = max(ceil(log2(amax / 448)), -100). A block that grows a larger value has its older codes
brought to the new e. Sequences have pages of ``page`` tokens in any order.

``own`` false: the operators in elementary torch operations; true: the framework's kernels.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 32  # tokens that share a scale
LOWEST = -100  # lowest exponent of a scale

LLAMA3 = {"type": "llama3", "factor": 8.0, "low": 1.0, "high": 4.0, "length": 8192}
YARN = {"type": "yarn", "factor": 16.0, "fast": 32.0, "slow": 1.0, "length": 4096}
LINEAR = {"type": "linear", "factor": 4.0}
PLAIN = {"type": "none"}
SCALINGS = {"llama3": LLAMA3, "yarn": YARN, "linear": LINEAR, "none": PLAIN}


def listed() -> list[dict]:
    return [
        # one token of the 8B model, its queries and keys as the f32 projections leave them: latency
        {"name": "rotary_m1", "kind": "rotary", "tokens": 1, "heads": 40, "dim": 128, "rotary": 128, "base": 500000.0,
         "scaling": "llama3", "interleaved": False, "dtype": "f32", "far": 131072},
        # a long prompt's queries, half of each head rotated in neighbouring pairs, at positions up to a million
        {"name": "rotary_m8192", "kind": "rotary", "tokens": 8192, "heads": 32, "dim": 128, "rotary": 64,
         "base": 10000.0, "scaling": "yarn", "interleaved": True, "dtype": "bf16", "far": 1 << 20},
        # a decoding step of one user: the new token's key and value join a block that has older ones
        {"name": "append_m1", "kind": "append", "seqs": 1, "new": 1, "context": 1000, "ragged": 0.0, "kv_heads": 8,
         "group": 4, "dim": 128, "page": 64, "rotary": 128, "base": 500000.0, "scaling": "llama3",
         "interleaved": False, "dtype": "f32"},
        # pieces of prompts that start and end inside blocks, small heads of a size that fills no tile
        {"name": "append_ragged", "kind": "append", "seqs": 7, "new": 77, "context": 300, "ragged": 1.0, "kv_heads": 5,
         "group": 3, "dim": 80, "page": 32, "rotary": 40, "base": 10000.0, "scaling": "none", "interleaved": True,
         "dtype": "bf16"},
        # a long prompt of the 8B model
        {"name": "append_m8192", "kind": "append", "seqs": 1, "new": 8192, "context": 0, "ragged": 0.0, "kv_heads": 8,
         "group": 4, "dim": 128, "page": 64, "rotary": 128, "base": 500000.0, "scaling": "llama3",
         "interleaved": False, "dtype": "f32"},
        # one user decodes after a short prompt: latency
        {"name": "attend_m1", "kind": "attend", "seqs": 1, "new": 1, "context": 1000, "ragged": 0.0, "empty": False,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 64, "window": 0},
        # a serving batch of 64 users of the 8B model, of all lengths, some slots without a user
        {"name": "attend_batch", "kind": "attend", "seqs": 64, "new": 1, "context": 8192, "ragged": 1.0, "empty": True,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 64, "window": 0},
        # one user of the 70B model decodes at the end of a long document
        {"name": "attend_long", "kind": "attend", "seqs": 1, "new": 1, "context": 131149, "ragged": 0.0, "empty": False,
         "kv_heads": 8, "group": 8, "dim": 128, "page": 128, "window": 0},
        # drafts of five tokens checked at once, small heads, a sliding window
        {"name": "attend_draft", "kind": "attend", "seqs": 16, "new": 5, "context": 4000, "ragged": 0.3, "empty": False,
         "kv_heads": 4, "group": 6, "dim": 64, "page": 32, "window": 1000},
        # pieces of several prompts of any length behind what was cached of them
        {"name": "attend_ragged", "kind": "attend", "seqs": 6, "new": 700, "context": 1500, "ragged": 1.0, "empty": False,
         "kv_heads": 3, "group": 5, "dim": 96, "page": 32, "window": 0},
        # a piece of a prompt far into a long document of the 70B model
        {"name": "attend_chunk", "kind": "attend", "seqs": 1, "new": 512, "context": 32768, "ragged": 0.0, "empty": False,
         "kv_heads": 8, "group": 8, "dim": 128, "page": 128, "window": 0},
        # a long prompt of the 8B model
        {"name": "attend_m8192", "kind": "attend", "seqs": 1, "new": 8192, "context": 0, "ragged": 0.0, "empty": False,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 64, "window": 0},
    ]


# What no drawn case exceeds: the largest listed ones' scores, cached values and rows.
MOST_SCORES = 8192 * 8192 * 32
MOST_CACHED = 64 * 8192 * 8 * 128
MOST_ROWS = 8192 * 32 * 128


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["rotary", "append", "append", "attend", "attend", "attend", "attend"])
    while True:
        dim = 8 * rng.randint(4, 32) if rng.random() < 0.5 else rng.choice([64, 128])
        turned = {"rotary": 2 * rng.randint(4, dim // 2) if rng.random() < 0.5 else dim,
                  "base": rng.choice([10000.0, 500000.0, 1e6]), "scaling": rng.choice(sorted(SCALINGS)),
                  "interleaved": rng.random() < 0.5, "dtype": rng.choice(["bf16", "f32"])}
        if kind == "rotary":
            case = {"kind": kind, "tokens": _log_int(rng, 1, 8192), "heads": _log_int(rng, 1, 64), "dim": dim, **turned,
                    "far": _log_int(rng, 100, 1 << 20)}
            if case["tokens"] * case["heads"] * dim <= MOST_ROWS:
                return case
            continue
        case = {"kind": kind, "seqs": _log_int(rng, 1, 128), "new": 1, "context": _log_int(rng, 1, 131072),
                "ragged": rng.choice([0.0, 0.3, 1.0]), "kv_heads": rng.choice([1, 2, 3, 4, 5, 8, 8, 16, 32]),
                "group": rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), "dim": dim, "page": rng.choice([32, 64, 128, 256])}
        form = rng.choice(["token", "token", "draft", "prompt", "prompt"])
        if form == "draft":
            case["new"] = rng.randint(2, 16)
        elif form == "prompt":
            case["new"] = _log_int(rng, 17, 8192)
        if case["group"] * case["kv_heads"] > 64:
            continue
        new, length = _sizes(case)
        longest = max(length)
        if case["seqs"] * longest * case["kv_heads"] * dim > MOST_CACHED:
            continue
        if kind == "append":
            case |= turned
            if sum(new) * case["kv_heads"] * case["group"] * dim <= MOST_ROWS:
                return case
            continue
        case |= {"empty": rng.random() < 0.3, "window": rng.choice([0, 0, _log_int(rng, 1, 4096)])}
        heads = case["kv_heads"] * case["group"]
        if case["seqs"] * max(new) * heads * longest <= MOST_SCORES // 2 and sum(new) * heads * dim <= MOST_ROWS:
            return case


def _sizes(case: dict) -> tuple[list[int], list[int]]:
    """New tokens and length (new ones included) of each sequence. ``ragged`` 0: all alike; up to 1: spread
    between one and the largest, most of them short."""
    new, length = [], []
    for s in range(case["seqs"]):
        share = 1.0 if s == 0 else math.fmod(0.618033988749895 * s, 1.0)
        share = 1.0 - case["ragged"] + case["ragged"] * share**2
        n = case["new"] if case["new"] <= 16 else max(1, round(case["new"] * share))
        c = round(case["context"] * (1.0 - case["ragged"] + case["ragged"] * math.fmod(0.754877666246693 * s + share, 1.0)))
        if case.get("empty") and s % 13 == 5:  # a slot without a user
            n, c = (n if case["new"] <= 16 else 0), -case["new"]
        new.append(n)
        length.append(max(0, n + c))
    return new, length


# ------------------------------------------------------------------------------ inputs
def _generator(seed: int) -> torch.Generator:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    return gen


def _i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _spread(dim: int, gen: torch.Generator) -> torch.Tensor:
    """Sizes of a head's channels: of keys a few are several times as large as the others."""
    return 0.5 + torch.rand(dim, generator=gen, device="cuda") + 4.0 * (torch.rand(dim, generator=gen, device="cuda") < 0.03)


def _rows(tokens: int, heads: int, dim: int, gen: torch.Generator, spread=None) -> torch.Tensor:
    x = torch.randn((tokens, heads, dim), generator=gen, device="cuda")
    return x if spread is None else x * spread


def _make(case: dict, seed: int) -> dict:
    """A case's data, the same for every form of the operators: the cached tokens as bf16 rows in the
    sequences' order, where they lie (``tables``, ``lengths``, ``offsets``), and the new rows."""
    gen, dim = _generator(seed), case["dim"]
    if case["kind"] == "rotary":
        return {"x": _rows(case["tokens"], case["heads"], dim, gen).to(DTYPES[case["dtype"]]),
                "positions": torch.randint(0, case["far"], (case["tokens"],), generator=gen, device="cuda").int()}
    new, length = _sizes(case)
    order = torch.randperm(case["seqs"], generator=gen, device="cuda").tolist()
    new, length = [new[s] for s in order], [length[s] for s in order]
    page, heads = case["page"], case["kv_heads"]
    counts = [-(-n // page) for n in length]
    width, pages = max(counts) + 1, sum(counts) + 3
    shuffled = torch.randperm(pages, generator=gen, device="cuda").int()
    tables = torch.full((case["seqs"], width), -1, dtype=torch.int32, device="cuda")
    column = torch.arange(width, device="cuda")
    taken = column[None] < torch.tensor(counts, device="cuda")[:, None]
    tables[taken] = shuffled[:sum(counts)]
    append = case["kind"] == "append"
    cached = [max(0, n - m) for n, m in zip(length, new)] if append else length
    spread = _spread(dim, gen)
    made = {"new": new, "length": length, "cached": cached, "pages": pages, "tables": tables,
            "k": _rows(sum(cached), heads, dim, gen, spread).to(torch.bfloat16),
            "v": _rows(sum(cached), heads, dim, gen).to(torch.bfloat16)}
    tokens, q_heads = sum(new), heads * case["group"]
    if append:
        dtype = DTYPES[case["dtype"]]
        made |= {"new_k": (1.3 * _rows(tokens, heads, dim, gen, spread)).to(dtype),
                 "new_v": _rows(tokens, heads, dim, gen).to(dtype), "q": _rows(tokens, q_heads, dim, gen).to(dtype)}
        # the tokens of every block that is written
        first = [c // BLOCK * BLOCK for c in cached]
        made["sequences"] = torch.cat([torch.full((n - f,), s, dtype=torch.int32) for s, (f, n) in enumerate(zip(first, length))]).cuda()
        made["positions"] = torch.cat([torch.arange(f, n, dtype=torch.int32) for f, n in zip(first, length)]).cuda()
    else:
        made["q"] = (1.5 * _rows(tokens, q_heads, dim, gen) / spread).to(torch.bfloat16)
    return made


def _uniform(case: dict) -> bool:
    """Whether every sequence has the same number of new tokens, so that no offsets are needed."""
    return case["new"] <= 16 or case["seqs"] == 1


def _offsets(counts: list[int]) -> list[int]:
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _places(tables: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor, tokens: int, page: int):
    """Sequence, position and row of the cache (page * page size + place) of each new token."""
    row = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(offsets.long(), row, right=True) - 1
    position = lengths.long()[seq] - offsets.long()[seq + 1] + row
    return seq, position, tables.long()[seq, position // page] * page + position % page


def prepare(case: dict, seed: int) -> dict:
    made = _make(case, seed)
    state = {"case": dict(case)}
    if case["kind"] == "rotary":
        state |= made
    else:
        state |= {k: made[k] for k in ("tables", "q", "new_k", "new_v", "sequences", "positions") if k in made}
        state["lengths"], state["offsets"] = _i32(made["length"]), _i32(_offsets(made["new"]))
        cached = _i32(made["cached"])
        if own:
            from mambo_amd.kernels.kv_cache import launch_append_kv
            from mambo_amd.utils.kv_cache import allocate_kv_cache
            state["cache"] = allocate_kv_cache(made["pages"], case["kv_heads"], case["dim"], page_size=case["page"])
            launch_append_kv(made["k"], made["v"], state["cache"], made["tables"], cached,
                             offsets=_i32(_offsets(made["cached"])))
        else:
            _, _, place = _places(made["tables"], cached, _i32(_offsets(made["cached"])), sum(made["cached"]), case["page"])
            for name in ("k", "v"):
                rows = torch.zeros((made["pages"] * case["page"], case["kv_heads"], case["dim"]), device="cuda")
                rows[place] = made[name].float()
                e = _exponents(rows.view(-1, BLOCK, *rows.shape[1:]).abs().amax((1, 3)))
                state["e_" + name] = e  # of [blocks, heads]
                state["codes_" + name] = _codes(rows, e.repeat_interleave(BLOCK, 0))
    if own and "rotary" in case:
        from mambo_amd.utils.rotary_table import prepare_rotary_table
        scaling = SCALINGS[case["scaling"]]
        names = {"low": "low_freq_factor", "high": "high_freq_factor", "length": "original_length", "fast": "beta_fast",
                 "slow": "beta_slow"}
        state["table"] = prepare_rotary_table(
            case["rotary"], base=case["base"], interleaved=case["interleaved"],
            scaling=None if scaling is PLAIN else {names.get(k, k): v for k, v in scaling.items()})
    return state


# ------------------------------------------------------------------------------- a pass
def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state: dict):
    from mambo_amd.kernels import attention, kv_cache, rotary
    case = state["case"]
    if case["kind"] == "rotary":
        return rotary.launch_rotary(state["x"], state["positions"], state["table"], out_dtype=torch.bfloat16)
    offsets = None if _uniform(case) else state["offsets"]
    if case["kind"] == "append":
        q = kv_cache.launch_append_kv(state["new_k"], state["new_v"], state["cache"], state["tables"], state["lengths"],
                                      offsets=offsets, rotary=state["table"], q=state["q"])
        return [q, *kv_cache.launch_read_kv(state["cache"], state["tables"], state["sequences"], state["positions"])]
    return list(attention.launch_attention_kv(state["q"], state["cache"], state["tables"], state["lengths"],
                                              offsets=offsets, window=case["window"], return_lse=True))


# ------------------------------------------------------------ the plain form, in 32 bits
def _frequencies(case: dict) -> torch.Tensor:
    """Radians a position of each pair, in 64 bits."""
    size, scaling = case["rotary"], SCALINGS[case["scaling"]]
    f = case["base"] ** (-2.0 * torch.arange(size // 2, dtype=torch.float64, device="cuda") / size)
    if scaling["type"] == "linear":
        return f / scaling["factor"]
    if scaling["type"] == "llama3":
        turns = scaling["length"] * f / (2.0 * math.pi)
        keep = ((turns - scaling["low"]) / (scaling["high"] - scaling["low"])).clamp(0.0, 1.0)
        return f * (keep + (1.0 - keep) / scaling["factor"])
    if scaling["type"] == "yarn":
        edges = [size * math.log(scaling["length"] / (2.0 * math.pi * t)) / (2.0 * math.log(case["base"]))
                 for t in (scaling["fast"], scaling["slow"])]
        low, high = max(math.floor(edges[0]), 0), min(math.ceil(edges[1]), size - 1)
        ramp = ((torch.arange(size // 2, device="cuda") - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return f * (1.0 - ramp + ramp / scaling["factor"])
    return f


def _magnitude(case: dict) -> float:
    """What the scaling multiplies rotated values by."""
    scaling = SCALINGS[case["scaling"]]
    return 0.1 * math.log(scaling["factor"]) + 1.0 if scaling["type"] == "yarn" else 1.0


def _rotated(case: dict, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    angle = positions.double()[:, None] * _frequencies(case)
    cos = (_magnitude(case) * torch.cos(angle)).float()[:, None]
    sin = (_magnitude(case) * torch.sin(angle)).float()[:, None]
    x, size = x.float(), case["rotary"]
    turned, rest = x[..., :size], x[..., size:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, rest), -1)


def _exponents(amax: torch.Tensor) -> torch.Tensor:
    mant, exp = torch.frexp(amax)
    return torch.where(amax > 0.0, torch.where(mant <= 0.875, exp - 9, exp - 8), LOWEST).clamp(min=LOWEST)


def _codes(rows: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    """E4M3 codes of rows [.., heads, D] with the exponents e [.., heads]."""
    return torch.ldexp(rows, -e[..., None]).to(torch.float8_e4m3fn)


def _values(codes: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(codes.float(), e[..., None])


def _append_plain(state: dict, name: str, rows: torch.Tensor, place: torch.Tensor) -> None:
    codes, e = state["codes_" + name], state["e_" + name]
    block = place // BLOCK
    fresh = torch.zeros(e.shape[0], dtype=torch.bool, device="cuda")
    fresh[block[place % BLOCK == 0]] = True
    old = torch.where(fresh[:, None], LOWEST, e)
    largest = torch.zeros(e.shape, device="cuda").index_reduce_(0, block, rows.abs().amax(2), "amax")
    grown = torch.maximum(old, _exponents(largest))
    touched = torch.unique(block)
    kept = codes.view(-1, BLOCK, *codes.shape[1:])[touched]
    kept = _codes(_values(kept, e[touched][:, None]), grown[touched][:, None])
    codes.view(torch.uint8).view(-1, BLOCK, *codes.shape[1:])[touched] = kept.view(torch.uint8)
    e[touched] = grown[touched]
    codes.view(torch.uint8)[place] = _codes(rows, grown[block]).view(torch.uint8)


def _run_plain(state: dict):
    case = state["case"]
    if case["kind"] == "rotary":
        return _rotated(case, state["x"], state["positions"]).to(torch.bfloat16)
    tables, lengths, page = state["tables"], state["lengths"], case["page"]
    tokens = state["q"].shape[0]
    if case["kind"] == "append":
        _, position, place = _places(tables, lengths, state["offsets"], tokens, page)
        _append_plain(state, "k", _rotated(case, state["new_k"], position), place)
        _append_plain(state, "v", state["new_v"].float(), place)
        at = state["positions"].long()
        place = tables.long()[state["sequences"].long(), at // page] * page + at % page
        out = [_rotated(case, state["q"], position).to(torch.bfloat16)]
        for name in ("k", "v"):
            codes = state["codes_" + name].view(torch.uint8)[place].view(torch.float8_e4m3fn)
            out.append(_values(codes, state["e_" + name][place // BLOCK]).to(torch.bfloat16))
        return out
    return _attend_plain(state)


def _cached(state: dict, name: str) -> torch.Tensor:
    """Cached rows of every sequence, [S, heads, L, D]; zeros where there is no page."""
    case, tables = state["case"], state["tables"].long()
    page, shape = case["page"], (case["kv_heads"], case["dim"])
    at = tables.clamp(min=0)
    codes = state["codes_" + name].view(torch.uint8).view(-1, page, *shape)[at].view(torch.float8_e4m3fn)
    e = state["e_" + name].view(-1, page // BLOCK, shape[0])[at].repeat_interleave(BLOCK, 2)
    rows = torch.where((tables < 0)[..., None, None, None], 0.0, _values(codes, e))
    return rows.flatten(1, 2).transpose(1, 2).contiguous()


def _attend_plain(state: dict):
    case, lengths = state["case"], state["lengths"].long()
    seqs, heads, group, dim = case["seqs"], case["kv_heads"], case["group"], case["dim"]
    q, offsets = state["q"], state["offsets"].long()
    counts, most = offsets[1:] - offsets[:-1], case["new"]
    k, v = _cached(state, "k"), _cached(state, "v")
    # queries padded to the most that a sequence has, [S, heads, most * group, D]
    i = torch.arange(most, device="cuda")
    rows = (offsets[:-1, None] + i).clamp(max=q.shape[0] - 1)
    padded = q.float()[rows].view(seqs, most, heads, group, dim).transpose(1, 2).reshape(seqs, heads, most * group, dim)
    scores = (padded / math.sqrt(dim)) @ k.transpose(2, 3).contiguous()
    position = (lengths - counts)[:, None] + i  # [S, most]
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key <= position[..., None]) & (key < lengths[:, None, None])
    if case["window"]:
        seen &= key > position[..., None] - case["window"]
    scores = scores.view(seqs, heads, most, group, -1)
    scores.masked_fill_(~seen[:, None, :, None], float("-inf"))
    largest = scores.amax(-1, keepdim=True)
    base = torch.where(largest == float("-inf"), 0.0, largest)
    p = scores.sub_(base).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(seqs, heads, most * group, -1) @ v).view(seqs, heads, most, group, dim)
    out = torch.where(total > 0.0, out / total, 0.0)
    lse = torch.where(total > 0.0, base + total.log(), float("-inf"))[..., 0]
    # back to the tokens' rows
    row = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(offsets, row, right=True) - 1
    at = row - offsets[seq]
    out = out.permute(0, 2, 1, 3, 4)[seq, at].reshape(q.shape)
    return [out.to(torch.bfloat16), lse.permute(0, 2, 1, 3)[seq, at].reshape(q.shape[:2])]


# ------------------------------------------------------------------- what a pass has to do
def work(case: dict) -> dict:
    dim = case["dim"]
    if case["kind"] == "rotary":
        values = case["tokens"] * case["heads"] * dim
        return {"bytes": values * (DTYPES[case["dtype"]].itemsize + 2) + 4 * case["tokens"],
                "flops": 3 * case["tokens"] * case["heads"] * case["rotary"]}
    new, length = _sizes(case)
    heads, q_heads = case["kv_heads"], case["kv_heads"] * case["group"]
    if case["kind"] == "append":
        size, tokens = DTYPES[case["dtype"]].itemsize, sum(new)
        read = sum(n - max(0, n - m) // BLOCK * BLOCK for n, m in zip(length, new))
        return {"bytes": tokens * dim * (q_heads * (size + 2) + 2 * heads * (size + 1)) + 2 * read * heads * dim * 3,
                "flops": 3 * tokens * (q_heads + heads) * case["rotary"]}
    pairs = cached = 0
    for n, m in zip(length, new):
        first = max(0, n - m)  # position of the first query that has a key
        window = case["window"] or n
        cached += min(n, n - first - 1 + window)
        full = max(0, min(n, window) - first)  # queries that see all keys before them
        pairs += full * first + full * (full + 1) // 2 + (n - first - full) * window
    rows = sum(new) * q_heads
    return {"bytes": cached * heads * (2 * dim + 2 / BLOCK) + rows * (4 * dim + 4), "flops": 4 * dim * pairs * q_heads}


# -------------------------------------------------- the definition in 64 bits, written apart
def _nearest_fp8(v: torch.Tensor) -> torch.Tensor:
    """Double values within +-448 (or less than half a step beyond) to the nearest E4M3 value, ties to even."""
    a = v.abs().clamp(min=2.0**-300)
    step = torch.exp2(torch.floor(torch.log2(a)).clamp(min=-6.0) - 3.0)
    return (v / step).round() * step


def _exact_scale(amax: torch.Tensor) -> torch.Tensor:
    """2^e of a block."""
    return torch.exp2(torch.ceil(torch.log2(amax.clamp(min=448.0 * 2.0**LOWEST) / 448.0)))


def _exact_blocks(rows: torch.Tensor, old: int) -> torch.Tensor:
    """Rows [L, heads, D] of a sequence from a block's start as the cache holds them after the first
    ``old`` had been there (in blocks of their own scale) when the others came."""
    length = rows.shape[0]
    full = torch.zeros((-(-length // BLOCK) * BLOCK, *rows.shape[1:]), dtype=torch.float64, device="cuda")
    full[:length] = rows
    blocks = full.view(-1, BLOCK, *rows.shape[1:])
    scale = _exact_scale(blocks.abs().amax((1, 3)))[:, None, :, None]
    if old:  # what was there was rounded before
        before = torch.where(torch.arange(full.shape[0], device="cuda")[:, None, None] < old, full, 0.0).view(blocks.shape)
        s = _exact_scale(before.abs().amax((1, 3)))[:, None, :, None]
        held = _nearest_fp8(before / s) * s
        was = (torch.arange(full.shape[0], device="cuda") < old).view(-1, BLOCK, 1, 1)
        blocks = torch.where(was, held, blocks)
    return (_nearest_fp8(blocks / scale) * scale).view(full.shape)[:length]


def _exact_rotated(case: dict, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """As a product of complex numbers."""
    size, d = case["rotary"], case["scaling"]
    i = torch.arange(size // 2, dtype=torch.float64, device="cuda")
    f = torch.exp(-2.0 * i / size * math.log(case["base"]))
    magnitude = 1.0
    if d == "linear":
        f = f / LINEAR["factor"]
    elif d == "llama3":
        wave = 2.0 * math.pi / f
        blend = (LLAMA3["length"] / wave - LLAMA3["low"]) / (LLAMA3["high"] - LLAMA3["low"])
        f = torch.where(blend >= 1.0, f, torch.where(blend <= 0.0, f / LLAMA3["factor"],
                                                      (1.0 - blend) * f / LLAMA3["factor"] + blend * f))
    elif d == "yarn":
        def edge(turns):
            return size * math.log(YARN["length"] / (turns * 2.0 * math.pi)) / (2.0 * math.log(case["base"]))
        low, high = max(0, math.floor(edge(YARN["fast"]))), min(size - 1, math.ceil(edge(YARN["slow"])))
        far = torch.clamp((i - low) / max(0.001, high - low), 0.0, 1.0)
        f = (f / YARN["factor"]) * far + f * (1.0 - far)
        magnitude = 1.0 + 0.1 * math.log(YARN["factor"])
    turn = torch.polar(torch.full_like(f, magnitude).expand(len(positions), -1).contiguous(), positions.double()[:, None] * f)
    x = x.double()
    out = x.clone()
    pairs = (slice(0, size, 2), slice(1, size, 2)) if case["interleaved"] else (slice(0, size // 2), slice(size // 2, size))
    z = torch.complex(x[..., pairs[0]].contiguous(), x[..., pairs[1]].contiguous()) * turn[:, None]
    out[..., pairs[0]], out[..., pairs[1]] = z.real, z.imag
    return out


def exact(case: dict, seed: int):
    made = _make(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotated(case, made["x"], made["positions"])
    new, length, cached = made["new"], made["length"], _offsets(made["cached"])
    starts = _offsets(new)
    if case["kind"] == "append":
        position = torch.cat([torch.arange(n - m, n) for n, m in zip(length, new)]).cuda()
        k_new, v_new = _exact_rotated(case, made["new_k"], position), made["new_v"].double()
        keys, values = [], []
        for s, old in enumerate(made["cached"]):
            tail = slice(cached[s] + old // BLOCK * BLOCK, cached[s + 1])
            for out, was, rows in ((keys, made["k"], k_new), (values, made["v"], v_new)):
                out.append(_exact_blocks(torch.cat([was[tail].double(), rows[starts[s]:starts[s + 1]]]), old % BLOCK))
        return [_exact_rotated(case, made["q"], position), torch.cat(keys), torch.cat(values)]
    out = torch.zeros(made["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(made["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    group, scale = case["group"], case["dim"] ** -0.5
    for s, (m, n) in enumerate(zip(new, length)):
        if not m or not n:
            continue
        rows = slice(cached[s], cached[s + 1])
        k, v = _exact_blocks(made["k"][rows].double(), 0), _exact_blocks(made["v"][rows].double(), 0)
        at = torch.arange(n - m, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        hidden = (key > at) | (key <= at - (case["window"] or n + 1))
        for h in range(case["kv_heads"]):
            for g in range(h * group, (h + 1) * group):
                t = scale * (made["q"][starts[s]:starts[s + 1], g].double() @ k[:, h].t())
                t = t.masked_fill(hidden, -math.inf)
                some = torch.isfinite(t).any(1)
                z = torch.logsumexp(t, 1)
                p = torch.exp(t - torch.where(some, z, 0.0)[:, None])
                out[starts[s]:starts[s + 1], g] = p @ v[:, h]
                lse[starts[s]:starts[s + 1], g] = z
    return [out, lse]
