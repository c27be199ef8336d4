"""Plain statements, in 64 bits on the CPU, of rotary positions, the paged 8-bit cache and attention over
it, and sequences to try them on. Written from the definitions; nothing of the package is used."""

from __future__ import annotations

import math

import numpy as np
import torch

from conftest import e4m3_encode_bruteforce, e4m3_values

VALUES = e4m3_values()
BLOCK, LOWEST = 32, -100


def rotate(x: np.ndarray, positions, frequencies, interleaved: bool, magnitude: float = 1.0) -> np.ndarray:
    """x [T,H,D] rotated in float64."""
    out = np.array(x, dtype=np.float64)
    size = 2 * len(frequencies)
    for t, p in enumerate(positions):
        for i, f in enumerate(frequencies):
            c, s = magnitude * math.cos(p * f), magnitude * math.sin(p * f)
            i0, i1 = (2 * i, 2 * i + 1) if interleaved else (i, i + size // 2)
            a, b = np.array(x[t, :, i0], dtype=np.float64), np.array(x[t, :, i1], dtype=np.float64)
            out[t, :, i0], out[t, :, i1] = a * c - b * s, a * s + b * c
    return out


def rotation_bound(x: np.ndarray, size: int, interleaved: bool, magnitude: float = 1.0) -> np.ndarray:
    """How far float32 rotations can be: the angle is off by 2^-24 of up to pi and by 2^-32 of a turn, the
    sine and cosine by four units, their product with the magnitude, the two products and the sum by half a unit each."""
    a = np.abs(np.array(x, dtype=np.float64))
    out = np.zeros_like(a)
    half = size // 2
    pairs = [(2 * i, 2 * i + 1) if interleaved else (i, i + half) for i in range(half)]
    for i, j in pairs:
        out[..., i] = out[..., j] = magnitude * (a[..., i] + a[..., j]) * 12 * 2.0**-24
    return out


def exponent(amax: float) -> int:
    """max(ceil(log2(amax / 448)), -100), exactly."""
    if amax == 0.0:
        return LOWEST
    mant, exp = math.frexp(amax)
    return max(LOWEST, exp - 9 if mant <= 0.875 else exp - 8)


def nearest(x: np.ndarray, e: int) -> np.ndarray:
    """E4M3(x 2^-e) 2^e, no more than 240 * 2^120."""
    if e >= 120:
        x = np.clip(x, -240 * 2.0**120, 240 * 2.0**120)
    return (VALUES[e4m3_encode_bruteforce(np.ldexp(x, -e))] * 2.0**e).reshape(np.shape(x))


class Model:
    """What the cache holds of one sequence: values [L,H,D] and exponents of blocks, keys and values apart."""

    def __init__(self, heads: int, dim: int):
        self.heads, self.dim = heads, dim
        self.k, self.v = np.zeros((0, heads, dim)), np.zeros((0, heads, dim))
        self.e = {}  # (block, head, "k" or "v")

    def append(self, k: np.ndarray, v: np.ndarray, start: int) -> None:
        """Tokens start .. of rows k, v [n,H,D] (float64 of what the kernel is given, rotated); what was at or
        behind start is overwritten or forgotten."""
        n = k.shape[0]
        for name, rows in (("k", k), ("v", v)):
            old = getattr(self, name)[:start]
            new = np.concatenate([old, np.zeros((n, self.heads, self.dim))])
            for block in range(start // BLOCK, -(-(start + n) // BLOCK)):
                lo, hi = max(start, block * BLOCK), min(start + n, (block + 1) * BLOCK)
                for h in range(self.heads):
                    part, mate = rows[lo - start:hi - start, h], (v if name == "k" else k)[lo - start:hi - start, h]
                    bad = ~(np.isfinite(part).all(1) & np.isfinite(mate).all(1))
                    e = exponent(float(np.abs(part[~bad]).max(initial=0.0)))
                    if lo > block * BLOCK:
                        before = self.e.get((block, h, name), LOWEST)
                        if e > before:
                            held = new[block * BLOCK:lo, h]
                            new[block * BLOCK:lo, h] = np.where(np.isnan(held), held, nearest(np.nan_to_num(held), e))
                        e = max(e, before)
                    self.e[block, h, name] = e
                    stored = nearest(np.where(bad[:, None], 0.0, part), e)
                    if name == "k":
                        stored[bad] = np.nan
                    new[lo:hi, h] = stored
            setattr(self, name, new)


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, group: int, scale: float, causal: bool, window: int, left_out=None):
    """(out, lse, bound of out's error, bound of lse's) of a sequence's rows q [n,Hq,D] over its cached k, v [L,H,D].
    ``left_out``: tokens that no page is for.

    float32 scores of D products, each addition off by a unit of its last place (a matrix instruction may cut), and
    scaled; exponentials off by a few units more; probabilities rounded to bfloat16 (half a step: 2^-8), sums in
    float32, the result rounded to bfloat16."""
    n, heads, dim = q.shape
    length = k.shape[0]
    out, lse = np.zeros(q.shape), np.full((n, heads), -np.inf)
    bound, lse_bound = np.zeros(q.shape), np.zeros((n, heads))
    token = np.arange(length)
    unit = 2.0**-23
    for i in range(n):
        position = length - n + i
        seen = token <= position if causal else token < length
        if window:
            seen = seen & (token > position - window)
        if left_out is not None:
            seen = seen & ~left_out
        if not seen.any():
            continue
        for h in range(heads):
            kk, vv = k[seen, h // group], v[seen, h // group]
            s = scale * (kk @ q[i, h])
            delta = (dim + 8) * unit * float((scale * (np.abs(kk) @ np.abs(q[i, h]))).max(initial=0.0)) + 8 * unit * float(np.abs(s).max())
            top = s.max()
            p = np.exp(s - top)
            total = p.sum()
            p /= total
            out[i, h], lse[i, h] = p @ vv, top + math.log(total)
            spread = p @ np.abs(vv)
            sums = (len(s) + 64) * unit
            bound[i, h] = spread * (2 * math.expm1(delta + 8 * unit) + 2.0**-8 + sums) + np.abs(out[i, h]) * 2.0**-8 + 1e-30
            lse_bound[i, h] = 2 * delta + sums + 8 * unit * (1.0 + abs(lse[i, h]))
    return out, lse, bound, lse_bound


def turn_bound(x: np.ndarray, positions, frequencies, interleaved: bool, magnitude: float = 1.0) -> np.ndarray:
    """How far a rotation in float32 by cosines and sines that are rounded once from 64 bits can be: half a unit of each, of the
    one product that is rounded by itself and of the sum, counted at the values that they have; of the angle what 53 bits of the
    frequency, here and there, leave at the position, and the ends of the two series (below 2^-36)."""
    x = np.array(x, dtype=np.float64)
    out = np.zeros_like(x)
    half, p = 2.0**-24, np.array(positions, dtype=np.float64)
    size = 2 * len(frequencies)
    for i, f in enumerate(frequencies):
        i0, i1 = (2 * i, 2 * i + 1) if interleaved else (i, i + size // 2)
        c, s = (magnitude * t(p * f)[:, None] for t in (np.cos, np.sin))
        a, b = x[:, :, i0], x[:, :, i1]
        far = magnitude * (np.abs(a) + np.abs(b)) * (2.0**-36 + np.abs(p) * abs(f) * 2.0**-51)[:, None]
        out[:, :, i0] = 1.001 * half * (np.abs(a * c) + 2 * np.abs(b * s) + np.abs(a * c - b * s)) + far
        out[:, :, i1] = 1.001 * half * (np.abs(a * s) + 2 * np.abs(b * c) + np.abs(a * s + b * c)) + far
    return out


# Keys and values by which every block of a long sequence shows in the results. Scores are 0 or, for two kinds of queries, 0 or 2
# times ln 2 by the block, so that probabilities are 1 and 4 to each other, and a block's values are 1 in one column of each half
# of the head and 0 elsewhere: sums are of small whole numbers, which float32 and the rounding to bfloat16 keep.
def block_rows(rng, length: int, heads: int, dim: int):
    """(keys, values) [L,H,D], exactly held by the cache."""
    k = rng.uniform(-3.0, 3.0, (length, heads, dim)).astype(np.float32)
    v = np.zeros((length, heads, dim), dtype=np.float32)
    block, half = np.arange(length) // BLOCK, dim // 2
    run = -(-(length // BLOCK + 1) // (dim - half))
    for h in range(heads):
        k[:, h, 0], k[:, h, 1] = 2 * ((5 * block + h) % 7 < 3), 2 * ((3 * block + h) % 5 < 2)
        v[np.arange(length), h, (block + h) % half] = 1
        v[np.arange(length), h, half + block // run] = 1
    return k, v


def block_queries(n: int, heads: int, dim: int) -> np.ndarray:
    """Rows [n,Hq,D] for them, to be scaled by ln 2: of kind (row + head) % 3, 0 for scores of 0."""
    q = np.zeros((n, heads, dim), dtype=np.float32)
    kind = (np.arange(n)[:, None] + np.arange(heads)) % 3
    q[..., 0], q[..., 1] = kind == 1, kind == 2
    return q


def block_attend(k: np.ndarray, v: np.ndarray, n: int, group: int, causal: bool, window: int):
    """(out, lse, bound of out's error, bound of lse's) of such rows over such tokens.

    Probabilities 1 are exact, their sums whole: what is left is the division and the product (half a unit each) and half a step of
    bfloat16, and of lse the logarithm (a unit), its factor and the product. Those of 4 are off by the scale's and the exponential's
    last bits, and the total by half a unit for each of up to a quarter of the tokens that a lane adds up."""
    length, heads, dim = k.shape
    out, lse = np.zeros((n, heads * group, dim)), np.full((n, heads * group), -np.inf)
    bound, lse_bound = np.zeros(out.shape), np.zeros(lse.shape)
    end = length - n + np.arange(n) + 1
    to = np.clip(end, 0, length) if causal else np.full(n, length)
    begin = np.clip(end - window, 0, to) if window else np.zeros(n, dtype=np.int64)
    for h in range(heads):
        for kind in range(3):
            w = np.ones(length) if kind == 0 else 2.0 ** k[:, h, kind - 1].astype(np.float64)
            weights = np.concatenate([[0.0], np.cumsum(w)])
            sums = np.concatenate([np.zeros((1, dim)), np.cumsum(w[:, None] * v[:, h], axis=0)])
            loose = 2.0**-22 if kind == 0 else 2.0**-20 + (length // 4 + 64) * 2.0**-24
            for g in range(h * group, (h + 1) * group):
                rows = np.flatnonzero(((np.arange(n) + g) % 3 == kind) & (to > begin))
                total = (weights[to[rows]] - weights[begin[rows]])[:, None]
                out[rows, g] = (sums[to[rows]] - sums[begin[rows]]) / total
                lse[rows, g] = np.log(total[:, 0])
                bound[rows, g] = out[rows, g] * (2.0**-8 + loose)
                lse_bound[rows, g] = 2.0**-22 * (1 + lse[rows, g]) + (loose if kind else 0.0)
    return out, lse, bound, lse_bound


def tables_of(rng, lengths, page: int, *, spare: int = 2, extra: int = 1):
    """(tables int32 [S,C], pages of the pool): every sequence's pages in any order, -1 behind them."""
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    order = rng.permutation(pages).astype(np.int32)
    tables = np.full((len(lengths), max(counts) + extra), -1, dtype=np.int32)
    at = 0
    for s, c in enumerate(counts):
        tables[s, :c] = order[at:at + c]
        at += c
    return tables, pages


def offsets_of(counts) -> np.ndarray:
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def device(gpu, *arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).to(gpu) for a in arrays]
