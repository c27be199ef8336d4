"""Plain statements, in 64 bits on the CPU, of what the expert-layer operators compute, and inputs for
their tests. Written from the definitions; nothing of the package is used."""

from __future__ import annotations

import numpy as np
import torch

from conftest import e4m3_encode_bruteforce, e4m3_values

VALUES = e4m3_values()


def quantize_block(x: np.ndarray):
    """(codes uint8 [M,K], scales float32 [M,G]) of float32 rows, bit for bit: the quotient is a float32
    division, which the kernel's must equal."""
    m, k = x.shape
    g = -(-k // 128)
    padded = np.zeros((m, g * 128), dtype=np.float32)
    padded[:, :k] = x
    parts = padded.reshape(m, g, 128)
    amax = np.maximum(np.abs(parts).max(2, keepdims=True), np.float32(448.0 * 2.0**-100))
    quotient = (np.float32(0.875) * parts) / (amax * np.float32(2.0**-9))
    codes = e4m3_encode_bruteforce(quotient).reshape(m, -1)[:, :k]
    return codes, (amax[..., 0] / np.float32(448.0)).astype(np.float32)


def dequantize(codes: np.ndarray, scales: np.ndarray, rows_per_scale: int) -> np.ndarray:
    """Codes [R,K] times the scales [ceil(R/rows_per_scale), ceil(K/128)], float64."""
    s = scales.astype(np.float64).repeat(rows_per_scale, 0)[:codes.shape[0]].repeat(128, 1)[:, :codes.shape[1]]
    return VALUES[codes] * s


def product(xv, xs, wv, ws):
    """(sums, sums of magnitudes) float64 [M,N]."""
    x, w = dequantize(xv, xs, 1), dequantize(wv, ws, 128)
    return x @ w.T, np.abs(x) @ np.abs(w).T


def bound(magnitudes: np.ndarray, k: int, values: np.ndarray, dtype) -> np.ndarray:
    """How far float32 sums of k products, in any order and each addition off by at most one unit of
    its last place (a matrix instruction may cut instead of round), can be from the exact ones: k
    additions, two scalings of each group and one rounding of the result to its type."""
    units = (k + 4 + 2 * (-(-k // 128))) * 2.0**-23 * magnitudes + 1e-37
    return units + (np.abs(values) + units) * 2.0**-8 if dtype == torch.bfloat16 else units


def random_codes(rng, shape) -> np.ndarray:
    """E4M3 codes of all exponents, no NaN."""
    codes = rng.integers(0, 256, size=shape, dtype=np.uint8)
    return np.where((codes & 127) == 127, 0, codes).astype(np.uint8)


def integer_codes(rng, shape) -> np.ndarray:
    """Codes of the integers -8 .. 8: products with scales of powers of two add up without rounding."""
    v = rng.integers(-8, 9, size=shape)
    return e4m3_encode_bruteforce(v.astype(np.float64)).reshape(shape)


def plan(ids: np.ndarray, experts: int):
    """(offsets, rows, slots) of chosen experts [M, top_k], -1 where a token has none."""
    m, top_k = ids.shape
    rows, slots, offsets = [], np.full((m, top_k), -1, dtype=np.int32), [0]
    for e in range(experts):
        for t in range(m):
            for j in range(top_k):
                if ids[t, j] == e:
                    slots[t, j] = len(rows)
                    rows.append(t)
        offsets.append(len(rows))
    rows += [-1] * (m * top_k - len(rows))
    return np.array(offsets, dtype=np.int32), np.array(rows, dtype=np.int32), slots


def route(logits: np.ndarray, top_k: int, renormalize: bool):
    """(ids int32, weights float64) of float64 logits [M,E]."""
    m, experts = logits.shape
    ids, weights = np.full((m, top_k), -1, dtype=np.int32), np.zeros((m, top_k))
    for t in range(m):
        left = [e for e in range(experts) if logits[t, e] > -np.inf]  # NaN compares false
        left.sort(key=lambda e: (-logits[t, e], e))
        if not left:
            continue
        top = logits[t, left[0]]
        term = {e: 1.0 if logits[t, e] == top else float(np.exp(logits[t, e] - top)) for e in left}
        chosen = left[:top_k]
        total = sum(term[e] for e in (chosen if renormalize else left))
        ids[t, :len(chosen)] = chosen
        weights[t, :len(chosen)] = [term[e] / total for e in chosen]
    return ids, weights


def some_offsets(rng, rows: int, experts: int, unrouted: int = 0) -> np.ndarray:
    """Offsets of rows spread unevenly over the experts, most of which get none where there are few."""
    share = rng.random(experts) ** 3
    share[rng.random(experts) < 0.3] = 0.0
    share[rng.integers(experts)] += 0.1
    cuts = np.floor(np.concatenate([[0.0], np.cumsum(share)]) / share.sum() * (rows - unrouted) + 1e-9)
    return cuts.astype(np.int32)
