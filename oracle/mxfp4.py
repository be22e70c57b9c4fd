"""MXFP4 in 64 bits (OCP Microscaling Formats): the quantiser, the values codes
stand for, and the products with bounds on what fp32 sums may differ by."""

from __future__ import annotations

import numpy as np

BLOCK = 32
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BF16_HALF_STEP = 2.0 ** -8  # relative, of one rounding to bf16
F32_HALF_STEP = 2.0 ** -24


def scale_codes(amax: np.ndarray) -> np.ndarray:
    """e8m0 codes of blocks with largest magnitude ``amax`` (float64)."""
    finite = np.isfinite(amax)
    _, exponent = np.frexp(np.where(finite, amax, 1.0))  # amax = m 2^exponent, 1/2 <= m < 1
    code = np.where(amax > 0, np.clip(exponent - 3, -127, 127) + 127, 0)
    return np.where(finite, code, 255).astype(np.int64)


def nearest(v: np.ndarray) -> np.ndarray:
    """Index of the grid value nearest to each magnitude, ties to the even index."""
    distance = np.abs(np.abs(v)[..., None] - GRID)
    best = distance.min(-1, keepdims=True)
    ties = distance == best
    even = np.where(ties, np.arange(8) % 2 * 8 + np.arange(8), 99)
    return even.argmin(-1)


def quantize(x: np.ndarray):
    """float64 [..., K] -> (codes uint8 [..., K / 2], scale codes uint8 [..., K / 32])."""
    v = x.reshape(*x.shape[:-1], -1, BLOCK)
    with np.errstate(invalid="ignore"):
        amax = np.where(np.isnan(v).any(-1), np.nan, np.abs(v).max(-1))
    scale = scale_codes(amax)
    finite = scale != 255
    scaled = np.where(finite[..., None], v, 0.0) / np.exp2(np.where(finite, scale, 127) - 127.0)[..., None]
    code = nearest(scaled) | (np.signbit(scaled).astype(np.int64) << 3)
    code = code.reshape(x.shape)
    return (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), scale.astype(np.uint8)


def dequantize(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    nibbles = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    value = np.where(nibbles & 8, -1.0, 1.0) * GRID[nibbles & 7]
    scale = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return value * np.repeat(scale, BLOCK, -1)


def product(a: np.ndarray, w: np.ndarray):
    """a [T, K] @ w [N, K]^T and a bound on an fp32 evaluation's error: every
    one of the K exact products enters at most K rounded sums."""
    y = a @ w.T
    return y, 2.0 * F32_HALF_STEP * a.shape[1] * (np.abs(a) @ np.abs(w).T)


def requantize(v: np.ndarray, error: np.ndarray):
    """MXFP4 values of v [T, K], and how far those of any v' with |v' - v| <=
    error can be from them: an element moves to the neighbouring code where its
    error reaches a border, a whole block to the other scale where its
    maximum's does."""
    def values(x, scale):
        s = np.exp2(scale - 127.0)[..., None]
        b = x.reshape(*scale.shape, BLOCK) / s
        return np.where(b < 0, -1.0, 1.0) * GRID[nearest(b)] * s

    blocks, err = v.reshape(len(v), -1, BLOCK), error.reshape(len(v), -1, BLOCK)
    mag = np.abs(blocks)
    centre = scale_codes(mag.max(-1))
    best = values(v, centre)
    low, high = scale_codes(np.maximum(mag - err, 0).max(-1)), scale_codes((mag + err).max(-1))
    worst = np.zeros_like(best)
    for scale in (low, centre, high):
        for x in (v - error, v, v + error):
            worst = np.maximum(worst, np.abs(values(x, scale) - best))
    return best.reshape(v.shape), worst.reshape(v.shape)


def moe(x, ids, weights, w13, w2):
    """Routed SwiGLU experts on dequantised weights w13 [E, 2I, H], w2 [E, H,
    I]; x the bf16 rows as float64.  Returns (out, bound): float64 results and
    how far an fp32 evaluation rounded to bf16 may be from them."""
    rows = dequantize(*quantize(x))
    out, bound = np.zeros((len(x), w2.shape[1])), np.zeros((len(x), w2.shape[1]))
    inter = w2.shape[2]
    for t in range(len(x)):
        for r in range(ids.shape[1]):
            e = int(ids[t, r])
            if not 0 <= e < len(w13):
                continue
            both, err = product(rows[t:t + 1], w13[e])
            g, u, ge, ue = both[:, :inter], both[:, inter:], err[:, :inter], err[:, inter:]
            sig = 1.0 / (1.0 + np.exp(-g))
            act = g * sig * u
            # silu's slope is below 1.1; the sigmoid is within 4 half steps,
            # the two products within one each
            act_err = 1.1 * ge * (np.abs(u) + ue) + np.abs(g * sig) * ue + 8 * F32_HALF_STEP * np.abs(act)
            a, a_err = requantize(act, act_err)
            y, y_err = product(a, w2[e])
            y_err = y_err * 1.01 + a_err @ np.abs(w2[e]).T
            w = float(weights[t, r])
            out[t] += w * y[0]
            bound[t] += np.abs(w) * (y_err[0] + 2 * ids.shape[1] * F32_HALF_STEP * np.abs(y[0]))
    return out, bound + BF16_HALF_STEP * (np.abs(out) + bound)
