"""Plain 64-bit restatement of the window attention with sinks, of 4-bit rows and of the position
rotation (numpy; test infrastructure only).  The reference has none of them: the definitions are
those of the entry points' documentation."""

from __future__ import annotations

import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
EXPONENTS = {"bf16": (-125, 125), "fp16": (-23, 13)}
LARGEST = {"bf16": 2.0**127 * (2 - 2.0**-7), "fp16": 65504.0}


def visible(first: int, n: int, total: int, left, right, sinks: int) -> np.ndarray:
    """[n, total]: which keys the queries at positions first .. first + n - 1 see (None: no limit)"""
    seen = np.zeros((n, total), bool)
    for i in range(n):
        s = first + i
        for j in range(total):
            if right is not None and j > s + right:
                continue
            seen[i, j] = left is None or j >= s - left or j < sinks
    return seen


def attend(q, k, v, seen, scale: float):
    """(o, P) of one head: q [n, D], k and v [m, D]; a row that sees nothing is zero.  Keys that a
    row does not see have no part in it, whatever they hold."""
    n = q.shape[0]
    o, P = np.zeros((n, v.shape[1])), np.zeros((n, k.shape[0]))
    for i in range(n):
        j = np.nonzero(seen[i])[0]
        if j.size:
            z = (k[j] @ q[i]) * scale
            e = np.exp(z - z.max())
            P[i, j] = e / e.sum()
            o[i] = P[i, j] @ v[j]
    return o, P


def attend_backward(q, k, v, seen, scale: float, do):
    """(dq, dk, dv) of :func:`attend`"""
    o, P = attend(q, k, v, seen, scale)
    dS = P * (do @ v.T - (do * o).sum(1)[:, None]) * scale
    return dS @ k, dS.T @ q, P.T @ do


def rotate(x, cos, sin, interleaved: bool):
    """x [..., D] with angles [..., R / 2] of its rows"""
    y = np.array(x, np.float64)
    r = 2 * cos.shape[-1]
    ia, ib = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = y[..., ia].copy(), y[..., ib].copy()
    y[..., ia], y[..., ib] = a * cos - b * sin, a * sin + b * cos
    return y


def fp4_encode(x, dtype: str):
    """(codes [..., D / 2], scales [..., D / 32]) uint8 of rows x [..., D]"""
    lo, hi = EXPONENTS[dtype]
    x = np.array(x, np.float64)
    x = np.where(np.isnan(x), 0.0, np.clip(x, -LARGEST[dtype], LARGEST[dtype]))
    blocks = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    top = np.abs(blocks).max(-1)
    e = np.full(top.shape, lo)
    for k in range(lo, hi):
        e = np.where(top >= 7 * 2.0**k, k + 1, e)
    y = np.abs(blocks) * 2.0 ** -e[..., None].astype(np.float64)
    gap = np.abs(y[..., None] - MAGNITUDES)
    # the nearest; of two as near the one with the even code
    code = np.argmin(np.where(gap == gap.min(-1, keepdims=True), np.arange(8) % 2, 2), -1)
    code = (code + 8 * np.signbit(blocks)).astype(np.uint8).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).astype(np.uint8)


def fp4_values(codes, scales):
    code = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[:-1] + (2 * codes.shape[-1],))
    x = MAGNITUDES[code & 7] * np.where(code >= 8, -1.0, 1.0)
    return x * np.repeat(2.0 ** (scales.astype(np.float64) - 127), 32, -1)
