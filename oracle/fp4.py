"""CPU oracle of the 4-bit KV pool -- TEST INFRASTRUCTURE ONLY.

Float64 restatement of the format (blocks of 16 features, an e4m3 scale
s = e4m3(min(max|x| / 6, 448)), e2m1 codes of x / s, nearest with ties to even,
finite values only) and of attention over given keys and values, with the
quantities the tests' error bounds are made of.
"""

from __future__ import annotations

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_values() -> np.ndarray:
    """The 127 finite non-negative e4m3 values, ascending; index = code."""
    sub = [m / 8 * 2.0 ** -6 for m in range(8)]
    norm = [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    return np.array((sub + norm)[:127])


def _nearest(x: np.ndarray, vals: np.ndarray) -> np.ndarray:
    """Index of the nearest value, ties to the even index, past the end to the last."""
    mid = (vals[1:] + vals[:-1]) / 2
    i = np.searchsorted(mid, x, side="left")
    tie = np.zeros(x.shape, bool)
    inside = i < len(mid)
    tie[inside] = mid[i[inside]] == x[inside]
    return np.where(tie & (i % 2 == 1), i + 1, i)


def quantise(x: np.ndarray, g: float = 1.0):
    """x [..., D] -> (codes uint8 [..., D] with the sign in bit 3, scale codes uint8 [..., D/16])."""
    x = np.asarray(x, np.float64) / g
    x = np.where(np.isnan(x), 0.0, x)
    blk = x.reshape(*x.shape[:-1], -1, 16)
    sc = _nearest(np.minimum(np.abs(blk).max(-1) / 6, 448.0), e4m3_values())
    s = e4m3_values()[sc][..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        r = np.where(s > 0, np.minimum(np.abs(blk) / s, 6.0), 0.0)
    code = _nearest(r, LEVELS) + 8 * (np.signbit(blk) & (s > 0))
    return code.reshape(x.shape).astype(np.uint8), sc.astype(np.uint8)


def values(codes: np.ndarray, scales: np.ndarray, g: float = 1.0) -> np.ndarray:
    v = LEVELS[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    blk = v.reshape(*v.shape[:-1], -1, 16) * e4m3_values()[scales][..., None]
    return blk.reshape(v.shape) * g


def roundtrip(x: np.ndarray, g: float = 1.0) -> np.ndarray:
    return values(*quantise(x, g), g)


def row_bytes(Hkv: int, D: int) -> int:
    n = (Hkv * (D + D // 8) + 15) // 16 * 16
    return n + 16 if n % 128 == 0 else n


def pack_rows(k: np.ndarray, v: np.ndarray, g=(1.0, 1.0)) -> np.ndarray:
    """Pool rows uint8 [T, row_bytes] of k, v [T, Hkv, D]."""
    T, Hkv, D = k.shape
    rows = np.zeros((T, row_bytes(Hkv, D)), np.uint8)
    codes, scales = [], []
    for x, gg in ((k, g[0]), (v, g[1])):
        c, s = quantise(x, gg)
        codes.append(c[..., 0::2] | (c[..., 1::2] << 4))
        scales.append(s)
    n = Hkv * D
    rows[:, :n] = np.concatenate(codes, -1).reshape(T, n)
    rows[:, n: n + n // 8] = np.concatenate(scales, -1).reshape(T, n // 8)
    return rows


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float, first_limit: int):
    """Float64 attention of q [n, Hq, D] over k, v [L, Hkv, D]; row i sees keys 0 .. first_limit + i.

    Returns (out, A, X, S): A = softmax-weighted |v| (what an error relative to the weights scales
    with), X [n, Hq, 1] = the largest sum |q||k| * scale * log2(e) over a row's keys (what a
    rounding of the scores scales with), S = sum of |v| over a row's keys (what an absolute error
    of the weights scales with). A row without keys is zero.
    """
    n, Hq, D = q.shape
    L, Hkv, _ = k.shape
    G = Hq // Hkv
    out, A, X, S = np.zeros((n, Hq, D)), np.zeros((n, Hq, D)), np.zeros((n, Hq, 1)), np.zeros((n, Hq, D))
    for i in range(n):
        m = min(L, first_limit + i + 1)
        if m <= 0:
            continue
        for h in range(Hq):
            kk, vv = k[:m, h // G], v[:m, h // G]
            s = kk @ q[i, h] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h], A[i, h], S[i, h] = w @ vv, w @ np.abs(vv), np.abs(vv).sum(0)
            X[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * scale * np.log2(np.e)
    return out, A, X, S


def tolerance(ref: np.ndarray, A: np.ndarray, X: np.ndarray, S: np.ndarray, dtype: str, D: int,
              L: int) -> np.ndarray:
    """Bound of an attention output's error over exact 4-bit values, elementwise.

    Scores: D products summed in fp32 (a term each may be truncated, 2^-23), fp32 queries split
    into two fp16 parts (2^-22); an absolute error e of a base-2 score is a relative error
    ln2 * e of its weight. Weights: exp2 (2^-22) and their rounding to the operand type (fp16:
    2^-11; two parts: 2^-22). The weighted sum and the row sum add up to L terms in fp32 and
    both carry the weights' error. The output is rounded once. A weight below fp16's normal range
    is off by up to 2^-25 in absolute terms; the largest weight of a row is at least 2^7, and so is
    the row sum: 2^-32 of every |v|.
    """
    f32 = dtype == "float32"
    e_score = X * (D * 2.0 ** -23 + (2.0 ** -22 if f32 else 0.0) + 4 * 2.0 ** -24)
    e_weight = np.log(2) * e_score + 2.0 ** -22 + (2.0 ** -22 if f32 else 2.0 ** -11)
    e_sum = (L + 64) * 2.0 ** -23
    return A * (2 * e_weight + 2 * e_sum) + np.abs(ref) * (2.0 ** -24 if f32 else 2.0 ** -8) + S * 2.0 ** -32
