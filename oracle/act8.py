"""Oracle of the 8-bit activation checkpoints (humaniflow_amd/act8.py): the definitions in float64 on the CPU, one block at a time.

A block = 32 consecutive rows of one column.  top = its largest finite magnitude; step = 2^e with e the smallest integer, at least -126, for which top / step
rounds to at most 127; code = top-relative value x / step rounded to nearest even; a value that is not finite has no code and comes back as NaN.
"""
import math

import numpy as np

BLOCK = 32


def step_exponent(top):
    if not top > 0:
        return -126
    e = math.frexp(top)[1] - 7                       # top = m 2^k, 0.5 <= m < 1: top / 2^(k - 7) in [64, 128)
    if top / 2.0 ** e >= 127.5:
        e += 1
    return min(max(e, -126), 121)                    # exponent byte in [7, 254]


def pack(x):
    """x (M, C) float64 (values of the input's own type) -> (codes int8, exponents e int (ceil(M / 32), C))."""
    x = np.asarray(x, np.float64)
    M, C = x.shape
    nb = (M + BLOCK - 1) // BLOCK
    codes = np.zeros((M, C), np.int8)
    exps = np.zeros((nb, C), np.int64)
    for t in range(nb):
        rows = x[t * BLOCK:(t + 1) * BLOCK]
        fine = np.isfinite(rows)
        tops = np.where(fine, np.abs(np.where(fine, rows, 0.0)), 0.0).max(axis=0) if rows.size else np.zeros(C)
        for c in range(C):
            e = exps[t, c] = step_exponent(float(tops[c]))
            q = np.clip(np.rint(np.where(fine[:, c], rows[:, c], 0.0) / 2.0 ** e), -127, 127)
            codes[t * BLOCK:(t + 1) * BLOCK, c] = np.where(fine[:, c], q, -128).astype(np.int8)
    return codes, exps


def values(codes, exps):
    M = codes.shape[0]
    step = np.exp2(exps.astype(np.float64)).repeat(BLOCK, axis=0)[:M]
    v = codes.astype(np.float64) * step
    v[codes == -128] = np.nan
    return v


def bits_of(on):
    """(M, C) truth values -> uint32 words (ceil(M / 32), C), bit i of word t = row 32 t + i."""
    M, C = on.shape
    nb = (M + BLOCK - 1) // BLOCK
    w = np.zeros((nb, C), np.uint32)
    for m in range(M):
        w[m // BLOCK] |= on[m].astype(np.uint32) << np.uint32(m % BLOCK)
    return w


def mask_of(words, M):
    return np.stack([(words[m // BLOCK] >> np.uint32(m % BLOCK)) & 1 for m in range(M)]).astype(bool) if M else np.zeros((0, words.shape[1]), bool)


def bn_backward(g, xhat, mask, rstd, gamma):
    """gz, d gamma, d beta, gy of out = relu?(gamma xhat + beta + identity) with batch statistics."""
    M = g.shape[0]
    gz = np.where(mask, g, 0.0)
    sg, sgx = gz.sum(axis=0), (gz * xhat).sum(axis=0)
    return gz, sgx, sg, gamma * rstd * (gz - sg / M - xhat * (sgx / M))
