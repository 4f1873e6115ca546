"""Oracle of the low-rank adapters (humaniflow_amd/adapters.py): the definitions in float64 on the CPU, one row at a time.

ids < 0: no adapter; ids >= L: the row's outputs are NaN and it adds to no gradient.  `bound` arrays are what 32-bit sums of the same terms may be off by: a sum of n
terms in 32 bits is a random walk of roundings of its partial sums, with a standard deviation of about eps sqrt(n) / 2.4 times the 2-norm of the terms; 10 of them.
"""
import numpy as np

EPS = 2.0 ** -24


def _walk(n, norm):
    return 4.0 * (np.sqrt(n) + 8.0) * EPS * norm


def _norm_of_products(p, q):
    """2-norm of the terms of p @ q."""
    return np.sqrt((p * p) @ (q * q))


def forward(x, w, bias, a, b, scale, ids):
    """y, t and the bounds of both."""
    M, K = x.shape
    N, r = w.shape[0], a.shape[1]
    y = x @ w.T + (0.0 if bias is None else bias)
    ey = _walk(K + r, _norm_of_products(x, w.T)) + EPS * np.abs(y) * 2
    t, et = np.zeros((M, r)), np.zeros((M, r))
    for m in range(M):
        l = int(ids[m])
        if l >= a.shape[0]:
            y[m], t[m] = np.nan, np.nan
        elif l >= 0:
            t[m] = scale[l] * (a[l] @ x[m])
            et[m] = _walk(K, abs(scale[l]) * np.sqrt((a[l] ** 2) @ (x[m] ** 2))) + 2 * EPS * np.abs(t[m])
            y[m] += b[l] @ t[m]
            # t's own error, t as two bfloat16 (2^-17), the r products
            ey[m] += np.abs(b[l]) @ (et[m] + 2.0 ** -17 * np.abs(t[m])) + _walk(r, np.sqrt((b[l] ** 2) @ (t[m] ** 2)))
    return y, t, ey, et


def backward(dy, x, t, w, a, b, scale, ids):
    M, N = dy.shape
    K, L, r = w.shape[1], a.shape[0], a.shape[1]
    dx = dy @ w
    edx = _walk(N + r, _norm_of_products(dy, w)) + EPS * np.abs(dx) * 2
    da, db = np.zeros_like(a), np.zeros_like(b)
    u, eu = np.zeros((M, r)), np.zeros((M, r))
    for m in range(M):
        l = int(ids[m])
        if l >= L:
            dx[m] = np.nan
        elif l >= 0:
            u[m] = scale[l] * (b[l].T @ dy[m])
            eu[m] = _walk(N, abs(scale[l]) * np.sqrt((b[l].T ** 2) @ (dy[m] ** 2))) + 2 * EPS * np.abs(u[m])
            dx[m] += a[l].T @ u[m]
            edx[m] += np.abs(a[l].T) @ (eu[m] + 2.0 ** -17 * np.abs(u[m])) + _walk(r, np.sqrt((a[l].T ** 2) @ (u[m] ** 2)))
    eda, edb = np.zeros_like(a), np.zeros_like(b)
    for l in range(L):
        rows = np.nonzero(np.asarray(ids) == l)[0]
        if len(rows):
            da[l] = u[rows].T @ x[rows]
            db[l] = dy[rows].T @ t[rows]
            eda[l] = _walk(len(rows), _norm_of_products(u[rows].T, x[rows])) + eu[rows].T @ np.abs(x[rows])
            edb[l] = _walk(len(rows), _norm_of_products(dy[rows].T, t[rows]))
    return dx, da, db, edx, eda, edb
