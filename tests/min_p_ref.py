"""Sampling with options per row in 64 bits, from the definition (plain numpy, one row at a time)."""
import numpy as np


def sample_row(x, T, k, p, m, u):
    """(token, kept, logprob) of one row of float64 values; T = 0 is greedy, k <= 0, p >= 1 and
    m = 0 are off."""
    x = np.asarray(x, np.float64)
    ids = np.flatnonzero(x > -np.inf)
    ids = ids[np.lexsort((ids, -x[ids]))]
    if T == 0:
        return int(ids[0]), 1, 0.0
    d = (x[ids] - x[ids[0]]) / np.float64(T)
    w = np.exp(d)
    mass = np.cumsum(w)
    n = len(ids) if k <= 0 else min(int(k), len(ids))
    if p < 1:
        n = min(n, int(np.count_nonzero(mass[:n] < np.float64(p) * mass[n - 1])) + 1)
    if m > 0:
        # w >= m, compared as logarithms: next to 1 the weights round (exp(-1e-38) is 1.0 in 64
        # bits and less than 1 by definition), their logarithms d do not
        n = min(n, int(np.count_nonzero(d >= np.log(np.float64(m)))))
    j = min(int(np.count_nonzero(mass[:n] <= np.float64(u) * mass[n - 1])), n - 1)
    return int(ids[j]), n, float(d[j] - np.log(mass[n - 1]))


def sample_rows(x, T, k, p, m, u):
    got = [sample_row(x[r], T[r], k[r], p[r], m[r], u[r]) for r in range(len(x))]
    return (np.array([g[0] for g in got]), np.array([g[1] for g in got]),
            np.array([g[2] for g in got]))
