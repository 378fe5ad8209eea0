"""The next token from temperature, top-k, top-p and min-p, plainly: one row at a time, sorted, in exact sums."""
import math
from fractions import Fraction

import numpy as np


def sample_filtered(row, temperature, top_k, top_p, min_p, u):
    """The token, and how near the decision was: the smallest distance of a running sum to the border that it was compared with, relative to the whole
    sum (a token chosen nearer than that to its border may as well be its neighbour)."""
    row = np.asarray(row, dtype=np.float64)
    row = np.where(np.isnan(row), -np.inf, row)
    order = np.argsort(-row, kind="stable")
    top = row[order[0]]
    if top == -np.inf:
        return -1, 1.0
    if not temperature > 0:
        return int(order[0]), 1.0
    if top == np.inf:
        w = np.where(row[order] == np.inf, 1.0, 0.0)
    else:
        w = np.exp((row[order] - top) / float(np.float32(temperature)))
    w = w[row[order] > -np.inf]
    if top_k > 0:
        w = w[:top_k]
    near = 1.0

    def first_over(w, share):
        nonlocal near
        running, border = np.cumsum(w), float(np.float32(share)) * math.fsum(w)
        near = min(near, float(np.abs(running - border).min() / running[-1]))
        over = np.nonzero(running > border)[0]
        return int(over[0]) if len(over) else len(w) - 1

    if 0 < top_p < 1:
        w = w[:first_over(w, top_p) + 1]
    least = min(float(np.float32(min_p)), 1.0)
    if least > 0:
        near = min(near, float(np.abs(w[1:] / least - 1).min()) if len(w) > 1 and least < 1 else 1.0)
        w = w[w >= least]
    return int(order[first_over(w, u)]), near


def xorshift(state):
    """The next state (a signed 64-bit pattern) and the number in [0, 1) drawn from it."""
    x = state & (2 ** 64 - 1)
    x ^= x >> 12
    x = (x ^ (x << 25)) & (2 ** 64 - 1)
    x ^= x >> 27
    u = ((x * 0x2545F4914F6CDD1D) & (2 ** 64 - 1)) >> 32
    return (x - 2 ** 64 if x >= 2 ** 63 else x), float(Fraction(u >> 8, 2 ** 24))
