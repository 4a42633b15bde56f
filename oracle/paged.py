"""CPU oracle of the paged key-value cache's operators (TEST INFRASTRUCTURE ONLY).

float64 numpy statements of include/tq4_paged.h, slot by slot: where a row lies, what the norm and
the rotation make of it, softmax over the slots in use, and the order that eviction keeps by. Each
also returns the bound that a 32-bit evaluation may be off by, so that the tests' tolerances follow
from the operands: u = 2^-24 is the f32 half step relative to a value.
"""

import math

import numpy as np

U = 2.0 ** -24


def place(table, page_size, seq, slot):
    return int(table[seq, slot // page_size]), slot % page_size


def norm_rotate(x, w, eps, cos, sin, pair_axis, positions, interleaved):
    """One head's values [D] -> (normed and turned [D], f32 error bound [D]).

    The sum of squares is a chain of at most 16 products a lane and 5 tree steps (with its mean 15 u or
    fewer are met by a value; halved by the root), the reciprocal root is within 4 u, the products by
    it and by w add 2 u, and a turned value takes 3 roundings of terms that together are at most
    sqrt(2) * hypot(pair): 20 u of the pair's length covers it."""
    y = np.asarray(x, np.float64)
    if w is not None:
        y = y / math.sqrt(np.mean(y * y) + eps) * np.asarray(w, np.float64)
    bound = np.abs(y) * 20 * U
    out = y.copy()
    pairs = cos.shape[1]
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        p = int(positions[pair_axis[i]])
        c, s = float(cos[p, i]), float(sin[p, i])
        out[a], out[b] = y[a] * c - y[b] * s, y[b] * c + y[a] * s
        bound[a] = bound[b] = math.hypot(y[a], y[b]) * 20 * U
    return out, bound


def attend(q, k, v, scale, lo, hi):
    """q [G, D], k and v [n, D] of one KV head -> (out [G, D], weights [G, hi - lo], bounds of both).

    A score is a sum of D products, rounded at most D + 4 times with its scaling: off by delta. All
    weights then share a relative error of at most 2 delta, plus 16 u for the exponentials, the join's
    factors and the quotient, plus the chain of the sums (a quarter of the slots for each of four
    warps, and the joins)."""
    g, d = q.shape
    if hi <= lo:
        return np.zeros((g, d)), np.zeros((g, 0)), np.zeros((g, d)), np.zeros((g, 0))
    q, k, v = (np.asarray(x, np.float64) for x in (q, k[lo:hi], v[lo:hi]))
    s = q @ k.T * scale
    e = np.exp(s - s.max(1, keepdims=True))
    w = e / e.sum(1, keepdims=True)
    delta = (np.abs(q) @ np.abs(k).T * abs(scale)).max(1, keepdims=True) * (d + 4) * U
    rel = 2 * delta + (16 + (hi - lo) / 4 + 40) * U
    return w @ v, w, (w @ np.abs(v)) * rel, w * rel


def attention(q, k_pages, v_pages, table, lengths, scale, window, scores=None):
    """q [B, H, D] -> (out [B, H, D], its bound, new scores or None, their bound)."""
    batch, heads, d = q.shape
    kv, ps = k_pages.shape[1], k_pages.shape[2]
    group = heads // kv
    out, bound = np.zeros((batch, heads, d)), np.zeros((batch, heads, d))
    new = None if scores is None else np.asarray(scores, np.float64).copy()
    new_bound = None if scores is None else np.zeros(scores.shape)
    for b in range(batch):
        n = int(lengths[b])
        lo = max(0, n - window) if window else 0
        at = [place(table, ps, b, j) for j in range(n)]
        for h in range(kv):
            k = np.array([k_pages[p, h, r] for p, r in at]).reshape(n, d)
            v = np.array([v_pages[p, h, r] for p, r in at]).reshape(n, d)
            hs = slice(h * group, (h + 1) * group)
            out[b, hs], w, bound[b, hs], wb = attend(q[b, hs], k, v, scale, lo, n)
            if new is not None:
                new[b, h, lo:n] += w.sum(0)
                new_bound[b, h, lo:n] = wb.sum(0) + np.abs(new[b, h, lo:n]) * U * (group + 1)
    return out, bound, new, new_bound


def keep_slots(scores, n, keep, recent):
    """The slots that stay of n with these scores, ascending."""
    if n <= keep:
        return list(range(n))
    key = [(-math.inf, 0) if math.isnan(x) else (float(x), 1) for x in scores[:n - recent]]  # NaN below -inf
    order = sorted(range(n - recent), key=lambda j: (-key[j][0], -key[j][1], j))
    return sorted(order[:keep - recent]) + list(range(n - recent, n))
