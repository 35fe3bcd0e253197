"""Plain 64-bit numpy forms of the paged key-value cache and of the verification
of drafted tokens (fg_paged_*, fg_draft_verify), written from the definitions in
include/forge_hip.h.  Parity with the reference unpinned: none of its outputs
covers them."""
import math

import numpy as np


def rotate(x, pos, cos, sin, rot, half):
    """x [heads, dH] of a token at position pos, tables [npos, rot / 2]; fp64."""
    y = np.asarray(x, np.float64).copy()
    for i in range(rot // 2):
        a, b = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
        c, s = (cos[pos, i], sin[pos, i]) if pos < len(cos) else (math.nan, math.nan)
        y[:, a], y[:, b] = x[:, a].astype(np.float64) * c - x[:, b].astype(np.float64) * s, x[:, a].astype(np.float64) * s + x[:, b].astype(np.float64) * c
    return y


def page_of(table, nPages, P, s, j):
    """Page and row of slot j of sequence s, or None."""
    if j // P >= table.shape[1]:
        return None
    p = int(table[s, j // P])
    return (p, j % P) if 0 <= p < nPages else None


def sees(pos, n, window, sinks):
    """Which of slots 0 .. n - 1 a query of position pos sees."""
    j = np.arange(n)
    m = j <= pos
    if window:
        m &= (j > pos - window) | (j < sinks)
    return m


def gather(pool, table, P, s, n):
    """Slots 0 .. n - 1 of sequence s of pool [nPages, nKV, P, dH]: values [n, nKV, dH] (fp64) and which exist."""
    nKV, dH = pool.shape[1], pool.shape[3]
    out, there = np.full((n, nKV, dH), np.nan), np.zeros(n, bool)
    for j in range(n):
        at = page_of(table, len(pool), P, s, j)
        if at:
            out[j], there[j] = pool[at[0], :, at[1]].astype(np.float64), True
    return out, there


def attend(q, K, V, seen, scale):
    """q [nH, dH], K, V [n, nKV, dH] (fp64), seen [n]: out [nH, dH] and p [nH, n]; what is not seen has no part in it."""
    nH, dH = q.shape
    nKV = K.shape[1]
    out, p = np.zeros((nH, dH)), np.zeros((nH, len(K)))
    at = np.flatnonzero(seen)
    if len(at):
        with np.errstate(all="ignore"):
            for h in range(nH):
                z = h // (nH // nKV)
                s = scale * (K[at, z] @ q[h].astype(np.float64))
                e = np.exp(s - s.max())
                p[h, at] = e / e.sum()
                out[h] = p[h, at] @ V[at, z]
    return out, p


def softmax(x, temperature):
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        e = np.exp((x - np.fmax.reduce(x)) / temperature)
        return e / e.sum()


def best(x):
    """The lowest token of greatest logit, NaN below all; -1 where all are NaN."""
    m = np.fmax.reduce(x)
    return -1 if np.isnan(m) else int(np.flatnonzero(x == m)[0])


def draw(w, u):
    """The least token whose cumulated weight exceeds u of the whole (the last of any weight if none); -1 if that is no number."""
    total = math.fsum(w) if np.isfinite(w).all() else math.nan
    if not total > 0:
        return -1
    reach = np.cumsum(w)
    over = np.flatnonzero((reach > u * reach[-1]) & (w > 0))
    return int(over[0]) if len(over) else int(np.flatnonzero(w > 0)[-1])


def verify(logits, draft_logits, draft, u, temperature, n):
    """One sequence: logits [D + 1, V], draft_logits [D, V] or None, draft [D], u [D + 1], n drafts (below 0: no part).
    Returns token [D + 1] and count."""
    D, V = len(draft), logits.shape[1]
    token = np.full(D + 1, -1, np.int32)
    n = min(n, D)
    if n < 0:
        return token, 0
    for t in range(n + 1):
        more, x = t < n, int(draft[t]) if t < n else -1
        if temperature == 0:
            last = best(logits[t])
            stands = more and x == last and x >= 0
        else:
            p = softmax(logits[t], temperature)
            q = np.zeros(V)
            if more and draft_logits is not None:
                q = softmax(draft_logits[t], temperature)
            elif more and 0 <= x < V:
                q[x] = 1.0
            stands = more and 0 <= x < V and bool(float(u[t]) * q[x] < p[x])
            if not stands:
                last = -1
                if not np.isnan(p).any():
                    w = np.fmax(p - q, 0.0)
                    last = draw(w if w.sum() > 2.0 ** -40 else p, float(u[D]))
        if not stands:
            token[t] = last
            return token, t + 1
        token[t] = x
