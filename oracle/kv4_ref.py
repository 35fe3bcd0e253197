"""Plain 64-bit numpy forms of the 4-bit key-value cache and of beam search
(fg_kv4_*, fg_kv_evict_select, fg_beam_*), written from the definitions in
include/forge_hip.h.  No counterpart in the reference."""
import math

import numpy as np


def quantize(x):
    """Codes (uint8) and steps (fp16) of x [..., dH] in blocks of 32: [..., nb, 32] and [..., nb]."""
    x = np.asarray(x, np.float32)
    b = x.reshape(*x.shape[:-1], -1, 32).astype(np.float64)
    with np.errstate(all="ignore"):
        at = np.abs(np.where(np.isnan(b), -1.0, b)).argmax(-1)  # the first of equals
        m = np.take_along_axis(b, at[..., None], -1)[..., 0]
        d = (m / -8.0).astype(np.float32).astype(np.float16)
        d = np.where(np.isfinite(b).all(-1) & np.isfinite(d), d, np.float16(np.nan))
        wide = d.astype(np.float64)[..., None]
        c = np.floor(b / wide + 8.5)
    c = np.where(np.isfinite(wide) & (wide != 0), c, 8.0)
    return np.clip(c, 0, 15).astype(np.uint8), d


def pack(codes):
    """Codes [..., nb, 32] as a slot's bytes [..., 16 nb]."""
    nb = codes.shape[-2]
    out = np.zeros(codes.shape[:-2] + (16 * nb,), np.uint8)
    for n in range(16):
        for b in range(nb):
            out[..., n * nb + b] = codes[..., b, n] | (codes[..., b, 16 + n] << 4)
    return out


def values(bytes_, steps):
    """The values [..., dH] (fp64) of bytes [..., 16 nb] and steps [..., nb]."""
    nb = steps.shape[-1]
    out = np.zeros(bytes_.shape[:-1] + (32 * nb,))
    with np.errstate(all="ignore"):
        for n in range(16):
            for b in range(nb):
                byte = bytes_[..., n * nb + b].astype(np.int64)
                d = steps[..., b].astype(np.float64)
                out[..., 32 * b + n] = d * ((byte & 15) - 8)
                out[..., 32 * b + 16 + n] = d * ((byte >> 4) - 8)
    return out


def attend(q, K, V, scale):
    """q [nH, dH], K, V [n, nKV, dH] (fp64): out [nH, dH] and p [nH, n]."""
    nH, dH = q.shape
    n, nKV = K.shape[:2]
    out, p = np.zeros((nH, dH)), np.zeros((nH, n))
    for h in range(nH if n else 0):
        z = h // (nH // nKV)
        s = scale * (K[:, z] @ q[h].astype(np.float64))
        e = np.exp(s - s.max())
        p[h] = e / e.sum()
        out[h] = p[h] @ V[:, z]
    return out, p


def evict(weight, pos, n, nxt, budget, recent):
    """Holes and movers (lists of slots) of one head."""
    if n <= budget:
        return [], []
    safe = [j for j in range(n) if pos[j] >= nxt - recent]
    rest = [j for j in range(n) if pos[j] < nxt - recent]
    rest.sort(key=lambda j: (1, 0.0, j) if math.isnan(weight[j]) else (0, -float(weight[j]), j))
    kept = set((safe + rest)[:budget])
    return [j for j in range(budget) if j not in kept], [j for j in range(budget, n) if j in kept]


def beam_select(logits, scores, done, eos, nReq, W):
    """(score fp64, token, parent, done) of nReq requests, each [nReq W]."""
    V = logits.shape[1]
    out = []
    for r in range(nReq):
        cand = []
        for b in range(W):
            i = r * W + b
            if done is not None and done[i]:
                cand.append((float(scores[i]), 0.0, b, eos))
                continue
            x = logits[i].astype(np.float64)
            with np.errstate(all="ignore"):
                m = np.nan if np.isnan(x).any() else x.max()
                base = -math.inf if m == -math.inf else float(np.float64(scores[i]) - (m + np.log(np.exp(x - m).sum())))
            if not math.isfinite(base):
                cand += [(base, 0.0, b, v) for v in range(min(V, W))]
                continue
            top = np.lexsort((np.arange(V), -x))[:W]
            cand += [(base + x[v], float(x[v]), b, int(v)) for v in top]
        cand.sort(key=lambda c: (math.isnan(c[0]), -c[0] if not math.isnan(c[0]) else 0.0, c[2], -c[1], c[3]))
        out += cand[:W]
    token = np.array([c[3] for c in out], np.int32)
    parent = np.array([c[2] for c in out], np.int32)
    fin = None
    if done is not None:
        fin = np.array([int(done[(i // W) * W + parent[i]] != 0 or token[i] == eos) for i in range(nReq * W)], np.int32)
    return np.array([c[0] for c in out]), token, parent, fin
