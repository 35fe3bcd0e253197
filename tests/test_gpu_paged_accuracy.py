"""How near attention over the paged cache comes to the formula on ordinary inputs, all
outputs of a call together: the bounds of test_gpu_paged.py are for the worst case of each
value, and would not notice a piece of q or p that is lost.

TOL: queries, keys and values of deviation 1, scale dH^-1/2, scores of deviation 1.  What
rounds, each as the deviation of a probability relative to itself:
  q in two fp16 pieces (22 bits), dH products of them    2^-22 / sqrt 3                       1.4e-7
  up to 2 dH = 512 roundings of a score's running sum    sqrt(512) 2^-24 / sqrt 3             7.8e-7
  scale, log2 e, the maximum taken off (below 2^3)       2^3 2^-24 ln 2                       3.3e-7
  exp2, and p in two pieces                              2^-22 and 2^-22 / sqrt 3             2.8e-7
Slots' errors are independent, so that the sums of p V are off by as much of themselves, and by their own roundings,
for 2600 slots by 16 sqrt(163) 2^-24 / sqrt 3 = 4.4e-7: 1.1e-6 in all.  Three times that are
allowed, and rounded up.  One piece of q or p alone (11 bits, 2^-12 / sqrt 3 or more) is off by 1.4e-4."""
import numpy as np
import pytest

import paged_ref as ref
from test_gpu_paged import Cache
from util import rel_l2

TOL = 4e-6
# kv heads, group, tokens, cached slots: tiles in registers and shared steps, a workgroup a head and cut into pieces
PATHS = [(2, 4, 1, 130), (1, 2, 3, 2600), (2, 16, 2, 300), (2, 4, 20, 100), (1, 4, 40, 2600)]


def emulated(q, K, V, seen, scale, pieces_q, pieces_p):
    """out [nH, dH] with q and p in one or two fp16 pieces, as an F16 cache multiplies them, all else in 64 bits."""
    def pieces(x, n):
        hi = x.astype(np.float16).astype(np.float64)
        return hi if n == 1 else hi + (x - hi).astype(np.float16).astype(np.float64)
    nH, dH = q.shape
    out = np.zeros((nH, dH))
    at = np.flatnonzero(seen)
    for h in range(nH):
        z = h // (nH // K.shape[1])
        x = q[h].astype(np.float64)
        e = 2.0 ** (15 - np.frexp(np.abs(x).max())[1])
        s = (K[at, z] @ pieces(x * e, pieces_q)) / e * scale
        p = 2048 * np.exp(s - s.max())
        out[h] = (pieces(p, pieces_p) @ V[at, z]) / p.sum()
    return out


def inputs(rng, nH, nKV, dH, n):
    q = rng.standard_normal((nH, dH)).astype(np.float32)
    K, V = (rng.standard_normal((n, nKV, dH)).astype(np.float16).astype(np.float64) for _ in range(2))
    return q, K, V


@pytest.mark.parametrize("dH", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("n", [40, 130, 2600])
def test_one_piece_would_show(dH, n):
    """On the CPU: two pieces are within the tolerance, one of q or p is far outside."""
    q, K, V = inputs(np.random.default_rng(dH + n), 8, 2, dH, n)
    seen = np.ones(n, bool)
    want, _ = ref.attend(q, K, V, seen, dH ** -0.5)
    off = {(a, b): rel_l2(emulated(q, K, V, seen, dH ** -0.5, a, b), want) for a in (1, 2) for b in (1, 2)}
    assert off[2, 2] < TOL / 4
    assert min(off[1, 2], off[2, 1], off[1, 1]) > 10 * TOL


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("dH", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("nKV,group,T,upto", PATHS)
def test_accuracy(fh, kind, dH, nKV, group, T, upto):
    rng = np.random.default_rng(dH + upto)
    c = Cache(fh, rng, 1, 1, nKV, dH, 16, -(-(upto + T) // 16), kind, [upto])
    k, v = c.fill(rng, 0, [upto + T])
    for pool in (k, v):
        pool[:] = rng.standard_normal(pool.shape)
    c.k.upload(k)
    c.v.upload(v)
    nH = nKV * group
    q = rng.standard_normal((T, nH, dH)).astype(np.float32)
    out, dq = fh.DeviceArray((1, T, nH, dH)), fh.DeviceArray.from_numpy(q[None])
    c.call("attn", 0, out, dq, nH, dH ** -0.5, T, None, 0, 0)
    K, _ = ref.gather(k[0], c.table_host, 16, 0, upto + T)
    V, _ = ref.gather(v[0], c.table_host, 16, 0, upto + T)
    want = np.stack([ref.attend(q[t], K, V, np.arange(upto + T) <= upto + t, dH ** -0.5)[0] for t in range(T)])
    assert rel_l2(out.numpy()[0], want) <= TOL
