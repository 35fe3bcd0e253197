"""Attention over the paged cache (fg_paged_attn) with infinities among the keys or the
values that a query sees: what the formula gives for them, in 64 bits, wherever in a
step, a piece or a wave's share they lie."""
import math

import numpy as np
import pytest

import paged_ref as ref
from test_gpu_paged import Cache, out_bound

pytestmark = pytest.mark.gpu

# heads, and cached slots: a row or a few (register tiles), many (shared steps; heads of 256 stay in registers),
# each a workgroup a head, and cut into pieces
SHAPES = [(32, 2, 2, 1, 16), (64, 1, 1, 1, 16), (128, 2, 4, 1, 600), (256, 1, 2, 1, 40), (96, 1, 1, 1, 700),
          (64, 1, 4, 5, 2600), (128, 1, 2, 3, 2600), (64, 1, 2, 40, 50), (128, 1, 4, 40, 2600), (96, 1, 3, 30, 33),
          (32, 1, 1, 80, 0), (256, 1, 2, 20, 100)]


def formula(q, K, V, seen, scale):
    """out [nH, dH] and p [nH, n], products and sums written out, so that 0 inf and inf - inf are NaN where the formula has them."""
    nH, dH = q.shape
    out, p = np.zeros((nH, dH)), np.zeros((nH, len(K)))
    at = np.flatnonzero(seen)
    with np.errstate(all="ignore"):
        for h in range(nH if len(at) else 0):
            z = h // (nH // K.shape[1])
            s = scale * (K[at, z] * q[h].astype(np.float64)).sum(-1)
            e = np.exp(s - s.max())
            p[h, at] = e / e.sum()
            out[h] = (p[h, at, None] * V[at, z]).sum(0)
    return out, p


def check(fh, c, q, k, v, scale, window=0, sinks=0):
    """Every output: NaN and infinities as the formula has them, the others within the roundings."""
    c.k.upload(k)
    c.v.upload(v)
    _, T, nH, _ = q.shape
    out, dq = fh.DeviceArray.from_numpy(np.full(q.shape, 7.25, np.float32)), fh.DeviceArray.from_numpy(q)
    c.call("attn", 0, out, dq, nH, scale, T, None, window, sinks)
    got, kind, odd = out.numpy(), "f16" if c.type else "f32", 0
    clean = lambda x: np.where(np.isfinite(x), x, 0.0)  # noqa: E731
    for s in range(c.nSeq):
        n0 = int(c.lens[s])
        K, there = ref.gather(k[0], c.table_host, c.P, s, n0 + T)
        V, _ = ref.gather(v[0], c.table_host, c.P, s, n0 + T)
        for t in range(T):
            seen = ref.sees(n0 + t, n0 + T, window, sinks) & there
            want, p = formula(q[s, t], K, V, seen, scale)
            bad = ~np.isfinite(want)
            odd += bad.sum()
            assert np.array_equal(got[s, t][bad], want[bad], equal_nan=True), (s, t, got[s, t][bad], want[bad])
            with np.errstate(all="ignore"):
                ok = np.abs(got[s, t] - want) <= out_bound(q[s, t], clean(K), clean(V), np.where(np.isnan(p), 0.0, p), seen, scale, kind)
            assert (ok | bad).all(), (s, t, got[s, t], want)
    return odd


def queries(rng, nSeq, T, nH, dH):
    """Queries whose first value is above zero, but for a few whose is below."""
    q = rng.standard_normal((nSeq, T, nH, dH)).astype(np.float32)
    q[..., 0] = np.abs(q[..., 0]) + 0.125
    q[:, 2::5, -1, 0] *= -1
    return q


@pytest.mark.parametrize("where", ["last", "first", "spread", "all"])
@pytest.mark.parametrize("dH,nKV,group,T,upto", SHAPES)
def test_infinite_keys(fh, dH, nKV, group, T, upto, where):
    """A score of -inf is a probability of zero wherever its slot lies: alone in a step, in all of a wave's first ones, among
    others.  With one of +inf, or none above -inf, the row is NaN."""
    rng = np.random.default_rng(dH + T + upto)
    n = upto + T
    c = Cache(fh, rng, 1, 1, nKV, dH, 16, -(-n // 16), "f32", [upto])
    k, v = c.fill(rng, 0, [n])
    slots = {"last": [n - 1], "first": range(min(70, n - 1)), "spread": range(0, n, 7), "all": range(n)}[where]
    for j in slots:
        p, i = c.at(0, j)
        k[0, p, :, i, 0] = -np.inf
    odd = check(fh, c, queries(rng, 1, T, nKV * group, dH), k, v, dH ** -0.5)
    assert odd > 0 or where != "all"


@pytest.mark.parametrize("group,T", [(1, 1), (2, 60)])
def test_nothing_but_infinite_keys(fh, group, T):
    """Rows that see no slot are zeros, rows that see scores of -inf alone are NaN, in windows and behind missing pages."""
    rng = np.random.default_rng(T)
    lens = [90, 90, 90]
    c = Cache(fh, rng, 1, 3, 1, 64, 16, 10, "f32", lens)
    k, v = c.fill(rng, 0, [160] * 3)
    for s in range(3):
        for j in range(80, 160):
            p, i = c.at(s, j)
            k[0, p, 0, i, 0] = -np.inf
    for p in range(10):
        if p < 5:
            c.drop(1, p)
        c.drop(2, p)
    q = queries(rng, 3, T, group, 64)
    check(fh, c, q, k, v, 0.125)
    check(fh, c, q, k, v, 0.125, window=5)
    assert check(fh, c, q, k, v, 0.125, window=5, sinks=3) > 0


def odd_values(c, v, s, slots):
    """Infinities of either sign and NaN at slots a < b < e of a sequence, in a column alone and two of them in one."""
    (pa, ia), (pb, ib), (pe, ie) = (c.at(s, j) for j in slots)
    v[0, pa, :, ia, :4] = [np.inf, -np.inf, np.inf, np.inf]
    v[0, pb, :, ib, 4:6] = [-np.inf, np.nan]
    v[0, pb, :, ib, c.dH - 1] = np.inf
    v[0, pe, :, ie, 2:4] = [-np.inf, np.inf]
    v[0, pe, :, ie, 6:9] = [np.inf, -np.inf, np.nan]


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("spread", [1.0, 80.0])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
@pytest.mark.parametrize("dH,nKV,group,T,upto", SHAPES)
def test_infinite_values(fh, kind, dH, nKV, group, T, upto, window, sinks, spread):
    """An infinite value makes its column infinite, one of either sign NaN, in steps that all rows see and in others, and where
    its probability is below what fp32 holds (scores 80 apart on the average; 2^-800 in fp64)."""
    rng = np.random.default_rng(dH + T + upto)
    n = upto + T
    c = Cache(fh, rng, 1, 2, nKV, dH, 16, -(-n // 16), kind, [upto, upto // 2])
    k, v = c.fill(rng, 0, [n, upto // 2 + T])
    odd_values(c, v, 0, (min(3, n - 3), max(n // 2, min(3, n - 3) + 1), n - 1))
    m = upto // 2 + T
    if m > 4:
        odd_values(c, v, 1, (1, 2, m - 1 - T // 2))
    # (values of K are of e^-1 .. e^1: 1.8 in their squares' mean)
    scale = spread / math.sqrt(1.8 * dH)
    assert check(fh, c, queries(rng, 2, T, nKV * group, dH), k, v, scale, window, sinks) > 0


@pytest.mark.parametrize("dH,nKV,group,T,upto", SHAPES)
def test_infinite_values_of_no_weight(fh, dH, nKV, group, T, upto):
    """A probability of exactly zero (a score of -inf) times an infinite value is NaN, beside slots where it is not."""
    rng = np.random.default_rng(dH + T + upto)
    n = upto + T
    c = Cache(fh, rng, 1, 1, nKV, dH, 16, -(-n // 16), "f32", [upto])
    k, v = c.fill(rng, 0, [n])
    for j, column in ((1, 3), (n - 1, 4), (n // 2, 5)):
        p, i = c.at(0, j)
        k[0, p, :, i, 0] = -np.inf
        v[0, p, :, i, column] = np.inf
    p, i = c.at(0, 2)
    v[0, p, :, i, 2:5] = np.inf
    assert check(fh, c, queries(rng, 1, T, nKV * group, dH), k, v, dH ** -0.5) > 0


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("group,T", [(1, 1), (2, 60)])
def test_large_values_and_unseen_infinities(fh, kind, group, T):
    """Values at the end of what the sums take (2^100; fp16: 65504), beside an infinite one in another column; infinities
    in slots behind the last token, which nothing sees."""
    rng = np.random.default_rng(T)
    c = Cache(fh, rng, 1, 2, 1, 64, 16, 10, kind, [70, 90])
    k, v = c.fill(rng, 0, [70 + T, 90 + T])
    for j in range(30):
        p, i = c.at(0, j)
        v[0, p, 0, i, 9] = (2.0 ** 100 if kind == "f32" else 65504) * (-1) ** j
    for s, j in ((0, 70 + T), (1, 90 + T), (1, 91 + T)):
        p, i = c.at(s, j)
        v[0, p, 0, i] = np.inf
        k[0, p, 0, i] = np.nan
    assert check(fh, c, queries(rng, 2, T, group, 64), k, v, 0.125) == 0
    p, i = c.at(0, 40)
    v[0, p, 0, i, 8] = np.inf
    assert check(fh, c, queries(rng, 2, T, group, 64), k, v, 0.125) > 0
