"""The paged key-value cache on the device (fg_paged_*) against the plain 64-bit
forms of oracle/paged_ref.py: stored rows within a rounding, untouched slots and
rows exactly, attention within bounds counted from the roundings."""
import math

import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu

HEADS = [32, 64, 96, 128, 256]
TYPES = {"f32": (0, np.float32, 2.0 ** -24), "f16": (1, np.float16, 2.0 ** -11)}


class Cache:
    """A cache on the device whose slots all hold NaN and whose pages are handed out shuffled."""

    def __init__(self, fh, rng, nLayers, nSeq, nKV, dH, P, maxPages, kind, lens, spare=3, upto=None):
        self.fh, self.nLayers, self.nSeq, self.nKV, self.dH, self.P, self.maxPages = fh, nLayers, nSeq, nKV, dH, P, maxPages
        self.type, self.dtype, self.half_step = TYPES[kind]
        # pages for the first upto[s] slots of a sequence, or for all of them
        need = [maxPages if upto is None else -(-int(n) // P) for n in (upto if upto is not None else [0] * nSeq)]
        self.nPages = sum(need) + spare
        order = iter(rng.permutation(self.nPages))
        self.table_host = np.array([[next(order) if p < n else -1 for p in range(maxPages)] for n in need], np.int32)
        shape = (nLayers, self.nPages, nKV, P, dH)
        up = fh.DeviceArray.from_numpy
        self.k, self.v = (up(np.full(shape, np.nan, self.dtype)) for _ in range(2))
        self.lens = np.array(lens, np.int32)
        self.len, self.table = up(self.lens), up(self.table_host)
        self.struct = fh.PagedCache(nLayers, nSeq, nKV, dH, P, self.nPages, maxPages, self.type, self.k.ptr, self.v.ptr,
                                    self.table.ptr, self.len.ptr)

    def call(self, name, *args):
        self.fh.call("paged_" + name, self.fh.ref(self.struct), *args)

    def drop(self, s, p, number=-1):
        self.table_host[s, p] = number
        self.table.upload(self.table_host)

    def at(self, s, j):
        return ref.page_of(self.table_host, self.nPages, self.P, s, j)

    def fill(self, rng, layer, upto):
        """Keys and values in the first upto[s] slots of every sequence."""
        k, v = self.k.numpy(), self.v.numpy()
        size = [np.exp(rng.uniform(-1, 1, (self.nKV, self.dH))) for _ in range(2)]
        for s in range(self.nSeq):
            for j in range(min(upto[s], self.maxPages * self.P)):
                at = self.at(s, j)
                if at:
                    for pool, z in ((k, size[0]), (v, size[1])):
                        pool[layer, at[0], :, at[1]] = rng.standard_normal((self.nKV, self.dH)) * z
        self.k.upload(k)
        self.v.upload(v)
        return k, v


def angles(fh, npos, rot, theta=10000.0):
    c, s = np.zeros((npos, max(rot // 2, 1))), np.zeros((npos, max(rot // 2, 1)))
    if rot:
        fh.check(fh.lib.fg_rope_table(c.ctypes.data, s.ctypes.data, npos, rot, theta))
    return c, s


def out_bound(q, K, V, p, seen, scale, kind):
    """Bounds of |out| errors, term by term.  A score's dH products are summed in dH roundings of 2^-24 at most, q in two
    fp16 pieces is off by 2^-22 of itself (F16), and scale, log2 e and the subtraction of the maximum round a
    few times more: 16 are counted, of the largest score.  exp2 is good to 2^-22; p's and the sums over n slots
    round at most n / 4 + 64 times in a chain (slots come 32 at a time, a running sum is rescaled at most once for
    each such step, parts are joined in a few steps).  p in two fp16 pieces is off by 2^-22 of itself, and where its low
    piece is subnormal by 2^-36 of the greatest."""
    nH, dH = q.shape
    nKV = K.shape[1]
    at = np.flatnonzero(seen)
    out = np.zeros((nH, dH))
    for h in range(nH if len(at) else 0):
        z = h // (nH // nKV)
        mass = abs(scale) * (np.abs(K[at, z]) @ np.abs(q[h].astype(np.float64))).max()
        es = mass * ((dH + 16) * 2.0 ** -24 + (2.0 ** -22 if kind == "f16" else 0))
        rel = 2 * es + 2.0 ** -21 + (len(at) / 4 + 64) * 2.0 ** -24
        out[h] = rel * (p[h, at] @ np.abs(V[at, z])) + len(at) * 2.0 ** -36 * np.abs(V[at, z]).max() + 1e-30
    return out


def check_attention(fh, c, rng, layer, nH, T, counts, window=0, sinks=0, scale=None, given=True):
    """Runs fg_paged_attn over what c holds and compares every row; rows behind a sequence's tokens stay as they were."""
    scale = 1.0 / math.sqrt(c.dH) if scale is None else scale
    q = rng.standard_normal((c.nSeq, T, nH, c.dH)).astype(np.float32)
    out = fh.DeviceArray.from_numpy(np.full(q.shape, 7.25, np.float32))
    dq = fh.DeviceArray.from_numpy(q)
    dc = fh.DeviceArray.from_numpy(np.array(counts, np.int32)) if given else None
    c.call("attn", layer, out, dq, nH, scale, T, dc, window, sinks)
    got = out.numpy()
    k, v = c.k.numpy()[layer], c.v.numpy()[layer]
    kind = "f16" if c.type else "f32"
    room = c.maxPages * c.P
    for s in range(c.nSeq):
        n0 = min(max(int(c.lens[s]), 0), room)
        n = min(max(int(counts[s]), 0), T) if given else T
        assert (got[s, n:] == 7.25).all(), s
        m = min(n0 + n, room)
        K, there = ref.gather(k, c.table_host, c.P, s, m)
        V, _ = ref.gather(v, c.table_host, c.P, s, m)
        for t in range(n):
            seen = ref.sees(n0 + t, m, window, sinks) & there
            want, p = ref.attend(q[s, t], K, V, seen, scale)
            ok = np.abs(got[s, t] - want) <= out_bound(q[s, t], K, V, p, seen, scale, kind)
            assert ok.all(), (s, t, np.abs(got[s, t] - want).max())
    return got


# ── store and read ────────────────────────────────────────────────────────
@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("dH,rot,half", [(32, 32, 0), (64, 32, 1), (96, 96, 1), (128, 128, 0), (256, 64, 1), (64, 0, 0), (32, 6, 0),
                                         (96, 50, 1), (128, 2, 1)])
@pytest.mark.parametrize("nSeq,nH,nKV,T,P,pad", [(1, 1, 1, 1, 4, 0), (3, 6, 2, 5, 4, 4), (4, 5, 5, 3, 16, 1), (2, 12, 3, 40, 8, 0)])
def test_append(fh, kind, dH, rot, half, nSeq, nH, nKV, T, P, pad):
    rng = np.random.default_rng(dH + rot + nSeq)
    maxPages = -(-(T + 9) // P)
    lens = rng.integers(0, 9, nSeq)
    c = Cache(fh, rng, 2, nSeq, nKV, dH, P, maxPages, kind, lens)
    npos = int(lens.max()) + T
    cos, sin = angles(fh, npos, rot)
    ld = (nH + 2 * nKV) * dH + pad
    qkv = rng.standard_normal((nSeq * T, ld)).astype(np.float32)
    counts = rng.integers(-1, T + 2, nSeq).astype(np.int32)
    counts[0] = T
    up = fh.DeviceArray.from_numpy
    d, dc, dcos, dsin = up(qkv), up(counts), up(cos), up(sin)
    qo = up(np.full((nSeq, T, nH, dH), 7.25, np.float32))
    c.call("append", 1, qo, d.ptr, d.ptr + 4 * nH * dH, d.ptr + 4 * (nH + nKV) * dH, ld, nH, T, dc, dcos, dsin, npos, rot, half)
    q, k, v = qo.numpy(), c.k.numpy(), c.v.numpy()
    want_k, want_v = np.full(k.shape, np.nan), np.full(v.shape, np.nan)
    rows = qkv[:, :(nH + 2 * nKV) * dH].reshape(nSeq, T, nH + 2 * nKV, dH)
    for s in range(nSeq):
        n = min(max(int(counts[s]), 0), T)
        assert (q[s, n:] == 7.25).all()
        for t in range(n):
            pos = int(lens[s]) + t
            want = ref.rotate(rows[s, t, :nH], pos, cos, sin, rot, half)
            # one rounding to fp32 after fp64's
            assert (np.abs(q[s, t] - want) <= 2.0 ** -24 * (1 + 2.0 ** -20) * np.abs(want) + 1e-37).all()
            p, j = c.at(s, pos)
            want_k[1, p, :, j] = ref.rotate(rows[s, t, nH:nH + nKV], pos, cos, sin, rot, half)
            want_v[1, p, :, j] = rows[s, t, nH + nKV:]
    for got, want in ((k, want_k), (v, want_v)):
        assert (np.isnan(got) == np.isnan(want)).all()
        at = ~np.isnan(want)
        # the type's rounding, after fp32's; fp16's subnormals are 2^-24 apart
        bound = (c.half_step + 2.0 ** -23) * np.abs(want[at]) + (2.0 ** -25 if kind == "f16" else 1e-37)
        assert (np.abs(got[at].astype(np.float64) - want[at]) <= bound).all()


def test_append_in_place_and_without_queries(fh):
    rng = np.random.default_rng(5)
    c = Cache(fh, rng, 1, 2, 4, 64, 8, 4, "f32", [3, 30])
    cos, sin = angles(fh, 40, 64)
    up = fh.DeviceArray.from_numpy
    q, k, v = (rng.standard_normal((6, 4 * 64)).astype(np.float32) for _ in range(3))
    dq, dk, dv, dcos, dsin = up(q), up(k), up(v), up(cos), up(sin)
    c.call("append", 0, dq, dq, dk, dv, 256, 4, 3, None, dcos, dsin, 40, 64, 0)
    first = c.k.numpy(), c.v.numpy()
    got = dq.numpy().reshape(2, 3, 4, 64)
    for s in range(2):
        for t in range(3):
            want = ref.rotate(q.reshape(2, 3, 4, 64)[s, t], [3, 30][s] + t, cos, sin, 64, 0)
            assert (np.abs(got[s, t] - want) <= 2.0 ** -24 * (1 + 2.0 ** -20) * np.abs(want)).all()
    c.k.upload(np.full(first[0].shape, np.nan, np.float32))
    c.call("append", 0, None, None, dk, dv, 256, 0, 3, None, dcos, dsin, 40, 64, 0)
    assert np.array_equal(c.k.numpy(), first[0], equal_nan=True) and np.array_equal(c.v.numpy(), first[1], equal_nan=True)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_append_beyond_pages_and_tables(fh, kind):
    """Slots without a page stay away, positions beyond the table turn to NaN, lengths are held to the room."""
    rng = np.random.default_rng(9)
    c = Cache(fh, rng, 1, 4, 2, 32, 4, 3, kind, [0, 7, 11, 0])
    c.drop(0, 1, -1)
    c.drop(1, 2, c.nPages)
    c.lens = np.array([0, 7, 1000, -5], np.int32)
    c.len.upload(c.lens)
    T, npos, rot = 6, 9, 16
    cos, sin = angles(fh, npos, rot)
    up = fh.DeviceArray.from_numpy
    x = rng.standard_normal((4 * T, 5 * 32)).astype(np.float32)
    d, dcos, dsin = up(x), up(cos), up(sin)
    qo = up(np.zeros((4, T, 1, 32), np.float32))
    c.call("append", 0, qo, d.ptr, d.ptr + 4 * 32, d.ptr + 4 * 96, 160, 1, T, None, dcos, dsin, npos, rot, 0)
    q, k, v = qo.numpy(), c.k.numpy()[0], c.v.numpy()[0]
    touched = np.zeros((c.nPages, 4), bool)
    for s, n0 in enumerate([0, 7, 12, 0]):
        for t in range(T):
            pos, at = n0 + t, c.at(s, n0 + t)
            assert np.isnan(q[s, t, 0, :rot]).all() == (pos >= npos) and (q[s, t, 0, rot:] == x[s * T + t, rot:32]).all()
            if at:
                touched[at] = True
                assert (v[at[0], :, at[1]] == x[s * T + t, 96:].reshape(2, 32).astype(c.dtype)).all()
                assert np.isnan(k[at[0], :, at[1], :rot]).all() == (pos >= npos)
    assert np.isnan(v.transpose(0, 2, 1, 3)[~touched]).all() and touched.sum() == 4 + 1 + 6


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("dH,pad", [(32, 0), (96, 4), (256, 3)])
def test_read(fh, kind, dH, pad):
    rng = np.random.default_rng(dH)
    c = Cache(fh, rng, 2, 3, 2, dH, 8, 4, kind, [0, 0, 0])
    c.drop(1, 1)
    k, v = c.fill(rng, 1, [32, 32, 20])
    ld = 2 * dH + pad
    for first, T in ((0, 32), (5, 9), (31, 1)):
        ok, ov = (fh.DeviceArray.from_numpy(np.full((3, T, ld), 7.25, np.float32)) for _ in range(2))
        c.call("read", 1, ok, ov, ld, first, T)
        for got, pool in ((ok.numpy(), k), (ov.numpy(), v)):
            assert (got[:, :, 2 * dH:] == 7.25).all()
            for s in range(3):
                want, there = ref.gather(pool[1], c.table_host, 8, s, 32)
                want[~there] = 0
                assert np.array_equal(got[s, :, :2 * dH].reshape(T, 2, dH), want[first:first + T].astype(np.float32), equal_nan=True)


def test_commit(fh):
    rng = np.random.default_rng(1)
    c = Cache(fh, rng, 1, 300, 1, 32, 4, 3, "f16", rng.integers(-3, 20, 300))
    counts = rng.integers(-4, 9, 300).astype(np.int32)
    dc = fh.DeviceArray.from_numpy(counts)
    c.call("commit", 5, dc)
    held = np.clip(c.lens, 0, 12)
    want = np.minimum(held + np.clip(counts, 0, 5), 12)
    assert (c.len.numpy() == want).all()
    c.call("commit", 2, None)
    assert (c.len.numpy() == np.minimum(want + 2, 12)).all()
    c.call("commit", 0, None)
    assert (c.len.numpy() == np.minimum(want + 2, 12)).all()


# ── attention ─────────────────────────────────────────────────────────────
@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("dH", HEADS)
@pytest.mark.parametrize("nKV,group,T,P,lens", [
    (1, 1, 1, 4, [0]), (2, 3, 1, 16, [40, 0, 7, 31]), (1, 8, 5, 8, [3, 64, 129]), (3, 4, 2, 32, [1, 95, 500, 0]), (2, 1, 33, 16, [0, 17]),
    (1, 5, 70, 64, [50, 0, 3]), (1, 12, 1, 128, [1300])])
def test_attention(fh, kind, dH, nKV, group, T, P, lens):
    rng = np.random.default_rng(dH + nKV + T)
    nSeq = len(lens)
    c = Cache(fh, rng, 2, nSeq, nKV, dH, P, -(-(max(lens) + T) // P) + 1, kind, lens)
    counts = [T if s == 0 else int(rng.integers(0, T + 1)) for s in range(nSeq)]
    c.fill(rng, 1, [n + t for n, t in zip(lens, counts)])
    check_attention(fh, c, rng, 1, nKV * group, T, counts)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (32, 0), (33, 40), (100, 3), (5000, 2), (64, 1 << 30)])
@pytest.mark.parametrize("dH,group,T", [(64, 2, 1), (128, 4, 9), (32, 1, 50)])
def test_window_and_sinks(fh, kind, window, sinks, dH, group, T):
    rng = np.random.default_rng(window + T)
    lens = [0, 230, 31, 700]
    c = Cache(fh, rng, 1, 4, 2, dH, 16, 48, kind, lens)
    c.fill(rng, 0, [n + T for n in lens])
    check_attention(fh, c, rng, 0, 2 * group, T, [T] * 4, window, sinks, given=False)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("T", [1, 6, 40])
def test_missing_pages_and_odd_lengths(fh, kind, T):
    """Slots of no page are not seen (a sequence without any gives zeros), nor is a length beyond the room taken at its word."""
    rng = np.random.default_rng(T)
    lens = [100, 77, 90, 10 ** 9, -8, 40]
    c = Cache(fh, rng, 1, 6, 2, 64, 8, 16, kind, lens)
    for p in (1, 2, 3, 7, 9):
        c.drop(0, p)
    for p in range(16):
        c.drop(1, p, c.nPages + p)
        if p >= 11:
            c.drop(2, p)
    c.drop(5, 0, -2147483648)
    c.fill(rng, 0, [128] * 6)
    got = check_attention(fh, c, rng, 0, 6, T, [T] * 6)
    assert (got[1] == 0).all()
    got = check_attention(fh, c, rng, 0, 6, T, [T] * 6, window=5, sinks=0)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("T,group", [(3, 2), (50, 1), (40, 4)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (2, 5), (30, 0)])
def test_windows_behind_the_end_of_the_room(fh, kind, T, group, window, sinks):
    """Queries of positions that the cache has no room for see what there is of their window, in caches that are cut into pieces."""
    rng = np.random.default_rng(T + window)
    c = Cache(fh, rng, 1, 3, 2, 64, 16, 70, kind, [1120, 1118, 600])
    c.fill(rng, 0, [1120, 1120, 600 + T])
    got = check_attention(fh, c, rng, 0, 2 * group, T, [T] * 3, window, sinks, given=False)
    if window and not sinks:
        assert (got[0, window:] == 0).all()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("dH,group,T,window", [(64, 1, 12, 0), (128, 4, 5, 0), (32, 2, 80, 0), (96, 3, 20, 9), (256, 1, 40, 30)])
def test_unseen_values_have_no_part(fh, kind, dH, group, T, window):
    """Infinities and NaN in later tokens' slots, behind the window and in unused slots leave what a query sees alone;
    a query that sees them is not finite where the formula is not."""
    rng = np.random.default_rng(T + dH)
    lens = [45, 0]
    c = Cache(fh, rng, 1, 2, 1, dH, 16, 9, kind, lens)
    k, v = c.fill(rng, 0, [n + T for n in lens])
    bad = {0: [45 + T // 2], 1: [T // 3]}
    for s in bad:
        for j in bad[s]:
            p, i = c.at(s, j)
            v[0, p, 0, i, :5] = [np.nan, np.inf, -np.inf, np.nan, np.inf]
    c.v.upload(v)
    nH = group
    q = rng.standard_normal((2, T, nH, dH)).astype(np.float32)
    out, dq = fh.DeviceArray.from_numpy(np.zeros(q.shape, np.float32)), fh.DeviceArray.from_numpy(q)
    scale = 1 / math.sqrt(dH)
    c.call("attn", 0, out, dq, nH, scale, T, None, window, 0)
    got = out.numpy()
    for s in range(2):
        n = lens[s] + T
        K, _ = ref.gather(k[0], c.table_host, 16, s, n)
        V, _ = ref.gather(v[0], c.table_host, 16, s, n)
        for t in range(T):
            seen = ref.sees(lens[s] + t, n, window, 0)
            hit = bool(seen[bad[s]].any())
            want, p = ref.attend(q[s, t], K, V, seen, scale)
            if hit:
                assert not np.isfinite(got[s, t, :, :5]).any(), (s, t)
                want, got_here = want[:, 5:], got[s, t, :, 5:]
            else:
                got_here = got[s, t]
            clean = np.where(np.isfinite(V), V, 0.0)
            bound = out_bound(q[s, t], K, clean, p, seen, scale, kind)[:, -got_here.shape[1]:]
            assert (np.abs(got_here - want) <= bound).all(), (s, t)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_keys_that_are_no_numbers(fh, kind):
    """A NaN key is seen by those queries that see its slot, and by no others; a NaN query harms its own row alone."""
    rng = np.random.default_rng(3)
    T, dH, lens = 30, 64, [20, 5]
    c = Cache(fh, rng, 1, 2, 2, dH, 8, 8, kind, lens)
    k, v = c.fill(rng, 0, [50, 35])
    p, i = c.at(0, 33)
    k[0, p, 1, i, 7] = np.nan
    c.k.upload(k)
    q = rng.standard_normal((2, T, 4, dH)).astype(np.float32)
    q[1, 11, 2, 5] = np.nan
    out, dq = fh.DeviceArray.from_numpy(np.zeros(q.shape, np.float32)), fh.DeviceArray.from_numpy(q)
    c.call("attn", 0, out, dq, 4, 0.125, T, None, 0, 0)
    bad = np.isnan(out.numpy()).any(-1)
    want = np.zeros((2, T, 4), bool)
    want[0, 13:, 2:] = True
    want[1, 11, 2] = True
    assert (bad == want).all()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("dH,T", [(64, 1), (128, 3), (128, 20)])
def test_large_and_small_scores(fh, kind, dH, T):
    """Scores of hundreds, of either sign, rising and falling over the slots, and a scale of zero and below it."""
    rng = np.random.default_rng(dH * T)
    lens = [300, 150]
    c = Cache(fh, rng, 1, 2, 2, dH, 16, 22, kind, lens)
    k, v = c.fill(rng, 0, [n + T for n in lens])
    grow = np.linspace(0.05, 6, 330)
    for s in range(2):
        for j in range(lens[s] + T):
            p, i = c.at(s, j)
            k[0, p, :, i] *= grow[j] if s == 0 else grow[329 - j]
    c.k.upload(k)
    for scale in (1.0, -1.0, 0.0, 1e-3):
        check_attention(fh, c, rng, 0, 4, T, [T, T], scale=scale)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("dH,group,T", [(64, 2, 1), (128, 4, 5), (32, 1, 40), (128, 4, 40), (256, 2, 3), (96, 3, 30)])
@pytest.mark.parametrize("nSeq", [1, 70, 200])
def test_pieces_of_many_sequences(fh, kind, dH, group, T, nSeq):
    """Caches that are cut into pieces, of lengths from nothing to long ones, more sequences than a wave has lanes, windows for some."""
    rng = np.random.default_rng(nSeq + T)
    longest = 2600 if nSeq == 1 else 700
    lens = [longest if s == 0 else int(longest * rng.random() ** 4) for s in range(nSeq)]
    counts = [T if s == 0 else int(rng.integers(0, T + 1)) for s in range(nSeq)]
    upto = [n + t for n, t in zip(lens, counts)]
    c = Cache(fh, rng, 1, nSeq, 1, dH, 16, -(-(2600 + T) // 16), kind, lens, upto=upto)
    c.fill(rng, 0, upto)
    check_attention(fh, c, rng, 0, group, T, counts)
    if nSeq < 100:
        check_attention(fh, c, rng, 0, group, T, counts, window=300, sinks=3)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("nSeq,nKV,group,T,dH", [(9, 8, 2, 70, 64), (43, 6, 2, 130, 64), (23, 3, 3, 90, 32), (64, 1, 5, 60, 128), (21, 3, 1, 200, 96)])
def test_many_heads_of_short_sequences(fh, kind, nSeq, nKV, group, T, dH):
    """A workgroup a head and tile, heads of sequences of all numbers of tokens on the dies in turn, numbers of heads that are no
    multiple of eight and some below the 64 that it takes."""
    rng = np.random.default_rng(nSeq + T)
    lens = [int(rng.integers(0, 40)) for _ in range(nSeq)]
    counts = [T if s == 0 else int(rng.integers(0, T + 1)) for s in range(nSeq)]
    upto = [n + t for n, t in zip(lens, counts)]
    c = Cache(fh, rng, 1, nSeq, nKV, dH, 16, -(-(40 + T) // 16), kind, lens, upto=upto)
    c.fill(rng, 0, upto)
    check_attention(fh, c, rng, 0, nKV * group, T, counts, window=5, sinks=2)


def test_a_long_cache(fh):
    """Offsets that pass 2^31 elements within a layer, the last slots of the room in use."""
    rng = np.random.default_rng(2)
    P, nKV, dH = 1024, 8, 128
    nPages = 2200  # 2200 x 8 x 1024 x 128 = 2.3e9 values a pool
    z = lambda: fh.DeviceArray.zeros((nPages, nKV, P, dH), np.float16)  # noqa: E731
    kp, vp = z(), z()
    table = np.array([[2199, 0, 2100, 2050, 1]], np.int32)
    lens = np.array([5 * P - 3], np.int32)
    up = fh.DeviceArray.from_numpy
    dt, dl = up(table), up(lens)
    cache = fh.PagedCache(1, 1, nKV, dH, P, nPages, 5, 1, kp.ptr, vp.ptr, dt.ptr, dl.ptr)
    T = 5 * P - 3
    k, v = (rng.standard_normal((T, nKV * dH)).astype(np.float32) for _ in range(2))
    dl.upload(np.zeros(1, np.int32))
    dk, dv = up(k), up(v)
    fh.call("paged_append", fh.ref(cache), 0, None, None, dk, dv, nKV * dH, 0, T, None, None, None, 0, 0, 0)
    fh.call("paged_commit", fh.ref(cache), T, None)
    assert (dl.numpy() == T).all()
    ok, ov = (fh.DeviceArray((T, nKV * dH)) for _ in range(2))
    fh.call("paged_read", fh.ref(cache), 0, ok, ov, nKV * dH, 0, T)
    K, V = k.astype(np.float16).astype(np.float64), v.astype(np.float16).astype(np.float64)
    assert (ok.numpy() == K).all() and (ov.numpy() == V).all()
    # two more tokens of three that came: the room ends at the third
    fh.call("paged_append", fh.ref(cache), 0, None, None, dk, dv, nKV * dH, 0, 3, None, None, None, 0, 0, 0)
    q = rng.standard_normal((3, 16, dH)).astype(np.float32)
    dq, out = up(q), fh.DeviceArray((3, 16, dH))
    fh.call("paged_attn", fh.ref(cache), 0, out, dq, 16, dH ** -0.5, 3, None, 0, 0)
    got = out.numpy()
    K, V = (np.concatenate([x, x[:3]]).reshape(-1, nKV, dH) for x in (K, V))
    for t in range(3):
        seen = np.arange(len(K)) <= T + t
        want, p = ref.attend(q[t], K, V, seen, dH ** -0.5)
        assert (np.abs(got[t] - want) <= out_bound(q[t], K, V, p, seen, dH ** -0.5, "f16")).all()
