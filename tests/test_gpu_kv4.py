"""The 4-bit key-value cache on the device (fg_kv4_*, fg_kv_evict_select)
against the plain 64-bit forms of oracle/kv4_ref.py: codes, steps, moves and
untouched slots exactly, attention within bounds counted from the roundings."""
import ctypes

import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu

HEADS = [32, 64, 96, 128, 256]


class Cache:
    """A cache on the device with every slot filled with what must not be seen:
    codes 0xFF, NaN steps and weights, position -7."""

    def __init__(self, fh, nLayers, nSeq, nKV, dH, maxSeq, track=True, lens=None):
        self.fh, self.dims = fh, (nLayers, nSeq, nKV, maxSeq)
        self.nSeq, self.nKV, self.dH, self.maxSeq, self.nb = nSeq, nKV, dH, maxSeq, dH // 32
        up = fh.DeviceArray.from_numpy
        self.k, self.v = (up(np.full(self.dims + (dH // 2,), 0xFF, np.uint8)) for _ in range(2))
        self.kd, self.vd = (up(np.full(self.dims + (self.nb,), np.nan, np.float16)) for _ in range(2))
        self.len = up(np.array(lens if lens is not None else [0] * nSeq, np.int32))
        self.next = up(np.arange(100, 100 + nSeq, dtype=np.int32))
        self.weight = up(np.full(self.dims, np.nan, np.float32)) if track else None
        self.pos = up(np.full(self.dims, -7, np.int32)) if track else None
        self.arrays = [a for a in (self.k, self.v, self.kd, self.vd, self.len, self.next, self.weight, self.pos)]
        self.struct = fh.Kv4Cache(nLayers, nSeq, nKV, dH, maxSeq, *[a.ptr if a else None for a in self.arrays])

    def call(self, name, *args):
        self.fh.call("kv4_" + name, self.fh.ref(self.struct), *args)

    def host(self):
        return [a.numpy() if a else None for a in self.arrays]

    def fill(self, rng, lens):
        """Random codes and steps, as if `lens` tokens had been stored."""
        code = rng.integers(0, 256, self.dims + (self.dH // 2,), dtype=np.uint8), rng.integers(0, 256, self.dims + (self.dH // 2,), dtype=np.uint8)
        step = [(rng.standard_normal(self.dims + (self.nb,)) * 0.2).astype(np.float16) for _ in range(2)]
        for s, n in enumerate(lens):
            for a in step:
                a[:, s, :, n:] = np.nan
        for d, a in zip((self.k, self.v, self.kd, self.vd), (*code, *step)):
            d.upload(a)
        if self.weight:
            self.weight.upload(np.exp(rng.standard_normal(self.dims)).astype(np.float32))


def rows(rng, *shape):
    x = rng.standard_normal(shape).astype(np.float32)
    return x * np.exp(rng.uniform(-3, 3, shape[-1])).astype(np.float32)


def attend_bound(q, K, V, p, scale, steps):
    """Bounds of |out| and |weight| errors, term by term: q in two fp16 pieces is off by 2^-22 of
    itself, a score's dH products and its nb block sums round at 2^-24 each (and scale, log2 e and the
    subtraction of the maximum, 4 more of the largest score), exp2 is good to 2^-22; p's and the sums over
    n positions round at most n / 4 + 64 times in a chain (a sum over a tile's positions stays in the
    matrix unit's order); p d is held in two fp16 pieces, 2^-22.  The pieces count from the greatest
    step and from a reference that the maximum may pass by 2^6 (and lies above 2^-6 of it): w = p d 2^(9 - E),
    2^E at most twice the greatest step, has an absolute error of 2^-25 where its low piece is subnormal,
    which is 2^-34 2^E <= 2^-33 max d of p d (and of less after the division by the sum of p, 1 or more),
    times |c - 8| <= 8, for each of n positions."""
    n, nKV, dH = K.shape
    nH = q.shape[0]
    out, weight = np.zeros((nH, dH)), np.zeros((nH, n))
    for h in range(nH if n else 0):
        z = h // (nH // nKV)
        mass = abs(scale) * (np.abs(K[:, z]) @ np.abs(q[h].astype(np.float64)))
        es = mass.max() * (2.0 ** -22 + (dH + 16) * 2.0 ** -24)
        rel = 2 * es + 2.0 ** -21 + (n / 4 + 64) * 2.0 ** -24
        out[h] = rel * (p[h] @ np.abs(V[:, z])) + n * 8 * 2.0 ** -33 * np.abs(steps[z].astype(np.float64)).max() + 1e-30
        weight[h] = rel * p[h] + 1e-30
    return out, weight


# ── store and read ────────────────────────────────────────────────────────
@pytest.mark.parametrize("dH", HEADS)
@pytest.mark.parametrize("nSeq,nKV,T,maxSeq,pad", [(1, 1, 1, 1, 0), (3, 2, 5, 17, 3), (2, 3, 40, 64, 0), (5, 5, 1, 9, 7)])
def test_append_and_read(fh, dH, nSeq, nKV, T, maxSeq, pad):
    rng = np.random.default_rng(dH + nSeq)
    lens = rng.integers(0, maxSeq, nSeq)
    c = Cache(fh, 2, nSeq, nKV, dH, maxSeq, lens=lens)
    before = c.host()
    ld = nKV * dH + pad
    k, v = rows(rng, nSeq * T, ld), rows(rng, nSeq * T, ld)
    count = rng.integers(-1, T + 2, nSeq).astype(np.int32)
    up = fh.DeviceArray.from_numpy
    dk, dv, dc = up(k), up(v), up(count)
    c.call("append", 1, dk, dv, ld, T, dc)
    got = c.host()
    want = [a.copy() for a in before]
    for s in range(nSeq):
        for t in range(min(max(count[s], 0), T)):
            at = lens[s] + t
            if at >= maxSeq:
                continue
            for x, codes, steps in ((k, 0, 2), (v, 1, 3)):
                q, d = ref.quantize(x[s * T + t, :nKV * dH].reshape(nKV, dH))
                want[codes][1, s, :, at], want[steps][1, s, :, at] = ref.pack(q), d
            want[6][1, s, :, at], want[7][1, s, :, at] = 0.0, 100 + s + t
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)
    first, n = maxSeq // 3, maxSeq - maxSeq // 3
    ok, ov = (fh.DeviceArray.from_numpy(np.full((nSeq * n, ld), 9.0, np.float32)) for _ in range(2))
    c.call("read", 1, ok, ov, ld, first, n)
    for o, codes, steps in ((ok, 0, 2), (ov, 1, 3)):
        g = o.numpy()
        x = ref.values(want[codes][1], want[steps][1])[:, :, first:].transpose(0, 2, 1, 3).reshape(nSeq * n, nKV * dH)
        np.testing.assert_array_equal(g[:, :nKV * dH], x.astype(np.float32))
        assert (g[:, nKV * dH:] == 9.0).all()


@pytest.mark.parametrize("dH", HEADS)
def test_append_edges(fh, dH):
    """Zeros, equal magnitudes of both signs, borders between codes, tiny and huge blocks, what is not finite."""
    rng = np.random.default_rng(dH)
    T = 600
    x = rows(rng, T, dH)
    x[0] = 0.0
    x[1, 3], x[1, 7], x[2, 3], x[2, 7] = 50.0, -50.0, -50.0, 50.0
    x[3, 20], x[3, 4] = 50.0, -50.0
    x[4, 5], x[5, 5], x[6, 5], x[7, 5] = np.nan, np.inf, -np.inf, 8 * 65519.0
    x[8, 5], x[9, 5], x[10] = 8 * 65520.0, -3e38, x[10] * 1e-8
    x[11], x[12], x[13] = x[11] * 1e-30, x[12] * 1e-42, -0.0
    for r in range(14, 300):  # values on and next to the borders (c + 1/2) d
        d = np.float16(rng.standard_normal() * np.exp(rng.uniform(-10, 6)))
        x[r] = np.float32(d) * (rng.integers(-8, 8, dH) - np.float32(0.5))
        x[r, ::32] = np.float32(d) * -8
        near = rng.random(dH) < 0.4
        x[r] = np.where(near, np.nextafter(x[r], np.float32(np.inf) * rng.choice([-1, 1], dH).astype(np.float32)), x[r])
    c = Cache(fh, 1, 1, 1, dH, T)
    up = fh.DeviceArray.from_numpy
    dx = up(x)
    c.call("append", 0, dx, dx, dH, T, None)
    q, d = ref.quantize(x)
    got = c.host()
    for codes, steps in ((0, 2), (1, 3)):
        np.testing.assert_array_equal(got[steps][0, 0, 0], d)
        good = np.repeat(np.isfinite(d), 16, -1).reshape(T, -1, 16).transpose(0, 2, 1).reshape(T, -1)
        np.testing.assert_array_equal(got[codes][0, 0, 0][good], ref.pack(q)[good])
    out = fh.DeviceArray((T, dH))
    out2 = fh.DeviceArray((T, dH))
    c.call("read", 0, out, out2, dH, 0, T)
    np.testing.assert_array_equal(out.numpy(), ref.values(ref.pack(q), d).astype(np.float32))
    np.testing.assert_array_equal(out2.numpy(), out.numpy())


@pytest.mark.parametrize("kind", ["zero", "tie", "overflow", "almost", "inf", "nan", "tiny", "one"])
def test_append_edges_alone(fh, kind):
    """Every row of the same kind, so that none takes its neighbours' path."""
    rng = np.random.default_rng(3)
    T, dH = 64, 64
    x = rows(rng, T, dH)
    far = x.reshape(T, 2, 32)
    if kind == "zero":
        x[:] = 0.0
    elif kind == "one":
        x[:] = 0.0
        far[:, :, 5] = rng.standard_normal((T, 2))
    elif kind == "tie":
        far[:, :, 30], far[:, :, 2] = 99.0, -99.0
    elif kind == "tiny":
        x *= 1e-7
    else:
        far[:, :, 9] = {"overflow": -8 * 65520.0, "almost": 8 * 65519.0, "inf": -np.inf, "nan": np.nan}[kind]
    c = Cache(fh, 1, 1, 1, dH, T)
    d = fh.DeviceArray.from_numpy(x)
    c.call("append", 0, d, d, dH, T, None)
    ok, ov = fh.DeviceArray((T, dH)), fh.DeviceArray((T, dH))
    c.call("read", 0, ok, ov, dH, 0, T)
    codes, steps = ref.quantize(x)
    np.testing.assert_array_equal(ok.numpy(), ref.values(ref.pack(codes), steps).astype(np.float32))
    np.testing.assert_array_equal(ov.numpy(), ok.numpy())


# ── attention ─────────────────────────────────────────────────────────────
def check_attend(fh, c, nH, rng, lens, T=0, count=None, scale=None, q=None, layer=0):
    scale = 1 / np.sqrt(c.dH) if scale is None else scale
    q = rng.standard_normal((c.nSeq, nH, c.dH)).astype(np.float32) if q is None else q
    before = c.host()
    up = fh.DeviceArray.from_numpy
    dq, out = up(q), up(np.full(q.shape, 7.0, np.float32))
    dc = up(np.array(count, np.int32)) if count is not None else None
    c.call("attn", layer, out, dq, nH, scale, T, dc)
    after = c.host()
    for i, (a, b) in enumerate(zip(before, after)):
        if i != 6 and a is not None:
            np.testing.assert_array_equal(a, b)
    got = out.numpy()
    for s in range(c.nSeq):
        n = min(max(lens[s], 0), c.maxSeq)
        n = min(n + (T if count is None else min(max(count[s], 0), T)), c.maxSeq)
        K = ref.values(before[0][layer, s, :, :n], before[2][layer, s, :, :n]).transpose(1, 0, 2)
        V = ref.values(before[1][layer, s, :, :n], before[3][layer, s, :, :n]).transpose(1, 0, 2)
        want, p = ref.attend(q[s], K, V, scale)
        eo, ew = attend_bound(q[s], K, V, p, scale, before[3][layer, s, :, :n])
        assert np.isfinite(got[s]).all(), (s, n)
        worst = (np.abs(got[s] - want) / eo).max() if n else np.abs(got[s]).max()
        assert worst <= (1.0 if n else 0.0), (s, n, worst)
        if before[6] is not None:
            group = nH // c.nKV
            add = p.reshape(c.nKV, group, n).sum(1)
            tol = ew.reshape(c.nKV, group, n).sum(1)
            w0, w1 = before[6][layer, s], after[6][layer, s]
            np.testing.assert_array_equal(w1[:, n:], w0[:, n:])
            # the sum of the group's heads and the addition round at 2^-24 each
            off = np.abs(w1[:, :n] - (w0[:, :n].astype(np.float64) + add))
            assert (off <= tol + (group + 1) * 2.0 ** -24 * (np.abs(w1[:, :n]) + add)).all()
            for other in range(c.dims[0]):
                if other != layer:
                    np.testing.assert_array_equal(before[6][other], after[6][other])


@pytest.mark.parametrize("dH", HEADS)
@pytest.mark.parametrize("nKV,group", [(1, 1), (2, 4), (3, 3), (1, 8), (2, 12)])
def test_attend(fh, dH, nKV, group):
    rng = np.random.default_rng(dH * 31 + nKV)
    lens = [0, 1, 31, 32, 33, 129, 200, 517]
    c = Cache(fh, 2, len(lens), nKV, dH, 517, lens=lens)
    c.fill(rng, lens)
    check_attend(fh, c, nKV * group, rng, lens, layer=1)


@pytest.mark.parametrize("dH,group", [(32, 2), (64, 1), (96, 5), (128, 4), (256, 8)])
@pytest.mark.parametrize("n", [1, 63, 64, 65, 127, 128, 257, 1024, 3333])
def test_attend_one_sequence(fh, dH, group, n):
    rng = np.random.default_rng(n)
    c = Cache(fh, 1, 1, 1, dH, n + rng.integers(0, 40), track=n % 2 == 0, lens=[n])
    c.fill(rng, [n])
    check_attend(fh, c, group, rng, [n])


@pytest.mark.parametrize("dH", HEADS)
@pytest.mark.parametrize("nKV,group,track", [(1, 1, True), (2, 4, False), (2, 3, True), (1, 12, True), (1, 20, False)])
def test_attend_in_pieces(fh, dH, nKV, group, track):
    """Room for far more slots than are in use: the cache is read in pieces whose sizes come from the lengths on the device."""
    rng = np.random.default_rng(dH * 7 + group)
    lens = [0, 1, 32, 127, 128, 129, 700, 1500]
    c = Cache(fh, 1, len(lens), nKV, dH, 9000 // group * 2, lens=lens, track=track)
    c.fill(rng, lens)
    check_attend(fh, c, nKV * group, rng, lens)


@pytest.mark.parametrize("nSeq,maxSeq", [(65, 40), (70, 6000), (130, 9000), (200, 3)])
def test_attend_many_sequences(fh, nSeq, maxSeq):
    """More sequences than a wave has lanes, most of them short, some empty."""
    rng = np.random.default_rng(nSeq)
    lens = [int(n) for n in rng.choice([0, 1, 5, 33, 140, 300], nSeq) % (maxSeq + 1)]
    lens[nSeq // 2] = min(maxSeq, 2000)
    c = Cache(fh, 1, nSeq, 1, 32, maxSeq, lens=lens, track=nSeq != 70)
    c.fill(rng, lens)
    check_attend(fh, c, 2, rng, lens)


@pytest.mark.parametrize("T,count", [(3, None), (3, [0, 1, 2, 3]), (3, [9, -4, 3, 0])])
def test_attend_new_tokens_and_bad_lengths(fh, T, count):
    """Lengths and counts outside their ranges count as the nearest inside; new tokens are attended to before the commit."""
    rng = np.random.default_rng(T)
    lens = [50, 0, 39, -3]
    c = Cache(fh, 1, 4, 2, 64, 40, lens=lens)
    c.fill(rng, [40] * 4)
    check_attend(fh, c, 6, rng, lens, T=T, count=count)


@pytest.mark.parametrize("dH", HEADS)
def test_attend_peaks_and_scales(fh, dH):
    """One slot that takes all, large and tiny steps, a scale of zero, negative scales, a zero query."""
    rng = np.random.default_rng(dH + 5)
    lens = [300, 40, 77]
    c = Cache(fh, 1, 3, 2, dH, 300, lens=lens)
    c.fill(rng, lens)
    kd, vd = c.kd.numpy(), c.vd.numpy()
    kd[0, 0, :, 211] = 12.0
    vd[0, 1] = vd[0, 1] * np.float16(2e4)
    vd[0, 2, :, 5:] = vd[0, 2, :, 5:] * np.float16(1e-4)
    c.kd.upload(kd)
    c.vd.upload(vd)
    q = rng.standard_normal((3, 4, dH)).astype(np.float32)
    q[2, 1] = 0.0
    q[1, 2] *= 1e-20
    for scale in (0.1, -0.05, 0.0):
        check_attend(fh, c, 4, rng, lens, scale=scale, q=q)


def test_attend_steps_of_very_different_sizes(fh):
    """Values whose steps grow and shrink by large factors along the cache: the running scale of the value products follows."""
    rng = np.random.default_rng(8)
    n = 2048
    c = Cache(fh, 1, 1, 1, 128, n, lens=[n])
    c.fill(rng, [n])
    for factors in (np.linspace(-14, 12, n), np.linspace(12, -14, n), rng.uniform(-14, 12, n)):
        vd = (rng.uniform(1, 2, (1, 1, 1, n, 4)) * np.exp2(factors)[None, None, None, :, None]).astype(np.float16)
        c.vd.upload(vd)
        check_attend(fh, c, 4, rng, [n], scale=0.02)


def test_attend_not_finite(fh):
    """A NaN key or value of a slot in use shows in its kv head's outputs and nowhere else."""
    rng = np.random.default_rng(9)
    lens = [100, 100]
    c = Cache(fh, 1, 2, 2, 64, 128, lens=lens, track=False)
    c.fill(rng, lens)
    kd, vd = c.kd.numpy(), c.vd.numpy()
    kd[0, 0, 1, 50, 1] = np.nan
    vd[0, 1, 0, 99, 0] = np.nan
    c.kd.upload(kd)
    c.vd.upload(vd)
    q = fh.DeviceArray.from_numpy(rng.standard_normal((2, 4, 64)).astype(np.float32))
    out = fh.DeviceArray.from_numpy(np.zeros((2, 4, 64), np.float32))
    c.call("attn", 0, out, q, 4, 0.125, 0, None)
    bad = np.isnan(out.numpy())
    assert bad[0, 2:].all() and not bad[0, :2].any()
    assert bad[1, :2, :32].all() and not bad[1, :, 32:].any() and not bad[1, 2:].any()


def test_attend_far_into_a_large_cache(fh):
    """Codes past 2^32 bytes from the arrays' start."""
    nLayers, maxSeq, dH, nKV = 9, 1 << 19, 256, 8
    up = fh.DeviceArray
    shape = (nLayers, 1, nKV, maxSeq)
    assert np.prod(shape) * 128 > 2 ** 32
    k, v = up(shape + (128,), np.uint8), up(shape + (128,), np.uint8)
    kd, vd = up(shape + (8,), np.float16), up(shape + (8,), np.float16)
    n = maxSeq - 3
    length, nxt = up.from_numpy(np.array([n], np.int32)), up.from_numpy(np.array([n], np.int32))
    c = fh.Kv4Cache(nLayers, 1, nKV, dH, maxSeq, k.ptr, v.ptr, kd.ptr, vd.ptr, length.ptr, nxt.ptr, None, None)
    rng = np.random.default_rng(1)
    row = np.zeros((1, nKV * dH), np.float32)
    zero, one = up.from_numpy(row), up.from_numpy(rng.standard_normal((1, nKV * dH)).astype(np.float32))
    for layer in (0, nLayers - 1):
        fh.call("kv4_append", fh.ref(c), layer, one, one, nKV * dH, 1, None)
    ok, ov = up((1, nKV * dH)), up((1, nKV * dH))
    fh.call("kv4_read", fh.ref(c), nLayers - 1, ok, ov, nKV * dH, n, 1)
    q, d = ref.quantize(one.numpy().reshape(nKV, dH))
    np.testing.assert_array_equal(ok.numpy().reshape(nKV, dH), ref.values(ref.pack(q), d).astype(np.float32))
    # all slots in use of the last head but the last hold zeros: uniform weights
    for a in (kd, vd):
        fh.check(fh.lib.fg_zero(ctypes.c_void_p(a.ptr), a.nbytes), "fg_zero")
    fh.call("kv4_append", fh.ref(c), nLayers - 1, zero, one, nKV * dH, 1, None)
    out = up((nKV, dH))
    fh.call("kv4_attn", fh.ref(c), nLayers - 1, out, one, nKV, 0.1, 1, None)
    want = ref.values(ref.pack(q), d) / (n + 1)
    np.testing.assert_allclose(out.numpy(), want, rtol=2.0 ** -13)  # the weights' sum: 2^19 ones in fp32


# ── eviction ──────────────────────────────────────────────────────────────
def run_select(fh, weight, pos, lens, nxt, budget, recent):
    nL, nS, nH, maxSeq = weight.shape
    most = max(1, min(budget, maxSeq - budget))
    up = fh.DeviceArray.from_numpy
    holes, movers = (up(np.full((nL, nS, nH, most), 77, np.int32)) for _ in range(2))
    moves = up(np.full((nL, nS, nH), 77, np.int32))
    a = [up(x) for x in (weight, pos, np.array(lens, np.int32), np.array(nxt, np.int32))]
    fh.call("kv_evict_select", holes, movers, moves, *a, nL, nS, nH, maxSeq, budget, recent)
    return holes.numpy(), movers.numpy(), moves.numpy()


def check_select(fh, weight, pos, lens, nxt, budget, recent):
    holes, movers, moves = run_select(fh, weight, pos, lens, nxt, budget, recent)
    maxSeq = weight.shape[-1]
    for l, s, h in np.ndindex(weight.shape[:3]):
        n = min(max(lens[s], 0), maxSeq)
        wh, wm = ref.evict(weight[l, s, h], pos[l, s, h], n, nxt[s], budget, recent)
        m = moves[l, s, h]
        assert m == len(wh) == len(wm)
        np.testing.assert_array_equal(holes[l, s, h], wh + [-1] * (holes.shape[-1] - m))
        np.testing.assert_array_equal(movers[l, s, h], wm + [-1] * (holes.shape[-1] - m))


def positions(rng, *shape):
    return rng.permuted(np.broadcast_to(np.arange(shape[-1], dtype=np.int32), shape), axis=-1)


@pytest.mark.parametrize("maxSeq", [2, 5, 63, 64, 65, 1000, 1024, 1025, 4096, 4097, 9000, 17000, 33000])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_select(fh, maxSeq, ties):
    rng = np.random.default_rng(maxSeq)
    for budget in sorted({1, maxSeq // 4 + 1, maxSeq // 2 + 1, maxSeq - 1}):
        if not 1 <= budget < maxSeq:
            continue
        w = np.exp(rng.standard_normal((2, 3, 2, maxSeq)) * 2).astype(np.float32)
        if ties:
            w = np.floor(w).astype(np.float32)
        lens = [maxSeq, rng.integers(0, maxSeq + 1), min(budget + 1, maxSeq)]
        for recent in {0, budget // 2, budget}:
            check_select(fh, w, positions(rng, 2, 3, 2, maxSeq), lens, [maxSeq] * 3, budget, recent)


@pytest.mark.parametrize("maxSeq", [32769, 65535, 65536, 65537, 70001, 150000])
def test_evict_select_long(fh, maxSeq):
    """Long heads: spread and even weights, all equal, all slots recent; budgets at either end."""
    rng = np.random.default_rng(maxSeq)
    w = np.exp(rng.standard_normal((1, 2, 3, maxSeq)) * 2).astype(np.float32)
    w[0, :, 1] = np.floor(w[0, :, 1])
    w[0, :, 2] = 1.5
    pos = positions(rng, 1, 2, 3, maxSeq)
    for budget, recent in ((1, 1), (maxSeq // 2 + 1, 1000), (maxSeq // 2, maxSeq // 2), (maxSeq - 1, 0)):
        check_select(fh, w, pos, [maxSeq, maxSeq - 77], [maxSeq] * 2, budget, recent)


def test_evict_select_odd_weights(fh):
    """All equal, zeros of both signs, negative, NaN and infinite weights; every slot recent; lengths out of range."""
    rng = np.random.default_rng(4)
    n = 300
    w = np.zeros((1, 5, 4, n), np.float32)
    w[0, :, 1] = rng.choice(np.array([0.0, -0.0], np.float32), n)
    w[0, :, 2] = rng.choice(np.array([-1, np.nan, np.inf, -np.inf, 2, 1e-40, -1e-40], np.float32), n)
    w[0, :, 3] = np.nan
    lens = [n, n + 50, -4, 0, 151]
    for budget, recent in ((150, 0), (150, 20), (150, 150), (1, 1), (299, 3)):
        check_select(fh, w, positions(rng, 1, 5, 4, n), lens, [n] * 5, budget, recent)


@pytest.mark.parametrize("maxSeq", [100, 5000, 20000, 40000])
def test_evict_select_more_recent_than_the_budget(fh, maxSeq):
    """Positions that say so against the rules: the lowest of those slots are kept, and nothing waits for more."""
    rng = np.random.default_rng(maxSeq)
    w = np.exp(rng.standard_normal((1, 2, 1, maxSeq))).astype(np.float32)
    pos = np.full(w.shape, maxSeq, np.int32)
    pos[0, 1, 0, ::3] = 0
    for budget in (1, maxSeq // 3, maxSeq - 1):
        check_select(fh, w, pos, [maxSeq, maxSeq - 1], [maxSeq] * 2, budget, budget // 2)


@pytest.mark.parametrize("dH", HEADS)
@pytest.mark.parametrize("maxSeq,budget,recent", [(33, 32, 4), (200, 50, 10), (200, 150, 0), (2100, 2048, 256)])
def test_evict(fh, dH, maxSeq, budget, recent):
    rng = np.random.default_rng(dH + maxSeq)
    lens = [maxSeq, budget, maxSeq - 1, 0]
    c = Cache(fh, 2, 4, 2, dH, maxSeq, lens=lens)
    c.fill(rng, [maxSeq] * 4)
    c.pos.upload(positions(rng, *c.dims))
    c.next.upload(np.array([maxSeq] * 4, np.int32))
    before = c.host()
    c.call("evict", budget, recent)
    want = [a.copy() for a in before]
    for l, s, h in np.ndindex(c.dims[:3]):
        holes, movers = ref.evict(before[6][l, s, h], before[7][l, s, h], lens[s], maxSeq, budget, recent)
        for i in (0, 1, 2, 3, 6, 7):
            want[i][l, s, h, holes] = before[i][l, s, h, movers]
    want[4] = np.minimum(lens, budget)
    for a, b in zip(c.host(), want):
        np.testing.assert_array_equal(a, b)
    c.call("evict", budget, recent)  # nothing is over the budget any more
    c.call("evict", maxSeq + 5, 0)
    for a, b in zip(c.host(), want):
        np.testing.assert_array_equal(a, b)


def test_commit(fh):
    c = Cache(fh, 1, 5, 1, 32, 20, lens=[0, 19, 25, -2, 7])
    c.call("commit", 3, None)
    np.testing.assert_array_equal(c.len.numpy(), [3, 20, 20, 3, 10])
    np.testing.assert_array_equal(c.next.numpy(), np.arange(100, 105) + 3)
    c.call("commit", 3, fh.DeviceArray.from_numpy(np.array([0, 1, -2, 8, 2], np.int32)))
    np.testing.assert_array_equal(c.len.numpy(), [3, 20, 20, 6, 12])
    np.testing.assert_array_equal(c.next.numpy(), np.arange(100, 105) + 3 + np.array([0, 1, 0, 3, 2]))


@pytest.mark.parametrize("maxSeq", [40, 9000])
def test_more_new_tokens_than_32_bits_add_up(fh, maxSeq):
    """A step of as many tokens as an int holds fills the sequences; nothing wraps round."""
    most = 2 ** 31 - 1
    rng = np.random.default_rng(maxSeq)
    lens = [0, 7, maxSeq]
    c = Cache(fh, 1, 3, 1, 64, maxSeq, lens=lens)
    c.fill(rng, [maxSeq] * 3)
    check_attend(fh, c, 2, rng, lens, T=most)
    check_attend(fh, c, 2, rng, lens, T=most, count=[most, 0, -most - 1])
    c.next.upload(np.array([0, -5, 0], np.int32))
    c.call("commit", most, fh.DeviceArray.from_numpy(np.array([most, most, 1], np.int32)))
    np.testing.assert_array_equal(c.len.numpy(), [maxSeq] * 3)
    np.testing.assert_array_equal(c.next.numpy(), [most, most - 5, 1])


# ── together ──────────────────────────────────────────────────────────────
@pytest.mark.parametrize("W", [1, 3, 4])
def test_reorder(fh, W):
    rng = np.random.default_rng(W)
    lens = rng.integers(0, 38, 2 * W)
    c = Cache(fh, 3, 2 * W, 2, 96, 37, lens=lens)
    c.fill(rng, [37] * 2 * W)
    c.pos.upload(positions(rng, *c.dims))
    parent = rng.integers(-1, W + 1, 2 * W).astype(np.int32)
    before = c.host()
    c.call("reorder", fh.DeviceArray.from_numpy(parent), W)
    want = [a.copy() for a in before]
    for b in range(2 * W):
        p = b // W * W + parent[b] if 0 <= parent[b] < W else b
        for i in (0, 1, 2, 3, 6, 7):
            want[i][:, b, :, :lens[p]] = before[i][:, p, :, :lens[p]]
        want[4][b], want[5][b] = before[4][p], before[5][p]
    for a, b in zip(c.host(), want):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("dH,nKV,group", [(32, 2, 2), (128, 1, 4)])
def test_a_generation_under_a_budget(fh, dH, nKV, group):
    """Prompts of their own lengths, then steps of append, attend, commit, evict, with two beams changing places."""
    rng = np.random.default_rng(dH)
    budget, recent, nSeq = 24, 6, 2
    c = Cache(fh, 2, nSeq, nKV, dH, 40)
    nH = nKV * group
    up = fh.DeviceArray.from_numpy
    c.next.upload(np.zeros(nSeq, np.int32))
    lens, seen = [0, 0], [0, 0]
    for step in range(30):
        T, count = (9, [9, 4]) if step == 0 else (1, None)
        per = count or [T] * nSeq
        for layer in range(2):
            k, v = rows(rng, nSeq * T, nKV * dH), rows(rng, nSeq * T, nKV * dH)
            dc = up(np.array(count, np.int32)) if count else None
            c.call("append", layer, up(k), up(v), nKV * dH, T, dc)
            check_attend(fh, c, nH, rng, lens, T=T, count=count, layer=layer)
        c.call("commit", T, dc)
        lens, seen = [n + a for n, a in zip(lens, per)], [n + a for n, a in zip(seen, per)]
        np.testing.assert_array_equal(c.len.numpy(), lens)
        before = c.host()
        c.call("evict", budget, recent)
        want = [a.copy() for a in before]
        for l, s, h in np.ndindex(c.dims[:3]):
            holes, movers = ref.evict(before[6][l, s, h], before[7][l, s, h], lens[s], seen[s], budget, recent)
            for i in (0, 1, 2, 3, 6, 7):
                want[i][l, s, h, holes] = before[i][l, s, h, movers]
        lens = [min(n, budget) for n in lens]
        want[4] = np.array(lens, np.int32)
        for a, b in zip(c.host(), want):
            np.testing.assert_array_equal(a, b)
        if step % 7 == 3:
            c.call("reorder", up(np.array([1, 1] if step == 3 else [1, 0], np.int32)), 2)
            lens, seen = ([lens[1]] * 2, [seen[1]] * 2) if step == 3 else (lens[::-1], seen[::-1])
    pos = c.pos.numpy()
    for l, s, h in np.ndindex(c.dims[:3]):  # the newest are there, once each
        kept = pos[l, s, h, :lens[s]]
        assert len(set(kept)) == len(kept) and set(range(seen[s] - recent, seen[s])) <= set(kept)


def test_a_recorded_step_replays(fh):
    """A graph of a step under a budget, replayed with eager work between, gives what the same eager steps give."""
    rng = np.random.default_rng(2)
    budget, nSeq, nKV, dH, nH = 60, 3, 2, 64, 4
    up = fh.DeviceArray.from_numpy
    k, v = (up(np.zeros((nSeq, nKV * dH), np.float32)) for _ in range(2))
    q = up(np.zeros((nSeq, nH, dH), np.float32))
    results = []
    for graph in (False, True):
        r = np.random.default_rng(6)
        c = Cache(fh, 1, nSeq, nKV, dH, 64, lens=[60, 30, 59])
        c.fill(np.random.default_rng(5), [60] * 3)
        c.pos.upload(positions(np.random.default_rng(7), *c.dims))
        out = up(np.zeros((nSeq, nH, dH), np.float32))
        parent = up(np.array([0, 0, 2], np.int32))

        def step():
            c.call("append", 0, k, v, nKV * dH, 1, None)
            c.call("attn", 0, out, q, nH, 0.125, 1, None)
            c.call("commit", 1, None)
            c.call("evict", budget, 10)
            c.call("reorder", parent, 3)

        handle = ctypes.c_void_p()
        if graph:
            fh.check(fh.lib.fg_graph_begin(), "begin")
            step()
            fh.check(fh.lib.fg_graph_end(ctypes.byref(handle)), "end")
        got = []
        for i in range(5):
            for d, shape in ((k, (nSeq, nKV * dH)), (v, (nSeq, nKV * dH)), (q, (nSeq, nH, dH))):
                d.upload(r.standard_normal(shape).astype(np.float32))
            if graph:
                fh.check(fh.lib.fg_graph_launch(handle), "launch")
                junk = [up(rng.standard_normal(50000).astype(np.float32)) for _ in range(3)]
                fh.sync()
                del junk
            else:
                step()
            got.append([a.copy() for a in c.host()] + [out.numpy()])
        if graph:
            fh.check(fh.lib.fg_graph_destroy(handle), "destroy")
        results.append(got)
    for a, b in zip(*results):
        for x, y in zip(a, b):
            np.testing.assert_array_equal(x, y)


def test_two_recorded_steps_take_turns(fh):
    """Graphs over two caches, and a beam choice in one of them, launched in turn without a wait between:
    neither's working memory is the other's."""
    up = fh.DeviceArray.from_numpy
    sizes = [(9000, 2, 64, 4, 300), (2500, 4, 128, 8, 700)]  # slots, kv heads, head size, query heads, budget
    results = []
    for graphs in (False, True):
        r = np.random.default_rng(3)
        parts, steps = [], []
        for maxSeq, nKV, dH, nH, budget in sizes:
            c = Cache(fh, 1, 4, nKV, dH, maxSeq, lens=[2000, 10, 1999, 700])
            c.fill(np.random.default_rng(dH), [maxSeq] * 4)
            c.pos.upload(positions(np.random.default_rng(nH), *c.dims))
            c.next.upload(np.full(4, maxSeq, np.int32))
            kv = [up(r.standard_normal((4, nKV * dH)).astype(np.float32)) for _ in range(2)]
            q, out = up(r.standard_normal((4, nH, dH)).astype(np.float32)), up(np.zeros((4, nH, dH), np.float32))
            logits, scores = up(r.standard_normal((4, 20000)).astype(np.float32)), up(np.zeros(4, np.float32))
            picked = [up(np.zeros(4, d)) for d in (np.float32, np.int32, np.int32)]
            parts.append((c, out, picked))

            def step(c=c, kv=kv, q=q, out=out, logits=logits, scores=scores, picked=picked, nH=nH, dH=dH, nKV=nKV, budget=budget):
                c.call("append", 0, *kv, nKV * dH, 1, None)
                c.call("attn", 0, out, q, nH, 0.125, 1, None)
                c.call("commit", 1, None)
                fh.call("beam_select", *picked, None, logits, 20000, scores, None, -1, 1, 4, 20000)
                c.call("reorder", picked[2], 4)
                c.call("evict", budget, 10)

            steps.append(step)
        handles = []
        if graphs:
            for step in steps:
                h = ctypes.c_void_p()
                fh.check(fh.lib.fg_graph_begin(), "begin")
                step()
                fh.check(fh.lib.fg_graph_end(ctypes.byref(h)), "end")
                handles.append(h)
        for turn in (0, 1, 0, 1, 1, 0):
            if graphs:
                fh.check(fh.lib.fg_graph_launch(handles[turn]), "launch")
            else:
                steps[turn]()
        results.append([x for c, out, picked in parts for x in c.host() + [out.numpy()] + [p.numpy() for p in picked]])
        for h in handles:
            fh.check(fh.lib.fg_graph_destroy(h), "destroy")
    for x, y in zip(*results):
        np.testing.assert_array_equal(x, y)
