"""Beam search on the device (fg_beam_select, fg_beam_reorder) against the plain
64-bit forms of oracle/kv4_ref.py: tokens, parents and moved bytes exactly."""
import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu


def select(fh, logits, scores, done, eos, nReq, W, V, offset=0):
    """Logits [nReq W, ld >= V], `offset` floats into their allocation."""
    up = fh.DeviceArray.from_numpy
    n = nReq * W
    flat = np.concatenate([np.zeros(offset, np.float32), logits.ravel()])
    dl, ds = up(flat), up(scores)
    dd = up(done.astype(np.int32)) if done is not None else None
    score = up(np.full(n, 5.0, np.float32))
    token, parent = (up(np.full(n, -9, np.int32)) for _ in range(2))
    fin = up(np.full(n, -9, np.int32)) if done is not None else None
    fh.call("beam_select", score, token, parent, fin, dl.ptr + 4 * offset, logits.shape[1], ds, dd, eos, nReq, W, V)
    return score.numpy(), token.numpy(), parent.numpy(), fin.numpy() if fin else None


def check(fh, logits, scores, done, eos, nReq, W, V, offset=0):
    got = select(fh, logits, scores, done, eos, nReq, W, V, offset)
    want = ref.beam_select(logits[:, :V], scores, done, eos, nReq, W)
    np.testing.assert_array_equal(got[2], want[2])
    np.testing.assert_array_equal(got[1], want[1])
    # one rounding to fp32, and the log of a sum whose terms are good to 2^-21
    fine = np.isfinite(want[0])
    assert (np.abs(got[0] - want[0])[fine] <= 2.0 ** -24 * np.abs(want[0][fine]) + 2.0 ** -20).all()
    np.testing.assert_array_equal(got[0][~fine], want[0][~fine])
    if done is not None:
        np.testing.assert_array_equal(got[3], want[3])


@pytest.mark.parametrize("W", [1, 2, 3, 4, 7, 8, 16, 31, 32, 33, 64])
@pytest.mark.parametrize("V", [1, 2, 31, 64, 257, 1000, 4096, 32000])
def test_select(fh, W, V):
    rng = np.random.default_rng(W * 100000 + V)
    nReq = 3
    x = (rng.standard_normal((nReq * W, V)) * 3).astype(np.float32)
    scores = (-rng.random(nReq * W) * 10).astype(np.float32)
    check(fh, x, scores, None, -1, nReq, W, V)
    done = rng.random(nReq * W) < 0.3
    check(fh, x, scores, done, V // 2, nReq, W, V)


@pytest.mark.parametrize("W", [1, 4, 8, 40])
@pytest.mark.parametrize("V,pad,offset", [(999, 1, 1), (4097, 3, 2), (128256, 0, 0), (2048, 5, 3)])
def test_select_ties_and_strides(fh, W, V, pad, offset):
    """Coarse logits: many equal values, inside a beam and at the border of the choice; rows off their alignment."""
    rng = np.random.default_rng(V + W)
    x = np.round(rng.standard_normal((2 * W, V + pad)) * 4).astype(np.float32) / 2
    x[:, V:] = 100.0  # behind the rows
    check(fh, x, (-rng.random(2 * W) * 3).astype(np.float32), None, -1, 2, W, V, offset)
    x[:] = 1.25  # all equal, in all beams
    x[:, V:] = 100.0
    check(fh, x, np.full(2 * W, -2.5, np.float32), None, -1, 2, W, V, offset)


@pytest.mark.parametrize("V", [5, 700, 9000])
def test_select_masks_and_what_is_not_finite(fh, V):
    rng = np.random.default_rng(V)
    W = 8
    x = (rng.standard_normal((5 * W, V)) * 2).astype(np.float32)
    scores = (-rng.random(5 * W) * 4).astype(np.float32)
    x[0:W][:, rng.random(V) < 0.7] = -np.inf  # masked tokens
    x[0, :] = -np.inf                        # a beam of masked tokens alone
    x[W:2 * W] = -np.inf                     # a request of them
    x[2 * W + 1, V // 2] = np.nan
    x[2 * W + 2, V - 1] = np.inf
    x[2 * W + 3, :] = np.nan
    scores[3 * W + 1:4 * W] = -np.inf        # the first step: one beam counts
    scores[4 * W], scores[4 * W + 1], scores[4 * W + 2] = np.nan, np.inf, -np.inf
    x[4 * W + 4] *= 1e30
    x[4 * W + 5] *= 1e-30
    check(fh, x, scores, None, -1, 5, W, V)
    done = np.zeros(5 * W, bool)
    done[[0, 5, W, 2 * W + 1, 4 * W, 4 * W + 2]] = True
    check(fh, x, scores, done, 0, 5, W, V)
    check(fh, x, scores, np.ones(5 * W, bool), V - 1, 5, W, V)


def test_select_first_steps_and_sorted_rows(fh):
    """The W best lie next to each other, at either end of the row, or one in each part of it."""
    W, V = 8, 20000
    rng = np.random.default_rng(0)
    base = rng.standard_normal((4 * W, V)).astype(np.float32)
    base[0:W] = np.sort(base[0:W])
    base[W:2 * W] = np.sort(base[W:2 * W])[:, ::-1]
    base[2 * W:3 * W, 777:777 + 64] += 50
    base[3 * W:, ::2500] += 50
    check(fh, base, np.zeros(4 * W, np.float32), None, -1, 4, W, V)


# ── states ────────────────────────────────────────────────────────────────
def reorder(fh, W, nReq, outer, inner, rows, row, pads, lens, parent, offset=0, count=1):
    rng = np.random.default_rng(rows + row)
    inner_stride = rows * row + pads[0]
    outer_stride = inner * inner_stride + pads[1]
    beam_stride = outer * outer_stride + pads[2]
    size = offset + nReq * W * beam_stride + 16
    host = [rng.integers(0, 256, size, dtype=np.uint8) for _ in range(count)]
    up = fh.DeviceArray.from_numpy
    dev = [up(h) for h in host]
    st = (fh.BeamState * count)(*[fh.BeamState(d.ptr + offset, beam_stride, outer, outer_stride, inner, inner_stride, row, rows) for d in dev])
    fh.call("beam_reorder", fh.ref(st), count, up(np.array(parent, np.int32)),
            up(np.array(lens, np.int32)) if lens is not None else None, nReq, W)
    for h, d in zip(host, dev):
        want = h.copy()
        for b in range(nReq * W):
            p = b // W * W + parent[b] if 0 <= parent[b] < W else b
            n = rows if lens is None else min(max(lens[p], 0), rows)
            for a in range(outer):
                for i in range(inner):
                    at = offset + a * outer_stride + i * inner_stride
                    want[at + b * beam_stride:at + b * beam_stride + n * row] = h[at + p * beam_stride:at + p * beam_stride + n * row]
        np.testing.assert_array_equal(d.numpy(), want)


@pytest.mark.parametrize("W", [1, 2, 4, 5, 8, 13, 16, 32, 33, 64])
@pytest.mark.parametrize("row,pads,offset", [(64, (0, 0, 0), 0), (64, (16, 32, 48), 16), (8, (0, 8, 0), 8), (4, (0, 0, 4), 4),
                                             (2, (0, 2, 6), 2), (6, (2, 0, 0), 0), (100, (0, 0, 0), 0)])
def test_reorder(fh, W, row, pads, offset):
    rng = np.random.default_rng(W + row)
    for nReq, outer, inner, rows in ((1, 1, 1, 1), (2, 3, 2, 50), (3, 2, 1, 333)):
        parent = rng.integers(-2, W + 2, nReq * W)
        reorder(fh, W, nReq, outer, inner, rows, row, pads, None, parent, offset)
        reorder(fh, W, nReq, outer, inner, rows, row, pads, rng.integers(-2, rows + 3, nReq * W), parent, offset, count=3)


@pytest.mark.parametrize("parents", ["same", "first", "cycle", "swap"])
def test_reorder_patterns(fh, parents):
    W = 8
    p = {"same": np.arange(W), "first": np.zeros(W, int), "cycle": (np.arange(W) + 1) % W, "swap": np.arange(W) ^ 1}[parents]
    reorder(fh, W, 1, 2, 2, 4099, 48, (0, 0, 0), None, p, count=8)
    reorder(fh, W, 1, 2, 2, 0, 48, (0, 0, 64), None, p)
