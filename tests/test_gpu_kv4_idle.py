"""fg_decode_step_kv4 and the sequences that take no part in a step (a token outside
the vocabulary, a full cache, a position past the RoPE table): every array of theirs
stays bit for bit, the accumulated weights among them, and a later eviction keeps
what those weights say."""
import ctypes

import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4_decode import CASES, Model

pytestmark = pytest.mark.gpu

# a workgroup a head; pieces and their join; pieces because two workgroups share a head's weights; units
SHAPES = {
    "short": (CASES["dh32"][0], None, 12),
    "short_gqa": (CASES["dh64_gqa"][0], None, 40),
    "pieces": (CASES["dh64_gqa"][0], None, 3000),
    "twelve_to_one": (dict(dim=384, hidden=64, nLayers=2, nHeads=12, nKvHeads=1, vocab=50, tied=1), None, 60),
    "units": (*CASES["units"], 5000),
}


def arrays(m):
    return [a.numpy() for a in (m.k, m.v, m.kd, m.vd, *m.extra)], [a.numpy() for a in (m.len, m.next)]


@pytest.mark.parametrize("name", list(SHAPES))
def test_idle_full_and_far_sequences_keep_their_weights(fh, name):
    kw, types, maxSeq = SHAPES[name]
    N, warm, maxPos = 5, 6, 20
    m = Model(fh, kw, 4, N, maxSeq, maxPos, types=types, track=True)
    rng = np.random.default_rng(maxSeq)
    V = m.cfg.vocab
    for _ in range(warm):
        assert np.isfinite(m.step(rng.integers(0, V, N))).all()
    # 0 goes on, 1 is idle, 2 full, 3 past the table, 4 outside the vocabulary
    lens, nexts = np.array([warm, warm, maxSeq, warm, warm], np.int32), np.array([warm, warm, warm, maxPos, warm], np.int32)
    m.len.upload(lens)
    m.next.upload(nexts)
    (slots0, heads0) = arrays(m)
    assert np.isfinite(slots0[4]).all() and (slots0[4][:, :, :, :warm] > 0).all()
    for _ in range(2):
        got = m.step([int(rng.integers(V)), -1, 3, 4, V])
        assert np.isfinite(got[0]).all() and np.isnan(got[1:]).all()
    slots1, heads1 = arrays(m)
    for a, b in zip(slots0, slots1):
        np.testing.assert_array_equal(a[:, 1:], b[:, 1:])
    for a, b in zip(heads0, heads1):
        np.testing.assert_array_equal(a[1:], b[1:])
        assert b[0] == a[0] + 2
    w0, w1 = slots0[4][:, 0, :, :warm + 2], slots1[4][:, 0, :, :warm + 2]
    assert np.isfinite(w1).all() and (w1 >= w0).all() and (w1 > 0).all()
    budget, recent = 4, 1
    fh.call("kv4_evict", fh.ref(m.cache), budget, recent)
    want = [a.copy() for a in slots1]
    for l, s, h in np.ndindex(slots1[4].shape[:3]):
        holes, movers = ref.evict(slots1[4][l, s, h], slots1[5][l, s, h], heads1[0][s], heads1[1][s], budget, recent)
        for a, b in zip(want, slots1):
            a[l, s, h, holes] = b[l, s, h, movers]
    slots2, heads2 = arrays(m)
    for a, b in zip(slots2, want):
        np.testing.assert_array_equal(a, b)
    np.testing.assert_array_equal(heads2[0], np.minimum(heads1[0], budget))


@pytest.mark.parametrize("N", [1, 3])
@pytest.mark.parametrize("name", ["short", "pieces"])
def test_all_sequences_idle(fh, name, N):
    """A step in which none takes part changes nothing."""
    kw, types, maxSeq = SHAPES[name]
    m = Model(fh, kw, 4, N, maxSeq, 20, types=types, track=True)
    for t in range(4):
        m.step([1, 2, 3 + t][:N])
    before = arrays(m)
    assert np.isnan(m.step([-1, m.cfg.vocab, -5][:N])).all()
    for a, b in zip(arrays(m), before):
        for x, y in zip(a, b):
            np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("name", ["short", "pieces"])
def test_a_recorded_step_with_idle_sequences(fh, name):
    """A graph of one step, replayed with other sequences idle each time and eager work between, does what the eager steps do."""
    kw, types, maxSeq = SHAPES[name]
    N, results = 4, []
    for graph in (False, True):
        rng = np.random.default_rng(11)
        m = Model(fh, kw, 4, N, maxSeq, 20, types=types, track=True)
        m.step(rng.integers(0, m.cfg.vocab, N))
        handle, got = ctypes.c_void_p(), []
        if graph:
            fh.check(fh.lib.fg_graph_begin(), "begin")
            fh.check(fh.lib.fg_decode_step_kv4(ctypes.byref(m.dec.m), ctypes.byref(m.cache), m.tokens.ptr, m.logits.ptr), "step")
            fh.check(fh.lib.fg_graph_end(ctypes.byref(handle)), "end")
        for _ in range(6):
            tokens = rng.integers(0, m.cfg.vocab, N).astype(np.int32)
            tokens[rng.random(N) < 0.5] = -1
            if graph:
                m.tokens.upload(tokens)
                fh.check(fh.lib.fg_graph_launch(handle), "launch")
                junk = [fh.DeviceArray.from_numpy(np.ones(50000, np.float32)) for _ in range(3)]
                fh.sync()
                del junk
                got.append(m.logits.numpy())
            else:
                got.append(m.step(tokens))
            np.testing.assert_array_equal(np.isnan(got[-1]).all(1), tokens < 0)
        slots, heads = arrays(m)
        assert np.isfinite(slots[4]).all()
        results.append(got + slots + heads)
        if graph:
            fh.check(fh.lib.fg_graph_destroy(handle), "destroy")
    for x, y in zip(*results):
        np.testing.assert_array_equal(x, y)
