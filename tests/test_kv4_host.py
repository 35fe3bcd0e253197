"""The 4-bit cache and beam search without a GPU: the plain forms against known
answers, the structures against the header, and every refusal (arguments are
checked before the device is)."""
import ctypes
import re

import numpy as np
import pytest

import forge_hip as fh
import kv4_ref as ref

A = 1 << 20  # an aligned address that is never read: the calls below are refused


def cache(**kw):
    f = dict(nLayers=2, nSeq=4, nKvHeads=2, dHead=64, maxSeq=40, k=A, v=A, kd=A, vd=A, len=A, next=A, weight=A, pos=A)
    f.update(kw)
    return fh.Kv4Cache(*[f[n] for n, _ in fh.Kv4Cache._fields_])


def state(**kw):
    f = dict(base=A, beam_stride=64, outer=1, outer_stride=0, inner=1, inner_stride=0, row_bytes=4, rows=3)
    f.update(kw)
    return fh.BeamState(*[f[n] for n, _ in fh.BeamState._fields_])


def refused(name, *args, says):
    rc = getattr(fh.lib, "fg_" + name)(*args)
    assert rc == -1, (name, args, rc)
    assert "fg_" + name in fh.last_error() and re.search(says, fh.last_error()), fh.last_error()


def test_structures_match_the_header():
    text = re.sub(r"/\*.*?\*/", "", open(fh.HEADER).read(), flags=re.S)
    for cls, name in ((fh.Kv4Cache, "fg_kv4_cache"), (fh.BeamState, "fg_beam_state")):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
        fields = [n.strip(" *") for d in body.split(";") if d.strip() for n in re.sub(r"^\s*\w+", "", d).split(",")]
        assert fields == [n for n, _ in cls._fields_]


CACHE_CALLS = {
    "kv4_append": lambda c: (c, 0, A, A, 128, 1, None),
    "kv4_read": lambda c: (c, 0, A, A, 128, 0, 1),
    "kv4_attn": lambda c: (c, 0, A, A, 4, 1.0, 0, None),
    "kv4_commit": lambda c: (c, 1, None),
    "kv4_evict": lambda c: (c, 8, 2),
    "kv4_reorder": lambda c: (c, A, 2),
}


@pytest.mark.parametrize("name", sorted(CACHE_CALLS))
def test_bad_caches_are_refused(name):
    args = CACHE_CALLS[name]
    refused(name, *args(None), says="null")
    for bad in (dict(nLayers=0), dict(nSeq=0), dict(nKvHeads=-1), dict(maxSeq=0)):
        refused(name, *args(fh.ref(cache(**bad))), says="bad dimensions")
    for d in (0, 16, 48, 160, 512):
        refused(name, *args(fh.ref(cache(dHead=d))), says="head size")
    for p in ("k", "v", "kd", "vd", "len", "next"):
        refused(name, *args(fh.ref(cache(**{p: None}))), says="null")
    for p in ("k", "v", "kd", "vd", "weight", "pos"):
        refused(name, *args(fh.ref(cache(**{p: A + 8}))), says="aligned")
    refused(name, *args(fh.ref(cache(nLayers=1 << 20, nSeq=1 << 10))), says="too many")
    refused(name, *args(fh.ref(cache(maxSeq=(1 << 30) + 1))), says="slots")


def test_bad_arguments_are_refused():
    c = cache()
    at = fh.ref(c)
    for name in ("kv4_append", "kv4_read", "kv4_attn"):
        for layer in (-1, 2):
            args = list(CACHE_CALLS[name](at))
            args[1] = layer
            refused(name, *args, says="layer")
    refused("kv4_append", at, 0, A, A, 127, 1, None, says="stride")
    refused("kv4_append", at, 0, A, None, 128, 1, None, says="null")
    refused("kv4_append", at, 0, A, A, 128, -1, None, says="negative")
    refused("kv4_read", at, 0, A, A, 127, 0, 1, says="stride")
    refused("kv4_read", at, 0, None, A, 128, 0, 1, says="null")
    for first, T in ((-1, 1), (0, 41), (40, 1), (2147483647, 2147483647), (0, -1)):
        refused("kv4_read", at, 0, A, A, 128, first, T, says="slots")
    refused("kv4_attn", at, 0, None, A, 4, 1.0, 0, None, says="null")
    refused("kv4_attn", at, 0, A, A, 3, 1.0, 0, None, says="query heads")
    refused("kv4_attn", at, 0, A, A, 0, 1.0, 0, None, says="query heads")
    refused("kv4_attn", at, 0, A, A, 4, 1.0, -1, None, says="negative")
    refused("kv4_commit", at, -1, None, says="negative")
    refused("kv4_evict", at, 0, 0, says="budget")
    refused("kv4_evict", at, 8, 9, says="recent")
    refused("kv4_evict", at, 8, -1, says="recent")
    refused("kv4_evict", fh.ref(cache(weight=None)), 8, 2, says="weights")
    refused("kv4_evict", fh.ref(cache(pos=None)), 8, 2, says="weights")
    refused("kv4_reorder", at, None, 2, says="null")
    for w in (0, 3, 65):
        refused("kv4_reorder", at, A, w, says="beams")


def test_bad_eviction_and_beams_are_refused():
    ok = [A] * 7 + [2, 4, 2, 40, 8, 2]
    for i in range(7):
        refused("kv_evict_select", *(ok[:i] + [None] + ok[i + 1:]), says="null")
    for i in (7, 8, 9, 10):
        refused("kv_evict_select", *(ok[:i] + [0] + ok[i + 1:]), says="dimensions|budget")
    refused("kv_evict_select", *(ok[:10] + [(1 << 30) + 1] + ok[11:]), says="dimensions")
    for budget, recent in ((0, 0), (40, 1), (8, 9), (8, -1)):
        refused("kv_evict_select", *(ok[:11] + [budget, recent]), says="budget|recent")
    ok = [A, A, A, A, A, 100, A, A, 2, 2, 4, 100]
    for i in (0, 1, 2, 4, 6):
        refused("beam_select", *(ok[:i] + [None] + ok[i + 1:]), says="null")
    for i, bad in ((9, 0), (10, 0), (10, 65), (11, 0), (9, 32768)):
        refused("beam_select", *(ok[:i] + [bad] + ok[i + 1:]), says="dimensions")
    refused("beam_select", *(ok[:5] + [99] + ok[6:]), says="stride")
    refused("beam_select", *(ok[:5] + [1 << 27] + ok[6:11] + [(1 << 26) + 1]), says="vocabulary")
    refused("beam_select", *(ok[:3] + [None] + ok[4:]), says="together")
    refused("beam_select", *(ok[:7] + [None] + ok[8:]), says="together")
    refused("beam_select", *(ok[:8] + [100] + ok[9:]), says="eos")
    refused("beam_select", *(ok[:8] + [-1] + ok[9:]), says="eos")
    s = state()
    refused("beam_reorder", None, 1, A, None, 1, 4, says="null")
    refused("beam_reorder", fh.ref(s), 1, None, None, 1, 4, says="null")
    for n in (0, 9):
        refused("beam_reorder", fh.ref(s), n, A, None, 1, 4, says="states")
    for req, w in ((0, 4), (1, 0), (1, 65), (65536, 2)):
        refused("beam_reorder", fh.ref(s), 1, A, None, req, w, says="dimensions")
    refused("beam_reorder", fh.ref(state(base=None)), 1, A, None, 1, 4, says="null")
    for bad in (dict(outer=0), dict(inner=0), dict(rows=-1), dict(row_bytes=0), dict(outer=65536)):
        refused("beam_reorder", fh.ref(state(**bad)), 1, A, None, 1, 4, says="parts")
    for bad in (dict(base=A + 1), dict(beam_stride=63), dict(outer_stride=1), dict(inner_stride=3), dict(row_bytes=5)):
        refused("beam_reorder", fh.ref(state(**bad)), 1, A, None, 1, 4, says="even")
    for bad in (dict(beam_stride=-64), dict(outer_stride=-2), dict(inner_stride=-2)):
        refused("beam_reorder", fh.ref(state(**bad)), 1, A, None, 1, 4, says="negative")


def test_good_arguments_need_a_device():
    if fh.device_count() > 0:
        pytest.skip("a GPU is visible")
    c = cache()
    for name, args in CACHE_CALLS.items():
        assert getattr(fh.lib, "fg_" + name)(*args(fh.ref(c))) == -4, name


def test_quantizer_known_answers():
    x = np.zeros((2, 32), np.float32)
    x[0, :] = np.arange(32) - 8.0  # greatest magnitude 23 at the end: d = -23/8
    x[1, :4] = (4.0, -4.0, 1.25, -0.25)  # of equals the first: d = -0.5
    c, d = ref.quantize(x)
    assert d[0, 0] == np.float16(-2.875) and d[1, 0] == np.float16(-0.5)
    assert c[0, 0, 31] == 0 and c[0, 0, 8] == 8
    np.testing.assert_array_equal(c[1, 0, :5], [0, 15, 6, 9, 8])  # -2.5 + 8.5 = 6, 0.5 + 8.5 = 9
    v = ref.values(ref.pack(c), d)
    np.testing.assert_array_equal(v[1, :5], [4.0, -3.5, 1.0, -0.5, 0.0])


def test_quantizer_is_the_nearest_step_inside_its_range():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((200, 96)).astype(np.float32) * np.exp(rng.uniform(-9, 9, (200, 1))).astype(np.float32)
    c, d = ref.quantize(x)
    v = ref.values(ref.pack(c), d)
    step = np.abs(np.repeat(d.astype(np.float64), 32, -1))
    off = np.abs(v - x)
    inside = c.reshape(200, 96)
    assert (off[(inside > 0) & (inside < 15)] <= 0.5 * step[(inside > 0) & (inside < 15)]).all()
    # the far end is half a step's rounding of d off, the other end is cut at 7 of 8 steps
    assert (off <= step * (1 + 8 * 2.0 ** -11)).all()


def test_quantizer_edges():
    x = np.zeros((5, 32), np.float32)
    x[1, 3] = np.nan
    x[2, 3] = np.inf
    x[3, 3] = 8 * 65520.0  # the step rounds past fp16
    x[4, 3] = 1e-9         # the step rounds to zero
    c, d = ref.quantize(x)
    assert d[0, 0] == 0 and (c[0] == 8).all() and np.isnan(d[1:4, 0]).all() and d[4, 0] == 0
    assert np.isnan(ref.values(ref.pack(c), d)[1:4]).all()


def test_eviction_known_answers():
    w = np.array([5, 1, 1, 0, 7, np.nan], np.float32)
    pos = np.arange(6)
    assert ref.evict(w, pos, 6, 6, 3, 1) == ([1, 2], [4, 5])  # the newest stays whatever its weight
    assert ref.evict(w, pos, 6, 6, 3, 0) == ([2], [4])        # of equals the lowest slot
    assert ref.evict(w, pos, 3, 6, 3, 1) == ([], [])


def test_beam_select_known_answers():
    x = np.log(np.array([[0.5, 0.25, 0.25], [0.125, 0.125, 0.75]])).astype(np.float32)
    s, t, p, f = ref.beam_select(x, np.array([0.0, 0.0], np.float32), np.array([0, 0]), 2, 1, 2)
    np.testing.assert_array_equal(t, [2, 0])
    np.testing.assert_array_equal(p, [1, 0])
    np.testing.assert_array_equal(f, [1, 0])
    np.testing.assert_allclose(s, np.log([0.75, 0.5]), rtol=1e-7)
    s, t, p, f = ref.beam_select(x, np.array([0.0, -0.1], np.float32), np.array([0, 1]), 2, 1, 2)
    np.testing.assert_array_equal((t, p, f), ([2, 0], [1, 0], [1, 0]))
    assert s[0] == np.float32(-0.1)


def test_handles_of_one_kind_are_not_read_as_another():
    """The addon's cache handle as a decode model, and things that are no handle at all."""
    import os
    import subprocess
    code = """
import { addonUninitialised } from './src/L2/device.js';
const a = addonUninitialised(), no = [null, null, null, null, null, null, null, null];
const cache = a.kv4Cache(1, 1, 1, 32, 8, ...no), say = (fn) => { try { fn(); return 'nothing'; } catch (e) { return e.message; } };
for (const x of [cache, {}, null, 7]) {
  console.log(say(() => a.decodeStep(x, null, null, null, null)));
  console.log(say(() => a.decodeStepKv4(x, cache, null, null)));
}
for (const x of [{}, null, 7]) console.log(say(() => a.kv4Commit(x, 1, null)));
"""
    r = subprocess.run(["node", "--input-type=module", "-e", code], cwd=os.path.dirname(os.path.abspath(fh.__file__)),
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert r.returncode == 0, r.stdout
    assert r.stdout.split("\n")[:-1] == ["expected a decode model handle"] * 8 + ["expected a 4-bit cache handle"] * 3, r.stdout
