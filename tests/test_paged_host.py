"""The paged cache and the verification of drafts without a GPU: the plain forms
against known answers, the structure against the header, and every refusal
(arguments are checked before the device is)."""
import math
import re

import numpy as np
import pytest

import forge_hip as fh
import paged_ref as ref

A = 1 << 20  # an aligned address that is never read: the calls below are refused


def cache(**kw):
    f = dict(nLayers=2, nSeq=4, nKvHeads=2, dHead=64, pageSize=16, nPages=9, maxPages=3, type=1, k=A, v=A, table=A, len=A)
    f.update(kw)
    return fh.PagedCache(*[f[n] for n, _ in fh.PagedCache._fields_])


def refused(name, *args, says):
    rc = getattr(fh.lib, "fg_" + name)(*args)
    assert rc == -1, (name, args, rc)
    assert "fg_" + name in fh.last_error() and re.search(says, fh.last_error()), fh.last_error()


def test_structure_matches_the_header():
    text = re.sub(r"/\*.*?\*/", "", open(fh.HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct fg_paged_cache \{(.*?)\}", text, flags=re.S).group(1)
    body = body.replace("const ", "")
    fields = [n.strip(" *") for d in body.split(";") if d.strip() for n in re.sub(r"^\s*\w+", "", d).split(",")]
    assert fields == [n for n, _ in fh.PagedCache._fields_]


CALLS = {
    "paged_append": lambda c: (c, 0, A, A, A, A, 512, 4, 1, None, A, A, 9, 64, 0),
    "paged_read": lambda c: (c, 0, A, A, 128, 0, 1),
    "paged_attn": lambda c: (c, 0, A, 2 * A, 4, 1.0, 1, None, 0, 0),
    "paged_commit": lambda c: (c, 1, None),
}


def but(args, **changes):
    args = list(args)
    for i, v in changes.items():
        args[int(i[1:])] = v
    return args


@pytest.mark.parametrize("name", sorted(CALLS))
def test_bad_caches_are_refused(name):
    args = CALLS[name]
    refused(name, *args(None), says="null")
    for bad in (dict(nLayers=0), dict(nSeq=0), dict(nKvHeads=-1), dict(nPages=0), dict(maxPages=0)):
        refused(name, *args(fh.ref(cache(**bad))), says="bad dimensions")
    for d in (0, 16, 48, 160, 512):
        refused(name, *args(fh.ref(cache(dHead=d))), says="head size")
    for p in (0, -16, 2, 24, 2048):
        refused(name, *args(fh.ref(cache(pageSize=p))), says="page size")
    refused(name, *args(fh.ref(cache(maxPages=(1 << 26) + 1))), says="above 2")
    refused(name, *args(fh.ref(cache(nKvHeads=1 << 20))), says="too many")
    for t in (-1, 2, 8):
        refused(name, *args(fh.ref(cache(type=t))), says="type")
    for p in ("k", "v", "table", "len"):
        refused(name, *args(fh.ref(cache(**{p: None}))), says="null")
    for p in ("k", "v"):
        refused(name, *args(fh.ref(cache(**{p: A + 8}))), says="aligned")


def test_bad_steps_are_refused():
    c = fh.ref(cache())
    for name in ("paged_append", "paged_attn", "paged_read"):
        ok = CALLS[name](c)
        for layer in (-1, 2):
            refused(name, *but(ok, _1=layer), says="layer")
    at = {"paged_append": "_8", "paged_attn": "_6", "paged_commit": "_1", "paged_read": "_6"}
    for name, i in at.items():
        refused(name, *but(CALLS[name](c), **{i: -1}), says="negative")
    big = fh.ref(cache(maxPages=1 << 26))
    for name in ("paged_append", "paged_attn", "paged_read"):
        refused(name, *but(CALLS[name](big), **{at[name]: 1 << 24}), says="too many")
    ok = CALLS["paged_append"](c)
    for i in ("_4", "_5"):
        refused("paged_append", *but(ok, **{i: None}), says="null")
    for i in ("_2", "_3"):
        refused("paged_append", *but(ok, **{i: None}), says="together")
    for h in (0, -1, 1 << 21):
        refused("paged_append", *but(ok, _7=h), says="query heads")
    refused("paged_append", *but(ok, _6=255), says="stride")
    refused("paged_append", *but(ok, _2=None, _3=None, _6=127), says="stride")
    refused("paged_append", *ok, says="in place")
    refused("paged_append", *but(ok, _6=128, _7=1), says="in place")  # rows of two kv heads, one query head
    ok = but(ok, _2=2 * A)
    for rot in (-2, 3, 66):
        refused("paged_append", *but(ok, _13=rot), says="rotated")
    for i, v in (("_10", None), ("_11", None), ("_12", 0)):
        refused("paged_append", *but(ok, **{i: v}), says="angles")
    ok = CALLS["paged_read"](c)
    for i in ("_2", "_3"):
        refused("paged_read", *but(ok, **{i: None}), says="null")
    refused("paged_read", *but(ok, _4=127), says="stride")
    for first, T in ((-1, 2), (48, 1), (0, 49)):
        refused("paged_read", *but(ok, _5=first, _6=T), says="slots")
    ok = CALLS["paged_attn"](c)
    for i in ("_2", "_3"):
        refused("paged_attn", *but(ok, **{i: None}), says="null")
    refused("paged_attn", *but(ok, _3=A), says="in place")
    for h in (0, 3, -2):
        refused("paged_attn", *but(ok, _4=h), says="heads")
    for i in ("_8", "_9"):
        refused("paged_attn", *but(ok, **{i: -1}), says="window")


def test_bad_verifications_are_refused():
    ok = [A, A, A, 100, A, 100, A, None, A, 1.0, 4, 3, 100]
    for i in (0, 1, 2, 6, 8):
        refused("draft_verify", *(ok[:i] + [None] + ok[i + 1:]), says="null")
    for i, bad in ((10, 0), (10, -1), (11, -1), (11, 1024), (12, 0), (12, (1 << 26) + 1), (10, 1 << 19)):
        refused("draft_verify", *(ok[:i] + [bad] + ok[i + 1:]), says="dimensions")
    for t in (-1.0, 1e-31, math.inf, math.nan):
        refused("draft_verify", *(ok[:9] + [t] + ok[10:]), says="temperature")
    for i in (3, 5):
        refused("draft_verify", *(ok[:i] + [99] + ok[i + 1:]), says="stride")


def test_good_arguments_need_a_device():
    if fh.device_count() > 0:
        pytest.skip("a GPU is visible")
    c = cache()
    for name, args in CALLS.items():
        ok = args(fh.ref(c))
        assert getattr(fh.lib, "fg_" + name)(*(but(ok, _2=2 * A) if name == "paged_append" else ok)) == -4, name
    assert fh.lib.fg_draft_verify(A, A, A, 100, None, 0, A, None, A, 0.5, 4, 3, 100) == -4
    assert fh.lib.fg_draft_verify(A, A, A, 100, None, 0, None, None, None, 0.0, 4, 0, 100) == -4


def test_handles_of_one_kind_are_not_read_as_another():
    """The addon's paged cache handle as a decode model or a 4-bit cache, and things that are no handle at all."""
    import os
    import subprocess
    code = """
import { addonUninitialised } from './src/L2/device.js';
const a = addonUninitialised(), no = [null, null, null, null, null, null, null, null];
const paged = a.pagedCache(1, 1, 1, 32, 16, 4, 4, 0, null, null, null, null), kv4 = a.kv4Cache(1, 1, 1, 32, 8, ...no);
const say = (fn) => { try { fn(); return 'nothing'; } catch (e) { return e.message; } };
for (const x of [paged, kv4, {}, null, 7]) console.log(say(() => a.decodeStepPaged(x, paged, null, 1, null, 0, 0, 1, null)));
for (const x of [kv4, {}, null, 7]) console.log(say(() => a.pagedCommit(x, 1, null)));
console.log(say(() => a.kv4Commit(paged, 1, null)));
"""
    r = subprocess.run(["node", "--input-type=module", "-e", code], cwd=os.path.dirname(os.path.abspath(fh.__file__)),
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert r.returncode == 0, r.stdout
    assert r.stdout.split("\n")[:-1] == ["expected a decode model handle"] * 5 + ["expected a paged cache handle"] * 4 + ["expected a 4-bit cache handle"], r.stdout


# ── the plain forms ───────────────────────────────────────────────────────
def test_rotation_by_hand():
    cos, sin = np.array([[1.0, 1.0], [0.0, 0.6]]), np.array([[0.0, 0.0], [1.0, 0.8]])
    x = np.array([[1.0, 2.0, 3.0, 4.0, 5.0]])
    assert ref.rotate(x, 0, cos, sin, 4, 0).tolist() == x.tolist()
    assert np.allclose(ref.rotate(x, 1, cos, sin, 4, 0), [[-2, 1, 1.8 - 3.2, 2.4 + 2.4, 5]])
    assert np.allclose(ref.rotate(x, 1, cos, sin, 4, 1), [[-3, 1.2 - 3.2, 1, 1.6 + 2.4, 5]])
    assert np.isnan(ref.rotate(x, 2, cos, sin, 4, 0)[0, :4]).all()


def test_window_by_hand():
    assert ref.sees(5, 8, 0, 0).tolist() == [True] * 6 + [False] * 2
    assert ref.sees(5, 8, 2, 1).tolist() == [True, False, False, False, True, True, False, False]
    assert ref.sees(1, 3, 1, 9).tolist() == [True, True, False]


def test_verification_by_hand():
    p = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.1, 0.8]]))
    q = np.log(np.array([[0.2, 0.6, 0.2]]))
    one = lambda d, u: [x.tolist() if hasattr(x, "tolist") else x for x in ref.verify(p, q, np.array([d]), np.array(u), 1.0, 1)]  # noqa: E731
    assert one(0, [0.99, 0.15]) == [[0, 1], 2]           # p > q: stands; then the second row from 0.1 on is token 1
    assert one(1, [0.41, 0.8]) == [[1, 2], 2]            # 0.41 0.6 < 0.25: stands
    assert one(1, [0.43, 0.8]) == [[0, -1], 1]           # does not; 0.3, 0, 0.05 are left, 0.28 of them is in token 0
    assert one(1, [0.43, 0.9]) == [[2, -1], 1]
    assert ref.verify(p, None, np.array([1]), np.array([0.2, 0.5]), 1.0, 1)[0].tolist() == [1, 2]


def test_greatest_by_hand():
    x = np.array([[1.0, 3.0, 3.0], [np.nan, -1.0, -2.0], [np.nan] * 3])
    assert [ref.best(r) for r in x] == [1, 1, -1]
    assert ref.verify(x, None, np.array([1, 1]), None, 0.0, 2)[0].tolist() == [1, 1, -1]
    assert ref.verify(x, None, np.array([2, 1]), None, 0.0, 2)[0].tolist() == [1, -1, -1]
    assert ref.verify(x, None, np.array([2, 1]), None, 0.0, -1)[1] == 0


def test_draw_by_hand():
    w = np.array([0.0, 0.25, 0.0, 0.75, 0.0])
    assert [ref.draw(w, u) for u in (0.0, 0.2, 0.25, 0.999, 1.0)] == [1, 1, 3, 3, 3]
    assert ref.draw(w * 0, 0.5) == -1 and ref.draw(w * np.nan, 0.5) == -1
