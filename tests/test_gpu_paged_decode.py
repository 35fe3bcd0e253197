"""fg_decode_step_paged: the inference forward of several tokens of every sequence over a
paged cache, a run of the paged cache's and the drafts' operators together, eager and
recorded, and the JavaScript API over them (tests/js/paged.mjs)."""
import ctypes
import json
import os
import subprocess

import numpy as np
import pytest

import oracle
import paged_ref as ref
from test_gpu_decode import Decoder
from test_gpu_kv4_decode import CASES
from test_gpu_paged import angles, out_bound
from util import TOL_FWD, rel_l2

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Model:
    """A decoder with vectors for nSeq T rows and its paged cache, every page of a sequence in place."""

    def __init__(self, fh, kw, seed, nSeq, T, P, maxPages, maxPos, types=None, kind=0):
        self.fh, self.cfg = fh, oracle.Cfg(**kw)
        cfg = self.cfg
        params = oracle.init_weights(cfg, seed)
        oracle.split_params(cfg, params)["tok_emb"][:] = np.random.default_rng(seed).standard_normal(cfg.vocab * cfg.dim).astype(np.float32) * 0.3
        self.dec = Decoder(fh, cfg, params, maxPos, types=types)
        self.one = [self.dec.m.x, self.dec.m.q, self.dec.m.h, self.dec.m.attn_part]
        A = fh.DeviceArray
        self.vec = [A((nSeq * T, n)) for n in (cfg.dim, cfg.dim, cfg.hidden)]
        self.nSeq, self.T, self.P, self.maxPages = nSeq, T, P, maxPages
        self.nPages = nSeq * maxPages
        self.table_host = np.random.default_rng(seed).permutation(self.nPages).reshape(nSeq, maxPages).astype(np.int32)
        shape = (cfg.nLayers, self.nPages, cfg.nKvHeads, P, cfg.dHead)
        fill = np.full(shape, np.nan, np.float16 if kind else np.float32)
        self.k, self.v = A.from_numpy(fill), A.from_numpy(fill)
        self.table, self.len = A.from_numpy(self.table_host), A.zeros((nSeq,), np.int32)
        self.cache = fh.PagedCache(cfg.nLayers, nSeq, cfg.nKvHeads, cfg.dHead, P, self.nPages, maxPages, kind, self.k.ptr, self.v.ptr,
                                   self.table.ptr, self.len.ptr)
        self.tokens, self.count, self.logits = A((nSeq, T), np.int32), A((nSeq,), np.int32), A((nSeq, T, cfg.vocab))

    def step(self, tokens, counts=None, window=0, sinks=0, commit=1):
        m = self.dec.m
        m.x, m.q, m.h, m.attn_part = self.vec[0].ptr, self.vec[1].ptr, self.vec[2].ptr, None
        self.tokens.upload(np.array(tokens, np.int32))
        if counts is not None:
            self.count.upload(np.array(counts, np.int32))
        self.fh.check(self.fh.lib.fg_decode_step_paged(ctypes.byref(m), ctypes.byref(self.cache), self.tokens.ptr, self.T,
                                                       self.count.ptr if counts is not None else None, window, sinks, commit, self.logits.ptr),
                      "fg_decode_step_paged")
        return self.logits.numpy()

    def alone(self, ids):
        """Logits of one sequence by fg_decode_step over the contiguous cache."""
        m = self.dec.m
        m.x, m.q, m.h, m.attn_part = self.one
        return np.stack([self.dec.step(int(t), i).copy() for i, t in enumerate(ids)])


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("name", list(CASES))
def test_chunks_against_single_steps(fh, name, kind):
    """Chunks of every size, ragged, uncommitted ones between them: each token's logits are those of the contiguous cache's
    single steps (an fp16 cache: within its rounding, 2^-11 of keys and values, of which a score sums dH and a layer follows)."""
    kw, types = CASES[name]
    nSeq, T, n = 3, 6, 21
    m = Model(fh, kw, 5, nSeq, T, 4, 8, 32, types, kind)
    rng = np.random.default_rng(17)
    ids = rng.integers(0, m.cfg.vocab, (nSeq, n))
    want = [m.alone(x) for x in ids]
    tol = TOL_FWD if kind == 0 else 2.0 ** -8
    at = np.zeros(nSeq, int)
    while (at < n).any():
        counts = [int(min(rng.integers(0, T + 1), n - a)) for a in at]
        tokens = np.full((nSeq, T), -1)
        tokens[:] = rng.integers(0, m.cfg.vocab, (nSeq, T))  # drafts that do not stand
        assert np.isfinite(m.step(tokens, [min(T, 32 - a) for a in at], commit=0)[0]).all()
        assert (m.len.numpy() == at).all()
        for s in range(nSeq):
            tokens[s, :counts[s]] = ids[s, at[s]:at[s] + counts[s]]
        got = m.step(tokens, counts)
        for s in range(nSeq):
            assert np.isnan(got[s, counts[s]:]).all()
            for t in range(counts[s]):
                assert rel_l2(got[s, t], want[s][at[s] + t]) <= tol, (s, t)
        at += counts
        assert (m.len.numpy() == at).all()


def test_tokens_that_take_no_part(fh):
    """A token outside the vocabulary, a position outside the table, a missing page or the end of the room ends its
    sequence's tokens there; what came before stands, other sequences do not notice."""
    kw, types = CASES["dh64_gqa"]
    m = Model(fh, kw, 5, 5, 4, 4, 3, 11, types)
    rng = np.random.default_rng(2)
    ids = rng.integers(0, m.cfg.vocab, (5, 12))
    want = [m.alone(x[:11]) for x in ids]
    m.table_host[3, 1] = -1
    m.table.upload(m.table_host)
    tokens = ids[:, :4].copy()
    tokens[1, 2], tokens[2, 0] = m.cfg.vocab, -1
    got = m.step(tokens)
    stood = [4, 2, 0, 4, 4]
    for s, k in enumerate(stood):
        assert np.isnan(got[s, k:]).all() and all(rel_l2(got[s, t], want[s][t]) <= TOL_FWD for t in range(k))
    assert m.len.numpy().tolist() == stood
    got = m.step(ids[:, 4:8], [4, 0, -3, 4, 9])
    assert m.len.numpy().tolist() == [8, 2, 0, 4, 8] and np.isnan(got[3]).all() and np.isnan(got[1:3]).all()
    got = m.step(ids[:, 8:12])  # positions end at 11, the room at 12
    assert m.len.numpy().tolist() == [11, 6, 4, 4, 11] and np.isnan(got[0, 3]).all()
    assert all(rel_l2(got[0, t], want[0][8 + t]) <= TOL_FWD for t in range(3))


def test_window_in_the_model(fh):
    """One chunk and token by token see the same windows."""
    kw, types = CASES["dh32"]
    a, b = Model(fh, kw, 9, 1, 24, 4, 6, 24, types), Model(fh, kw, 9, 1, 1, 4, 6, 24, types)
    ids = np.random.default_rng(3).integers(0, a.cfg.vocab, 24)
    all_ = a.step([ids], window=5, sinks=2)[0]
    full = a.alone(ids)
    for t in range(24):
        assert rel_l2(b.step([[ids[t]]], window=5, sinks=2)[0, 0], all_[t]) <= TOL_FWD
    assert rel_l2(all_[4], full[4]) <= TOL_FWD and rel_l2(all_[20], full[20]) > 1e-3


def test_refusals(fh):
    kw, types = CASES["dh64_gqa"]
    m = Model(fh, kw, 5, 2, 2, 4, 3, 16, types)
    call = fh.lib.fg_decode_step_paged
    ok = [ctypes.byref(m.dec.m), ctypes.byref(m.cache), m.tokens.ptr, 2, None, 0, 0, 1, m.logits.ptr]
    for i in (0, 1, 2, 8):
        assert call(*(ok[:i] + [None] + ok[i + 1:])) == -1 and "null" in fh.last_error()
    for i, bad in ((3, 0), (3, -1), (3, 32768), (5, -1), (6, -1)):
        assert call(*(ok[:i] + [bad] + ok[i + 1:])) == -1
    for field, bad in (("nLayers", 1), ("nKvHeads", 4), ("dHead", 128), ("type", 3), ("pageSize", 6), ("len", None)):
        was = getattr(m.cache, field)
        setattr(m.cache, field, bad)
        assert call(*ok) == -1, field
        setattr(m.cache, field, was)


class Drafting:
    """Append, attend, verify and commit of a few drafted tokens of every sequence, as a step of a serving loop makes them:
    fp16 pages, a layer's keys, values and queries given from outside."""

    def __init__(self, fh, rng, nSeq=3, D=3, nH=6, nKV=2, dH=64, P=8, maxPages=30, V=500):
        self.fh, self.nSeq, self.D, self.nH, self.nKV, self.dH, self.P, self.V = fh, nSeq, D, nH, nKV, dH, P, V
        up, T = fh.DeviceArray.from_numpy, D + 1
        self.table_host = rng.permutation(nSeq * maxPages).reshape(nSeq, maxPages).astype(np.int32)
        self.table, self.len = up(self.table_host), up(np.zeros(nSeq, np.int32))
        self.k, self.v = (fh.DeviceArray.zeros((1, nSeq * maxPages, nKV, P, dH), np.float16) for _ in range(2))
        self.cache = fh.PagedCache(1, nSeq, nKV, dH, P, nSeq * maxPages, maxPages, 1, self.k.ptr, self.v.ptr, self.table.ptr, self.len.ptr)
        self.cos_h, self.sin_h = angles(fh, P * maxPages, dH)
        self.cos, self.sin = up(self.cos_h), up(self.sin_h)
        self.qkv = fh.DeviceArray((nSeq, T, nH + 2 * nKV, dH))
        self.q, self.out = fh.DeviceArray.zeros((nSeq, T, nH, dH)), fh.DeviceArray.zeros((nSeq, T, nH, dH))
        self.logits, self.drafted_from = fh.DeviceArray((nSeq, T, V)), fh.DeviceArray((nSeq, D, V))
        self.draft, self.u = fh.DeviceArray((nSeq, D), np.int32), fh.DeviceArray((nSeq, T))
        self.token, self.count = fh.DeviceArray((nSeq, T), np.int32), fh.DeviceArray((nSeq,), np.int32)
        self.K, self.Vv = [[] for _ in range(nSeq)], [[] for _ in range(nSeq)]

    def upload(self, rng):
        n, D, T = self.nSeq, self.D, self.D + 1
        self.h = {"qkv": rng.standard_normal(self.qkv.shape).astype(np.float32), "logits": rng.standard_normal((n, T, self.V)).astype(np.float32) * 2}
        self.h["from"] = (self.h["logits"][:, :D] + rng.standard_normal((n, D, self.V)) * 0.3).astype(np.float32)
        self.h["draft"] = np.array([[ref.draw(ref.softmax(self.h["from"][s, t], 1.0), rng.random()) for t in range(D)] for s in range(n)], np.int32)
        self.h["u"] = rng.random((n, T)).astype(np.float32)
        for d, k in ((self.qkv, "qkv"), (self.logits, "logits"), (self.drafted_from, "from"), (self.draft, "draft"), (self.u, "u")):
            d.upload(self.h[k])

    def queue(self):
        fh, c, T, row = self.fh, self.fh.ref(self.cache), self.D + 1, 4 * self.dH
        at = self.qkv.ptr
        fh.call("paged_append", c, 0, self.q, at, at + self.nH * row, at + (self.nH + self.nKV) * row, (self.nH + 2 * self.nKV) * self.dH, self.nH, T, None,
                self.cos, self.sin, len(self.cos_h), self.dH, 1)
        fh.call("paged_attn", c, 0, self.out, self.q, self.nH, self.dH ** -0.5, T, None, 0, 0)
        fh.call("draft_verify", self.token, self.count, self.logits, self.V, self.drafted_from, self.V, self.draft, None, self.u, 1.0, self.nSeq, self.D, self.V)
        fh.call("paged_commit", c, T, self.count)

    def check(self):
        out, token, count = self.out.numpy(), self.token.numpy(), self.count.numpy()
        for s in range(self.nSeq):
            base = len(self.K[s])
            x = self.h["qkv"][s]
            turn = lambda y, t: ref.rotate(y, base + t, self.cos_h, self.sin_h, self.dH, 1)  # noqa: E731
            K = self.K[s] + [turn(x[t, self.nH:self.nH + self.nKV], t).astype(np.float32).astype(np.float16).astype(np.float64) for t in range(self.D + 1)]
            V = self.Vv[s] + [x[t, self.nH + self.nKV:].astype(np.float16).astype(np.float64) for t in range(self.D + 1)]
            Ka, Va = np.array(K), np.array(V)
            for t in range(self.D + 1):
                seen = np.arange(len(K)) <= base + t
                q = turn(x[t, :self.nH], t).astype(np.float32)
                want, p = ref.attend(q, Ka, Va, seen, self.dH ** -0.5)
                assert (np.abs(out[s, t] - want) <= out_bound(q, Ka, Va, p, seen, self.dH ** -0.5, "f16")).all(), (s, t)
            want = ref.verify(self.h["logits"][s], self.h["from"][s], self.h["draft"][s], self.h["u"][s], 1.0, self.D)
            assert count[s] == want[1] and (token[s] == want[0]).all(), s
            self.K[s], self.Vv[s] = K[:base + want[1]], V[:base + want[1]]
        assert self.len.numpy().tolist() == [len(k) for k in self.K]


def test_a_run_of_the_operators(fh):
    rng = np.random.default_rng(40)
    d = Drafting(fh, rng)
    for _ in range(12):
        d.upload(rng)
        d.queue()
        d.check()


def test_a_recorded_run_of_the_operators(fh):
    """One recorded step serves them all: lengths move on the device, from some slots of one piece to lengths that are cut into pieces;
    eager steps of another cache run between the replays."""
    rng = np.random.default_rng(41)
    d, other = Drafting(fh, rng, maxPages=100), Drafting(fh, rng, nSeq=2, D=2)
    d.upload(rng)
    d.queue()  # (a first step outside: recording starts with a warm allocator)
    d.check()
    d.upload(rng)
    fh.check(fh.lib.fg_graph_begin(), "begin")
    graph = ctypes.c_void_p()
    try:
        d.queue()
    finally:
        fh.check(fh.lib.fg_graph_end(ctypes.byref(graph)), "end")
    for n in range(40):
        d.upload(rng)
        fh.check(fh.lib.fg_graph_launch(graph), "launch")
        if n % 10 == 0:
            other.upload(rng)
            other.queue()
        d.check()
        if n % 10 == 0:
            other.check()
    fh.check(fh.lib.fg_graph_destroy(graph), "destroy")
    assert min(len(k) for k in d.K) > 60


def test_paged_js(fh):
    r = subprocess.run(["node", os.path.join(ROOT, "tests", "js", "paged.mjs")], cwd=ROOT, stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True, timeout=100)
    res = [json.loads(x) for x in r.stdout.splitlines() if x.startswith("{")]
    for x in res:
        print(x["test"], "ok" if x["ok"] else "FAIL", x.get("detail") or x.get("error", ""))
    assert r.returncode == 0 and res and all(x["ok"] for x in res), r.stdout[-4000:]
