"""fg_decode_step_kv4: the inference forward over a 4-bit cache of several
sequences, and the JavaScript API over it (tests/js/kv4.mjs).

The reference forward runs in 64 bits (RMSNorm, RoPE on the fp32 table, SwiGLU) and
attends to the values that the device's cache stands for, read back after every
step; the keys and values it computes itself have to be within the quantizer's
rounding of those.  (Quantizing its own would differ by a whole step wherever
the last bit of a key decides a code.)"""
import ctypes
import json
import os
import subprocess

import numpy as np
import pytest

import kv4_ref as ref
import oracle
from test_gpu_decode import Decoder, rope_f32
from util import TOL_FWD, rel_l2

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def rms(x, w, eps):
    return x / np.sqrt(np.mean(x * x) + eps) * w


class Model:
    """A decoder with vectors for nSeq sequences, its 4-bit cache, and the 64-bit forward."""

    def __init__(self, fh, kw, seed, nSeq, maxSeq, maxPos, types=None, track=False):
        self.fh, self.cfg = fh, oracle.Cfg(**kw)
        cfg = self.cfg
        params = oracle.init_weights(cfg, seed)
        P = oracle.split_params(cfg, params)
        P["tok_emb"][:] = np.random.default_rng(seed).standard_normal(P["tok_emb"].size).astype(np.float32) * 0.3
        self.dec = Decoder(fh, cfg, params, maxPos, types=types)
        self.N, self.maxSeq, self.dH = nSeq, maxSeq, cfg.dHead
        L, nKV, nb = cfg.nLayers, cfg.nKvHeads, cfg.dHead // 32
        A = fh.DeviceArray
        self.vec = [A((nSeq, n)) for n in (cfg.dim, cfg.dim, cfg.hidden)]
        self.dec.m.x, self.dec.m.q, self.dec.m.h = (a.ptr for a in self.vec)
        self.dec.m.attn_part = None
        slots = (L, nSeq, nKV, maxSeq)
        self.k, self.v = A.zeros(slots + (16 * nb,), np.uint8), A.zeros(slots + (16 * nb,), np.uint8)
        self.kd, self.vd = A.zeros(slots + (nb,), np.float16), A.zeros(slots + (nb,), np.float16)
        self.len, self.next = A.zeros((nSeq,), np.int32), A.zeros((nSeq,), np.int32)
        self.extra = [A.zeros(slots, np.float32), A.zeros(slots, np.int32)] if track else [None, None]
        self.cache = fh.Kv4Cache(L, nSeq, nKV, cfg.dHead, maxSeq, *[a.ptr if a else None for a in (
            self.k, self.v, self.kd, self.vd, self.len, self.next, *self.extra)])
        self.tokens, self.logits = A((nSeq,), np.int32), A((nSeq, cfg.vocab))
        self.cos, self.sin = (t.reshape(maxPos, -1) for t in rope_f32(maxPos, cfg.dHead, cfg.ropeTheta))

        def host(name, rows, cols):
            t, b = self.dec.host[name]
            return (oracle.dequantize(t, b, rows * cols) if t else b).astype(np.float64).reshape(rows, cols)

        D, H = cfg.dim, cfg.hidden
        self.emb, self.cls = host("tok_emb", cfg.vocab, D), host("wcls", cfg.vocab, D)
        self.layers = []
        for l in range(L):
            p = "layer.%d." % l
            self.layers.append({"wqkv": host(p + "wqkv", D + 2 * nKV * cfg.dHead, D), "wo": host(p + "wo", D, D),
                                "gate": host(p + "ffn_gate", H, D), "up": host(p + "ffn_up", H, D), "down": host(p + "ffn_down", D, H),
                                "ln1": self.dec.P[p + "ln1"].astype(np.float64), "ln2": self.dec.P[p + "ln2"].astype(np.float64)})
        self.ln_f = self.dec.P["ln_f"].astype(np.float64)

    def step(self, tokens):
        self.tokens.upload(np.array(tokens, np.int32))
        self.fh.check(self.fh.lib.fg_decode_step_kv4(ctypes.byref(self.dec.m), ctypes.byref(self.cache), self.tokens.ptr, self.logits.ptr),
                      "fg_decode_step_kv4")
        return self.logits.numpy()

    def turn(self, x, pos):
        a, b = x[..., 0::2], x[..., 1::2]
        c, s = self.cos[pos].astype(np.float64), self.sin[pos].astype(np.float64)
        return np.stack([a * c - b * s, a * s + b * c], -1).reshape(x.shape)

    def reference(self, s, token, pos, n):
        """Logits of sequence s, whose n-th slot is this token's, over the device's cache."""
        cfg = self.cfg
        nH, nKV, dH, D = cfg.nHeads, cfg.nKvHeads, self.dH, cfg.dim
        K, V = ref.values(self.k.numpy(), self.kd.numpy()), ref.values(self.v.numpy(), self.vd.numpy())
        step = {0: self.kd.numpy(), 1: self.vd.numpy()}
        x = self.emb[token].copy()
        for l, w in enumerate(self.layers):
            y = w["wqkv"] @ rms(x, w["ln1"], cfg.normEps)
            q = self.turn(y[:D].reshape(nH, dH), pos)
            k, v = self.turn(y[D:D + nKV * dH].reshape(nKV, dH), pos), y[D + nKV * dH:].reshape(nKV, dH)
            for i, (mine, cached) in enumerate(((k, K), (v, V))):
                # half a step inside the range, a whole one at its cut end, and the last bits of mine
                d = np.repeat(np.abs(step[i][l, s, :, n - 1].astype(np.float64)), 32, -1)
                assert (np.abs(mine - cached[l, s, :, n - 1]) <= d * (1 + 2.0 ** -8) + 1e-5 * np.abs(mine).max()).all()
            att, _ = ref.attend(q, K[l, s, :, :n].transpose(1, 0, 2), V[l, s, :, :n].transpose(1, 0, 2), 1 / np.sqrt(dH))
            x = x + w["wo"] @ att.ravel()
            z = rms(x, w["ln2"], cfg.normEps)
            g = w["gate"] @ z
            x = x + w["down"] @ (g / (1 + np.exp(-g)) * (w["up"] @ z))
        return self.cls @ rms(x, self.ln_f, cfg.normEps)


CASES = {
    "dh32": (dict(dim=64, hidden=96, nLayers=2, nHeads=2, nKvHeads=1, vocab=50, tied=1), None),
    "dh64_gqa": (dict(dim=256, hidden=300, nLayers=2, nHeads=4, nKvHeads=2, vocab=99, tied=0), None),
    "dh96": (dict(dim=192, hidden=101, nLayers=1, nHeads=2, nKvHeads=2, vocab=40, tied=1), None),
    "dh128_q8": (dict(dim=512, hidden=512, nLayers=2, nHeads=4, nKvHeads=1, vocab=64, tied=1),
                 dict(emb=8, cls=8, wqkv=8, wo=8, gate=8, down=8)),
    "dh256_q4k": (dict(dim=512, hidden=256, nLayers=1, nHeads=2, nKvHeads=1, vocab=40, tied=0),
                  dict(emb=12, cls=14, wqkv=12, wo=12, gate=12, down=14)),
    # wide enough for the unit forms of the products
    "units": (dict(dim=1536, hidden=2560, nLayers=1, nHeads=12, nKvHeads=4, vocab=64, tied=1),
              dict(emb=8, cls=8, wqkv=8, wo=8, gate=8, down=8)),
}


@pytest.mark.parametrize("name", list(CASES))
def test_step_against_the_reference_forward(fh, name):
    kw, types = CASES[name]
    N = 3
    m = Model(fh, kw, 5, N, 12, 16, types=types)
    rng = np.random.default_rng(3)
    at = [0] * N
    for t in range(9):
        tokens = rng.integers(0, m.cfg.vocab, N)
        tokens[1] = tokens[1] if t % 3 else -1  # idle every third step
        tokens[2] = m.cfg.vocab + 3 if t == 4 else tokens[2]
        got = m.step(tokens)
        for s in range(N):
            if not 0 <= tokens[s] < m.cfg.vocab:
                assert np.isnan(got[s]).all()
                continue
            at[s] += 1
            assert rel_l2(got[s], m.reference(s, tokens[s], at[s] - 1, at[s])) <= TOL_FWD, (t, s)
        np.testing.assert_array_equal(m.len.numpy(), at)
        np.testing.assert_array_equal(m.next.numpy(), at)


@pytest.mark.parametrize("name", ["dh64_gqa", "dh96", "units"])
def test_many_sequences_are_each_as_alone(fh, name):
    """One launch serves all sequences: each one's logits are those of a cache of its own, idle ones between them."""
    kw, types = CASES[name]
    N, steps = 37, 4
    rng = np.random.default_rng(8)
    m = Model(fh, kw, 5, N, 6, 16, types=types)
    tokens = rng.integers(0, m.cfg.vocab, (steps, N))
    tokens[rng.random((steps, N)) < 0.2] = -1
    got = [m.step(x) for x in tokens]
    for s in (0, 1, 17, N - 1):
        one = Model(fh, kw, 5, 1, 6, 16, types=types)
        for t in range(steps):
            want = one.step(tokens[t, s:s + 1])[0]
            if tokens[t, s] < 0:
                assert np.isnan(got[t][s]).all() and np.isnan(want).all()
            else:
                assert rel_l2(got[t][s], want) <= TOL_FWD, (s, t)
    np.testing.assert_array_equal(m.len.numpy(), (tokens >= 0).sum(0))
    m.cache.nSeq = 65536  # refused before anything is launched
    with pytest.raises(fh.ForgeError, match="above 65535"):
        m.step(tokens[0])


def test_full_caches_and_far_positions_stay_as_they_were(fh):
    kw = CASES["dh32"][0]
    m = Model(fh, kw, 6, 2, 3, 5, track=True)
    for t in range(3):
        assert np.isfinite(m.step([1, 2])).all()
    before = [a.numpy() for a in (m.k, m.v, m.kd, m.vd, m.len, m.next, m.extra[1])]
    assert np.isnan(m.step([1, 2])).all()  # full
    for a, b in zip((m.k, m.v, m.kd, m.vd, m.len, m.next, m.extra[1]), before):
        np.testing.assert_array_equal(a.numpy(), b)
    fh.call("kv4_evict", fh.ref(m.cache), 2, 1)
    assert np.isfinite(m.step([1, 2])).all()  # position 3
    fh.call("kv4_evict", fh.ref(m.cache), 2, 1)
    assert np.isfinite(m.step([1, -1])).all(1).tolist() == [True, False]
    fh.call("kv4_evict", fh.ref(m.cache), 2, 1)
    got = m.step([1, 2])  # the first is at position 5, past the table
    assert np.isnan(got[0]).all() and np.isfinite(got[1]).all()
    np.testing.assert_array_equal(m.next.numpy(), [5, 5])


def test_refusals(fh):
    kw = CASES["dh64_gqa"][0]
    m = Model(fh, kw, 7, 2, 8, 8)

    def refused(says):
        with pytest.raises(fh.ForgeError, match=says):
            m.step([1, 2])

    for field, bad, says in (("nLayers", 3, "for a model"), ("nKvHeads", 1, "for a model"), ("dHead", 32, "for a model"),
                             ("dHead", 48, "head size"), ("k", None, "null"), ("len", None, "null"), ("maxSeq", 0, "dimensions")):
        was = getattr(m.cache, field)
        setattr(m.cache, field, bad)
        refused(says)
        setattr(m.cache, field, was)
    m.dec.m.h = None
    refused("null model")


def test_kv4_js(fh):
    r = subprocess.run(["node", os.path.join(ROOT, "tests", "js", "kv4.mjs")], cwd=ROOT, stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True, timeout=100)
    res = [json.loads(x) for x in r.stdout.splitlines() if x.startswith("{")]
    for x in res:
        print(x["test"], "ok" if x["ok"] else "FAIL", x.get("detail") or x.get("error", ""))
    assert r.returncode == 0 and res and all(x["ok"] for x in res), r.stdout[-4000:]
