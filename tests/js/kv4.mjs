// The 4-bit cache and beam search through the JS API (KV4Cache, Transformer.forward /
// forwardAll over it, beamSelect, beamSearch).  Prints one JSON line per case.
import { Config, Transformer, KV4Cache, initWeights, beamSelect, beamSearch, RNG, hip } from "../../forge-llm_amd/src/index.js";

const out = [];
function rec(test, fn) {
  try {
    const r = fn();
    out.push({ test, ok: !!r.ok, detail: r.detail });
  } catch (e) {
    out.push({ test, ok: false, error: String(e && e.stack || e) });
  }
}
const throws = (fn, T) => { try { fn(); return false; } catch (e) { return e instanceof T; } };
const same = (x, y) => x.length === y.length && x.every((v, i) => Object.is(v, y[i]));
function normal(r, n) { const x = new Float32Array(n); for (let i = 0; i < n; i++) x[i] = r.normal(); return x; }
function model(seed = 7, o = {}) {
  const cfg = new Config(Object.assign({ dim: 128, hidden: 192, nLayers: 2, nHeads: 4, nKvHeads: 2, vocabSize: 90, maxSeq: 64, normEps: 1e-5, eosId: 2 }, o));
  const w = initWeights(cfg, seed), t = { tok_emb: w.tok_emb, ln_f: w.ln_f, wcls: null };
  const r = new RNG(seed + 1);
  for (let i = 0; i < w.tok_emb.length; i++) w.tok_emb[i] = r.normal() * 0.4;  // logits of some size
  for (let l = 0; l < cfg.nLayers; l++) t[`layer.${l}`] = w[`layer.${l}`];
  return { cfg, w: t };
}
const cacheFor = (cfg, maxSeq, opts) => new KV4Cache(cfg.nLayers, maxSeq, cfg.nKvHeads, cfg.dHead, opts);
function logProbs(x) {
  let m = -Infinity, s = 0;
  for (const v of x) m = Math.max(m, v);
  for (const v of x) s += Math.exp(v - m);
  return Array.from(x, (v) => v - m - Math.log(s));
}

rec("append, views and attention of several sequences", () => {
  const r = new RNG(3), S = 2, T = 5, nKV = 2, dH = 64, nH = 6, kvD = nKV * dH;
  const c = new KV4Cache(1, 8, nKV, dH, { sequences: S });
  const k = normal(r, S * T * kvD), v = normal(r, S * T * kvD), q = normal(r, S * nH * dH);
  c.append(0, k, v, T);
  const early = c.attend(0, q, nH, T);
  c.commit(T);
  const got = c.attend(0, q, nH);
  let worst = 0, far = 0;
  for (let s = 0; s < S; s++) {
    const K = c.kView(0, T, s), V = c.vView(0, T, s);
    // a stored value is at most a step off (the largest magnitude of its 32 over 8)
    for (let b = 0; b < T * kvD; b += 32) {
      let m = 0;
      for (let i = b; i < b + 32; i++) m = Math.max(m, Math.abs(k[s * T * kvD + i]));
      for (let i = b; i < b + 32; i++) far = Math.max(far, Math.abs(K[i] - k[s * T * kvD + i]) / (m / 8));
    }
    for (let h = 0; h < nH; h++) {
      const z = Math.floor(h / (nH / nKV)), x = [];
      for (let j = 0; j < T; j++) { let d = 0; for (let i = 0; i < dH; i++) d += q[(s * nH + h) * dH + i] * K[j * kvD + z * dH + i]; x.push(d / Math.sqrt(dH)); }
      const p = logProbs(x).map(Math.exp);
      for (let i = 0; i < dH; i++) {
        let o = 0;
        for (let j = 0; j < T; j++) o += p[j] * V[j * kvD + z * dH + i];
        worst = Math.max(worst, Math.abs(o - got[(s * nH + h) * dH + i]));
      }
    }
  }
  const ok = worst < 1e-5 && far < 1.01 && same(early, got) && c.len === T && c.nexts[1] === T && c.bytes() === 8 * S * nKV * (dH + dH / 8);
  c.free();
  return { ok, detail: `attention ${worst.toExponential(1)}, values ${far.toFixed(3)} steps` };
});

rec("forward over a 4-bit cache: recorded == op by op, one sequence == several", () => {
  const { cfg, w } = model();
  const r = new RNG(5), ids = [];
  for (let t = 0; t < 20; t++) ids.push(r.int(cfg.vocabSize));
  const G = new Transformer(cfg).loadWeights(w), E = new Transformer(cfg, { graph: false }).loadWeights(w);
  const M = new Transformer(cfg).loadWeights(w);
  const cG = cacheFor(cfg, 32), cE = cacheFor(cfg, 32), cM = cacheFor(cfg, 32, { sequences: 3 });
  let ok = true, worst = 0;
  for (let t = 0; t < ids.length; t++) {
    const g = Float32Array.from(G.forward(ids[t], t, cG)), e = E.forward(ids[t], t, cE);
    ok = ok && same(g, e) && g.every(Number.isFinite);
    // the second sequence sits out every other token, the third gets others
    const m = M.forwardAll([ids[t], t % 2 ? -1 : ids[t], ids[(t + 3) % ids.length]], cM), V = cfg.vocabSize;
    for (let i = 0; i < V; i++) worst = Math.max(worst, Math.abs(m[i] - g[i]));
    ok = ok && m.subarray(V, 2 * V).every((x) => (t % 2 ? Number.isNaN(x) : Number.isFinite(x)));
  }
  ok = ok && same(cG.kView(1, 20), cE.kView(1, 20)) && cM.lens[0] === 20 && cM.lens[1] === 10 && cM.nexts[2] === 20 && cG.len === 20;
  G.release(); E.release(); M.release();
  return { ok: ok && worst < 1e-4, detail: `one of three ${worst.toExponential(1)}` };
});

rec("a generation past the cache's size under a budget", () => {
  const { cfg, w } = model(11);
  const tr = new Transformer(cfg).loadWeights(w), c = cacheFor(cfg, 13, { trackWeights: true });
  let ok = true;
  for (let t = 0; t < 40; t++) {
    ok = ok && tr.forward((t * 7) % cfg.vocabSize, t, c).every(Number.isFinite);
    c.evict(12, 4);
    ok = ok && c.len === Math.min(t + 1, 12) && c.nexts[0] === t + 1;
  }
  for (let l = 0; l < cfg.nLayers; l++)
    for (let h = 0; h < cfg.nKvHeads; h++) {
      const p = Array.from(c.positions(l, 0, h)).sort((a, b) => a - b), wt = c.weights(l, 0, h);
      ok = ok && p.length === 12 && new Set(p).size === 12 && same(p.slice(8), [36, 37, 38, 39]) && wt.every((x) => x >= 0 && x < 1e3);
    }
  const full = cacheFor(cfg, 2);
  tr.forward(1, 0, full); tr.forward(1, 1, full);
  ok = ok && throws(() => tr.forward(1, 2, full), RangeError) && throws(() => full.evict(1), Error);
  tr.release();
  return { ok, detail: "" };
});

rec("an idle sequence keeps its weights, and what an eviction keeps goes by them", () => {
  const { cfg, w } = model(13);
  const tr = new Transformer(cfg).loadWeights(w);
  let ok = true;
  for (const slots of [20, 4000]) {  // a workgroup a head, and pieces
    const c = cacheFor(cfg, slots, { sequences: 3, trackWeights: true });
    for (let t = 0; t < 9; t++) tr.forwardAll([t, 3 * t % 90, 2 * t], c);
    const read = (s) => { const x = []; for (let l = 0; l < cfg.nLayers; l++) for (let h = 0; h < cfg.nKvHeads; h++) x.push(...c.weights(l, s, h)); return x; };
    const before = [read(0), read(1), read(2)];
    const logits = tr.forwardAll([5, -1, 900], c);
    ok = ok && logits.subarray(cfg.vocabSize).every(Number.isNaN) && before.every((x) => x.every((v) => v > 0)) &&
      same(read(1), before[1]) && same(read(2), before[2]) && !same(read(0).slice(0, 9), before[0].slice(0, 9));
    c.evict(4, 1);
    for (let l = 0; l < cfg.nLayers; l++)
      for (let h = 0; h < cfg.nKvHeads; h++) {
        const at = (l * cfg.nKvHeads + h) * 9, all = before[1].slice(at, at + 9);
        const keep = all.slice(0, 8).map((x, i) => [x, i]).sort((a, b) => b[0] - a[0] || a[1] - b[1]).slice(0, 3).map((x) => x[1]).concat([8]).sort((a, b) => a - b);
        ok = ok && same(Array.from(c.positions(l, 1, h)).sort((a, b) => a - b), keep);
      }
    c.free();
  }
  tr.release();
  return { ok, detail: "" };
});

rec("reorder and reset", () => {
  const r = new RNG(9), c = new KV4Cache(2, 6, 1, 32, { sequences: 4, trackWeights: true });
  for (let l = 0; l < 2; l++) c.append(l, normal(r, 4 * 3 * 32), normal(r, 4 * 3 * 32), 3);
  c.commit(3);
  const before = [0, 1, 2, 3].map((s) => c.kView(1, 3, s));
  c.reorder([1, 1, 0, 1], 4);
  let ok = [1, 1, 0, 1].every((p, s) => same(c.kView(1, 3, s), before[p]));
  c.reorder([1, 0, 0, 0], 2);
  ok = ok && same(c.kView(1, 3, 2), before[0]) && same(c.kView(1, 3, 3), before[0]);
  c.reset();
  return { ok: ok && c.len === 0 && c.attend(0, normal(r, 4 * 32), 1).every((x) => x === 0), detail: "" };
});

rec("beamSelect", () => {
  const r = new RNG(2), W = 3, V = 50, x = normal(r, 2 * W * V), s = normal(r, 2 * W), done = [0, 1, 0, 0, 0, 0];
  const got = beamSelect(x, s, { beams: W, vocab: V, requests: 2, done, eos: 7 });
  let ok = true;
  for (let q = 0; q < 2; q++) {
    const cand = [];
    for (let b = 0; b < W; b++) {
      const i = q * W + b;
      if (done[i]) cand.push([s[i], b, 7]);
      else logProbs(x.subarray(i * V, (i + 1) * V)).forEach((p, t) => cand.push([s[i] + p, b, t]));
    }
    cand.sort((a, b) => b[0] - a[0]);
    for (let i = 0; i < W; i++)
      ok = ok && got.tokens[q * W + i] === cand[i][2] && got.parents[q * W + i] === cand[i][1] && Math.abs(got.scores[q * W + i] - cand[i][0]) < 1e-5 &&
        got.done[q * W + i] === (done[q * W + cand[i][1]] || cand[i][2] === 7 ? 1 : 0);
  }
  return { ok, detail: Array.from(got.tokens).join(" ") };
});

rec("beamSearch: one beam is greedy, scores are the tokens' log probabilities, finished beams keep theirs", () => {
  const { cfg, w } = model(21);
  const tr = new Transformer(cfg).loadWeights(w), prompt = [3, 14, 15, 9];
  const rescore = (tokens) => {
    const c = cacheFor(cfg, 40);
    let s = 0, x;
    prompt.concat(tokens).forEach((t, i) => {
      if (i >= prompt.length) s += logProbs(x)[t];
      if (i < prompt.length + tokens.length - 1) x = Float32Array.from(tr.forward(t, i, c));
    });
    c.free();
    return s;
  };
  const greedy = [], c = cacheFor(cfg, 40);
  let x;
  prompt.forEach((t, i) => { x = tr.forward(t, i, c); });
  for (let n = 0; n < 8; n++) {
    let best = 0;
    x.forEach((v, t) => { if (v > x[best]) best = t; });
    greedy.push(best);
    x = tr.forward(best, prompt.length + n, c);
  }
  const one = beamSearch(tr, prompt, { beams: 1, maxNew: 8, eos: -1 });
  const four = beamSearch(tr, prompt, { beams: 4, maxNew: 8, eos: -1 });
  let worst = 0;
  for (const b of four.concat(one)) worst = Math.max(worst, Math.abs(b.score - rescore(b.tokens)));
  let ok = same(one[0].tokens, greedy) && worst < 1e-3 && four.every((b, i) => b.tokens.length === 8 && (i === 0 || four[i - 1].score >= b.score)) &&
    four[0].score >= one[0].score - 1e-4 && new Set(four.map((b) => b.tokens.join())).size === 4;
  const stop = four[0].tokens[2];  // a token that the search takes, as the end
  const ended = beamSearch(tr, prompt, { beams: 4, maxNew: 8, eos: stop });
  ok = ok && ended.some((b) => b.done) && ended.every((b) => b.done === (b.tokens[b.tokens.length - 1] === stop) && b.tokens.indexOf(stop) === (b.done ? b.tokens.length - 1 : -1));
  for (const b of ended) worst = Math.max(worst, Math.abs(b.score - rescore(b.tokens)));
  const held = beamSearch(tr, prompt, { beams: 3, maxNew: 20, eos: -1, budget: 10, recent: 3 });
  ok = ok && worst < 1e-3 && held.length === 3 && held.every((b) => b.tokens.length === 20 && Number.isFinite(b.score));
  tr.release();
  return { ok, detail: `rescored ${worst.toExponential(1)}` };
});

rec("beamSearch up to the model's last position", () => {
  const { cfg, w } = model(23, { maxSeq: 20 });
  const tr = new Transformer(cfg).loadWeights(w), prompt = [4, 8, 15, 16, 23];
  let ok = true;
  for (const o of [{}, { budget: 6, recent: 2 }]) {
    const long = beamSearch(tr, prompt, Object.assign({ beams: 3, maxNew: 50, eos: -1 }, o));
    const just = beamSearch(tr, prompt, Object.assign({ beams: 3, maxNew: 16, eos: -1 }, o));
    ok = ok && long.every((b, i) => b.tokens.length === 16 && same(b.tokens, just[i].tokens) && b.score === just[i].score);
  }
  const full = Array.from({ length: 20 }, (_, i) => i);
  const last = beamSearch(tr, full, { beams: 2, maxNew: 8, eos: -1 });
  ok = ok && last.every((b) => b.tokens.length === 1) && throws(() => beamSearch(tr, full.concat(1)), RangeError);
  tr.release();
  return { ok, detail: "" };
});

rec("errors", () => {
  const { cfg, w } = model();
  const tr = new Transformer(cfg).loadWeights(w), c = cacheFor(cfg, 8), c2 = cacheFor(cfg, 8, { sequences: 2 });
  const e = [
    throws(() => new KV4Cache(1, 8, 2, 48), RangeError), throws(() => new KV4Cache(0, 8, 2, 64), RangeError),
    throws(() => new KV4Cache(1, 8, 2, 64, { sequences: 0 }), RangeError),
    throws(() => tr.forward(1, 1, c), RangeError), throws(() => tr.forward(1, 0, c2), TypeError),
    throws(() => tr.forwardAll([1], c2), RangeError), throws(() => tr.forwardAll([1], {}), TypeError),
    throws(() => tr.forward(1, 0, new KV4Cache(cfg.nLayers, 8, cfg.nKvHeads, 64)), RangeError),
    throws(() => c.append(2, new Float32Array(64), new Float32Array(64)), RangeError),
    throws(() => c.append(0, new Float32Array(63), new Float32Array(64)), RangeError),
    throws(() => c.append(0, new Float32Array(64 * 9), new Float32Array(64 * 9), 9), RangeError),
    throws(() => c2.reorder([0, 2]), RangeError), throws(() => c2.reorder([0]), RangeError), throws(() => c2.reorder([0, 1], 3), RangeError),
    throws(() => cacheFor(cfg, 8, { trackWeights: true }).weights(0, 0.5), RangeError),
    throws(() => c.kView(0, 9), RangeError), throws(() => c.weights(0), Error), throws(() => c.attend(0, new Float32Array(96), 3), Error),
    throws(() => beamSearch(tr, []), RangeError), throws(() => beamSearch(tr, [1], { beams: 0 }), RangeError),
    throws(() => beamSearch(tr, [400]), RangeError), throws(() => beamSelect(new Float32Array(4), [0], { beams: 1, vocab: 5 }), RangeError),
    throws(() => beamSelect(new Float32Array(5), [0], { beams: 1, vocab: 5, eos: 5 }), Error),
  ];
  c.free();
  e.push(throws(() => tr.forward(1, 0, c), Error), throws(() => c.commit(), Error));
  tr.release();
  return { ok: e.every((x) => x), detail: e.map(Number).join("") };
});

rec("numbers that a call would not take as they are", () => {
  const { cfg, w } = model();
  const tr = new Transformer(cfg).loadWeights(w), r = new RNG(6);
  const c = new KV4Cache(1, 12, 2, 32, { trackWeights: true });
  c.append(0, normal(r, 9 * 64), normal(r, 9 * 64), 9);
  c.commit(9);
  const x = new Float32Array(10), s = [0, 0], q = normal(r, 128);
  const e = [
    // 2^32 + 5 is 5 in 32 bits: the device would evict, the lengths here would stay
    throws(() => c.evict(2 ** 32 + 5), RangeError), throws(() => c.evict(4.5), RangeError), throws(() => c.evict(4, 0.5), RangeError),
    throws(() => c.evict(), RangeError), throws(() => c.evict(4, 5), RangeError), throws(() => c.evict(4, null), RangeError),
    throws(() => c.evict(0), RangeError), c.len === 9, c.positions(0).length === 9,
    throws(() => c.attend(0, q, 4, 0, null), TypeError), throws(() => c.attend(0, q, 4, 0, "0.1"), TypeError),
    throws(() => c.attend(0, q), RangeError), throws(() => c.attend(0, q, 3), RangeError), throws(() => c.attend(0, q, 0), RangeError),
    throws(() => beamSelect(x, s, { beams: 2, vocab: 5, eos: 2.5 }), RangeError), throws(() => beamSelect(x, s, { beams: 2, vocab: 5, eos: null }), RangeError),
    throws(() => beamSelect(x, s, { beams: 2, vocab: 5, eos: NaN }), RangeError), throws(() => beamSelect(x, s, { beams: 2, vocab: 5, eos: 5 }), RangeError),
    throws(() => beamSearch(tr, [1], { eos: 2.5 }), RangeError), throws(() => beamSearch(tr, [1], { eos: null }), RangeError),
    throws(() => beamSearch(tr, [1], { eos: cfg.vocabSize }), RangeError), throws(() => beamSearch(tr, [1], { budget: 1.5 }), RangeError),
    throws(() => beamSearch(tr, [1], { budget: -1 }), RangeError), throws(() => beamSearch(tr, [1], { budget: 4, recent: 5 }), RangeError),
    beamSearch(tr, [1], { beams: 2, maxNew: 2, eos: -7, budget: 0, recent: 5 }).length === 2,
    c.attend(0, q, 4).every(Number.isFinite),
  ];
  c.evict(4, 1);
  e.push(c.len === 4);
  tr.release();
  return { ok: e.every((v) => v), detail: e.map(Number).join("") };
});

rec("caches in turn on one Transformer keep their recorded steps, a beam search leaves them", () => {
  const { cfg, w } = model(31), a = hip(), V = cfg.vocabSize;
  const calls = {};
  for (const name of ["decodeStepKv4", "graphEnd", "graphLaunch", "graphDestroy"]) {
    const f = a[name];
    calls[name] = { n: 0, restore: () => { a[name] = f; } };
    a[name] = (...x) => { calls[name].n++; return f(...x); };
  }
  let ok = true, detail = "";
  try {
    const tr = new Transformer(cfg).loadWeights(w), alone = new Transformer(cfg, { graph: false }).loadWeights(w);
    const caches = [1, 2, 1, 3].map((n) => cacheFor(cfg, 24, { sequences: n }));
    const refs = caches.map((c) => cacheFor(cfg, 24, { sequences: c.sequences }));
    const turn = (i, t) => {
      const ids = Array.from({ length: caches[i].sequences }, (_, s) => (7 * t + 13 * s + i) % V);
      return same(tr.forwardAll(ids, caches[i]), alone.forwardAll(ids, refs[i]));
    };
    for (let t = 0; t < 8; t++) for (let i = 0; i < 4; i++) ok = ok && turn(i, t);
    // the first step of a cache runs op by op, the second is recorded (one call each), the others replay
    ok = ok && calls.graphEnd.n === 4 && calls.graphLaunch.n === 4 * 7 && calls.graphDestroy.n === 0 && calls.decodeStepKv4.n === 4 * 2 + 4 * 8;
    detail += `${calls.graphEnd.n} ${calls.graphLaunch.n} ${calls.decodeStepKv4.n}`;
    caches[0].free();
    beamSearch(tr, [3, 1, 4], { beams: 2, maxNew: 4, eos: -1 });  // takes the freed cache's place
    const recorded = calls.graphEnd.n;
    for (let i = 1; i < 4; i++) ok = ok && turn(i, 9);
    ok = ok && calls.graphEnd.n === recorded;
    // one more than are kept, in turn
    caches.push(...[1, 2].map((n) => cacheFor(cfg, 24, { sequences: n })));
    refs.push(...[1, 2].map((n) => cacheFor(cfg, 24, { sequences: n })));
    for (let t = 10; t < 14; t++) for (let i = 1; i < 6; i++) ok = ok && turn(i, t);
    tr.release();
    ok = ok && calls.graphDestroy.n === calls.graphEnd.n;
    alone.release();
  } finally {
    for (const c of Object.values(calls)) c.restore();
  }
  return { ok, detail };
});

for (const r of out) console.log(JSON.stringify(r));
process.exit(out.every((r) => r.ok) ? 0 : 1);
