// The paged cache and speculative decoding through the JS API (PagedKVCache, Transformer.forwardChunk, verifyDrafts,
// speculate).  Prints one JSON line per case.
import { Config, Transformer, KVCache, PagedKVCache, initWeights, verifyDrafts, speculate, RNG } from "../../forge-llm_amd/src/index.js";

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
  for (let i = 0; i < w.tok_emb.length; i++) w.tok_emb[i] = r.normal() * 0.4;
  // a head of its own: tied to such an embedding it gives every token its own successor with certainty
  t.wcls = new Float32Array(w.tok_emb.length).map(() => r.normal() * 0.15);
  for (let l = 0; l < cfg.nLayers; l++) t[`layer.${l}`] = w[`layer.${l}`];
  return { cfg, w: t };
}
const paged = (cfg, pages, opts) => new PagedKVCache(cfg.nLayers, pages, cfg.nKvHeads, cfg.dHead, opts);
const best = (x) => x.reduce((b, v, i) => (v > x[b] ? i : b), 0);
// Worst difference of two rows of logits, to the largest of the second (both of fp32 models of this size).
const far = (x, y) => { let d = 0, m = 0; for (let i = 0; i < y.length; i++) { d = Math.max(d, Math.abs(x[i] - y[i])); m = Math.max(m, Math.abs(y[i])); } return d / m; };

rec("append, views, attention, commit and truncate of several sequences", () => {
  const r = new RNG(3), S = 2, T = 6, nKV = 2, dH = 32, nH = 4, kvD = nKV * dH;
  const c = new PagedKVCache(1, 9, nKV, dH, { sequences: S, pageSize: 4, maxPages: 5 });
  const k = normal(r, S * T * kvD), v = normal(r, S * T * kvD), q = normal(r, S * T * nH * dH), counts = [6, 3];
  c.append(0, k, v, T, { counts });
  const got = c.attend(0, q, nH, T, { counts });
  let worst = 0, ok = c.len === 0 && c.freePages === 9 - 3;
  for (let s = 0; s < S; s++)
    for (let t = 0; t < T; t++)
      for (let h = 0; h < nH; h++) {
        const z = Math.floor(h / 2), at = (s * T + t) * nH * dH + h * dH, x = [];
        if (t >= counts[s]) { for (let i = 0; i < dH; i++) ok = ok && got[at + i] === 0; continue; }
        for (let j = 0; j <= t; j++) { let d = 0; for (let i = 0; i < dH; i++) d += q[at + i] * k[(s * T + j) * kvD + z * dH + i]; x.push(Math.exp(d / Math.sqrt(dH))); }
        const sum = x.reduce((a, b) => a + b, 0);
        for (let i = 0; i < dH; i++) {
          let o = 0;
          for (let j = 0; j <= t; j++) o += x[j] / sum * v[(s * T + j) * kvD + z * dH + i];
          worst = Math.max(worst, Math.abs(o - got[at + i]));
        }
      }
  c.commit(counts);
  ok = ok && worst < 1e-5 && c.lens[0] === 6 && c.lens[1] === 3 && same(c.kView(0, 3, 1), k.subarray(T * kvD, (T + 3) * kvD)) && same(c.vView(0, 6, 0), v.subarray(0, 6 * kvD));
  c.truncate(0, 4);
  ok = ok && c.lens[0] === 4 && c.freePages === 7 && c.vView(0, 6, 0).subarray(4 * kvD).every((x) => x === 0);
  c.append(0, k, v, 1);
  c.commit();
  ok = ok && c.lens[0] === 5 && same(c.kView(0, 5, 0).subarray(4 * kvD), k.subarray(0, kvD)) && c.bytes() === 2 * 9 * nKV * 4 * dH * 4;
  c.forget(2, 0);
  ok = ok && c.kView(0, 4, 0).every((x) => x === 0) && c.freePages === 9 - 1 - 1;
  c.free();
  return { ok, detail: `attention ${worst.toExponential(1)}` };
});

rec("truncate after forget", () => {
  // 20 tokens in pages of 4, a window of 6: slots 0..11 of pages 0 to 2 are behind it for good, and 17 tokens see slot 12 on.
  const r = new RNG(5), kvD = 32, c = new PagedKVCache(1, 8, 1, 32, { pageSize: 4 }), k = normal(r, 20 * kvD);
  c.append(0, k, k, 20); c.commit(20); c.forget(6);
  let ok = c.freePages === 8 - 2 && c.lens[0] === 20;
  c.truncate(0, 17);
  ok = ok && throws(() => c.truncate(0, 16), RangeError) && c.lens[0] === 17 && same(c.kView(0, 17).subarray(12 * kvD), k.subarray(12 * kvD, 17 * kvD));
  c.truncate(0, 0);
  ok = ok && c.freePages === 8;
  c.append(0, k, k, 3); c.commit(3); c.truncate(0, 1);
  ok = ok && same(c.kView(0, 1), k.subarray(0, kvD));
  c.free();
  return { ok };
});

rec("rotation on the way into the pages", () => {
  const r = new RNG(9), T = 5, nKV = 1, dH = 64, nH = 3, theta = 1e4, c = new PagedKVCache(1, 8, nKV, dH, { type: "f16" });
  const k = normal(r, T * dH), v = normal(r, T * dH), q = normal(r, T * nH * dH);
  let worst = 0;
  for (const half of [false, true]) {
    const turned = c.append(0, k, v, T, { q, nHeads: nH, rope: { theta, dims: 32, half } }), K = c.kView(0, T);
    const turn = (x, at, t) => {
      const y = Array.from(x.subarray(at, at + dH));
      for (let i = 0; i < 16; i++) {
        const [a, b] = half ? [i, i + 16] : [2 * i, 2 * i + 1], w = t * theta ** (-2 * i / 32), p = y[a], z = y[b];
        y[a] = p * Math.cos(w) - z * Math.sin(w); y[b] = p * Math.sin(w) + z * Math.cos(w);
      }
      return y;
    };
    for (let t = 0; t < T; t++) {
      for (let h = 0; h < nH; h++) turn(q, (t * nH + h) * dH, t).forEach((x, i) => { worst = Math.max(worst, Math.abs(x - turned[(t * nH + h) * dH + i]) / 2 ** -24 / 4); });
      turn(k, t * dH, t).forEach((x, i) => { worst = Math.max(worst, Math.abs(x - K[t * dH + i]) / 2 ** -11 / 4); });  // values up to 4
    }
  }
  c.free();
  return { ok: worst <= 1.01, detail: `${worst.toFixed(3)} roundings` };
});

rec("forwardChunk == token by token, whatever the chunks; uncommitted tokens do not count", () => {
  const { cfg, w } = model(), r = new RNG(5), ids = [], V = cfg.vocabSize;
  for (let t = 0; t < 40; t++) ids.push(r.int(V));
  const M = new Transformer(cfg).loadWeights(w), one = new KVCache(cfg.nLayers, 64, cfg.kvDim);
  const want = ids.map((id, t) => Float32Array.from(M.forward(id, t, one)));
  let worst = 0, ok = true;
  for (const chunks of [[40], [1, 1, 38], [7, 20, 13], [33, 7]]) {
    const c = paged(cfg, 8, { pageSize: 8 });
    let at = 0;
    for (const n of chunks) {
      const lost = M.forwardChunk([ids.slice(at, at + n).reverse()], c, { commit: false });
      ok = ok && lost.every(Number.isFinite) && c.len === at;
      const got = M.forwardChunk([ids.slice(at, at + n)], c);
      for (let t = 0; t < n; t++) worst = Math.max(worst, far(got.subarray(t * V, (t + 1) * V), want[at + t]));
      at += n;
    }
    ok = ok && c.len === 40;
    c.free();
  }
  // a ragged batch: each sequence as alone
  const c = paged(cfg, 24, { sequences: 3, maxPages: 4 });
  const got = M.forwardChunk([ids.slice(0, 9), [], ids.slice(0, 4)], c), more = M.forwardChunk([ids.slice(9, 10), ids.slice(0, 2), ids.slice(4, 7)], c);
  for (let t = 0; t < 9; t++) worst = Math.max(worst, far(got.subarray(t * V, (t + 1) * V), want[t]));
  for (let t = 0; t < 4; t++) worst = Math.max(worst, far(got.subarray((18 + t) * V, (19 + t) * V), want[t]));
  ok = ok && got.subarray(9 * V, 18 * V).every(Number.isNaN) && got.subarray(22 * V).every(Number.isNaN);
  worst = Math.max(worst, far(more.subarray(0, V), want[9]), far(more.subarray(4 * V, 5 * V), want[1]), far(more.subarray(8 * V, 9 * V), want[6]));
  ok = ok && same(Array.from(c.lens), [10, 2, 7]);
  c.free(); one.free(); M.release();
  // fp32 products and sums of the same terms in another order, through two layers
  return { ok: ok && worst < 1e-5, detail: worst.toExponential(1) };
});

rec("forward of one token at the cache's next position", () => {
  const { cfg, w } = model(), V = cfg.vocabSize, M = new Transformer(cfg).loadWeights(w), ids = [3, 50, 89];
  const c = paged(cfg, 4), d = paged(cfg, 4), two = paged(cfg, 4, { sequences: 2 });
  let ok = throws(() => M.forward(1, 1, c), RangeError) && throws(() => M.forward(V, 0, c), RangeError) && throws(() => M.forward(1, 0, two), TypeError) && c.len === 0;
  ids.forEach((id, t) => { ok = ok && same(M.forward(id, t, c), M.forwardChunk([[id]], d)) && c.len === t + 1; });
  for (const x of [c, d, two]) x.free();
  M.release();
  return { ok };
});

rec("a window with sinks, and pages given back behind it", () => {
  const { cfg, w } = model(11), r = new RNG(6), V = cfg.vocabSize, ids = [];
  for (let t = 0; t < 50; t++) ids.push(r.int(V));
  const M = new Transformer(cfg).loadWeights(w), opts = { window: 10, sinks: 3 };
  const a = paged(cfg, 16, { pageSize: 4 }), b = paged(cfg, 16, { pageSize: 4 });
  let worst = 0;
  const all = M.forwardChunk([ids], a, opts);
  for (let t = 0; t < 50; t++) {
    worst = Math.max(worst, far(M.forwardChunk([[ids[t]]], b, opts), all.subarray(t * V, (t + 1) * V)));
    b.forget(10, 3);
  }
  const ok = worst < 1e-5 && b.freePages >= 16 - 5 && M.forwardChunk([[1]], b, opts).every(Number.isFinite);
  a.free(); b.free(); M.release();
  return { ok, detail: worst.toExponential(1) };
});

rec("speculate at temperature 0 is the target's greedy decoding, whoever drafts", () => {
  const big = model(21), small = model(22, { dim: 64, hidden: 96, nLayers: 1, nHeads: 2, nKvHeads: 1 });
  const T = new Transformer(big.cfg).loadWeights(big.w), S = new Transformer(small.cfg).loadWeights(small.w);
  let ok = true, detail = "";
  for (const prompt of [[5], [1, 2, 3, 4, 5, 6, 7], Array.from({ length: 60 }, (_, i) => (i * 7) % 90)]) {
    const c = new KVCache(big.cfg.nLayers, 64, big.cfg.kvDim), want = [];
    let x;
    prompt.forEach((id, t) => { x = T.forward(id, t, c); });
    for (let t = prompt.length; want.length < 30; t++) {
      want.push(best(x));
      if (want[want.length - 1] === 2 || t >= 64) break;
      x = T.forward(want[want.length - 1], t, c);
    }
    c.free();
    for (const [draft, drafts] of [[S, 4], [T, 3], [S, 0], [S, 1]]) {
      const got = speculate(T, draft, prompt, { maxNew: 30, drafts, temperature: 0, pageSize: 8 });
      ok = ok && same(got.tokens, want) && (draft !== T || got.accepted === got.drafted) && (draft !== S || got.accepted < got.drafted || got.drafted < 3) && got.steps <= want.length;
      detail += `${got.accepted}/${got.drafted} `;
    }
  }
  T.release(); S.release();
  return { ok, detail };
});

rec("speculate with random numbers: the same ones give the same tokens; a model drafting for itself is always right", () => {
  const big = model(31), small = model(32, { dim: 64, hidden: 96, nLayers: 1, nHeads: 2, nKvHeads: 1 });
  const T = new Transformer(big.cfg).loadWeights(big.w), S = new Transformer(small.cfg).loadWeights(small.w);
  const go = (draft, seed) => speculate(T, draft, [3, 1, 4], { maxNew: 25, drafts: 4, temperature: 0.9, seed, eos: -1, type: "f16" });
  const a = go(S, 5), b = go(S, 5), c = go(S, 6), d = go(T, 7);
  const ok = same(a.tokens, b.tokens) && !same(a.tokens, c.tokens) && a.tokens.length === 25 && d.accepted >= d.drafted - 1 && a.tokens.every((t) => t >= 0 && t < 90);
  T.release(); S.release();
  return { ok, detail: `${a.accepted}/${a.drafted}, itself ${d.accepted}/${d.drafted}` };
});

rec("verifyDrafts from host arrays", () => {
  const p = [0.5, 0.25, 0.25, 0.1, 0.1, 0.8].map(Math.log), q = [0.2, 0.6, 0.2].map(Math.log);
  const one = (d, u, o) => verifyDrafts(p, [[d]], u, Object.assign({ vocab: 3, draftLogits: q }, o)).tokens[0];
  const ok = same(one(0, [0.99, 0.15]), [0, 1]) && same(one(1, [0.41, 0.8]), [1, 2]) && same(one(1, [0.43, 0.8]), [0]) && same(one(1, [0.43, 0.9]), [2]) &&
    same(one(0, null, { temperature: 0 }), [0, 2]) && same(one(1, [0.2, 0.5], { draftLogits: null }), [1, 2]) && same(one(1, [0, 0], { drafted: [-1] }), []);
  return { ok };
});

rec("refusals", () => {
  const { cfg, w } = model(), M = new Transformer(cfg).loadWeights(w), c = paged(cfg, 3, { pageSize: 4, sequences: 2, maxPages: 2 });
  const R = RangeError, ok = [
    () => new PagedKVCache(1, 0, 1, 32), () => new PagedKVCache(1, 1, 1, 48), () => new PagedKVCache(1, 1, 1, 32, { pageSize: 12 }),
    () => new PagedKVCache(1, 1, 1, 32, { type: "bf16" }), () => new PagedKVCache(1, 2 ** 30, 1, 32, { maxPages: 2 ** 30 }),
    () => c.append(2, new Float32Array(128), new Float32Array(128)), () => c.append(0, new Float32Array(12), new Float32Array(128)),
    () => c.append(0, new Float32Array(128), new Float32Array(128), 1, { counts: [2, 0] }), () => c.append(0, new Float32Array(128), new Float32Array(128), 1, { rope: { theta: 0 } }),
    () => c.attend(0, new Float32Array(128), 3), () => c.attend(0, new Float32Array(256), 4, 1, { window: -1 }), () => c.reserve([5, 5]), () => c.reserve(9),
    () => c.commit([9, 0]), () => c.truncate(0, 1), () => c.truncate(2, 0), () => c.forget(0), () => c.kView(0, 9, 0), () => c.kView(0, 1, 2),
    () => M.forwardChunk([[1]], c), () => M.forwardChunk([[], []], c), () => M.forwardChunk([[90], []], c), () => M.forwardChunk([[1], [1]], c, { window: 1.5 }),
    () => speculate(M, M, []), () => speculate(M, M, [90]), () => speculate(M, M, [1], { temperature: -1 }), () => speculate(M, M, [1], { drafts: 2000 }),
    () => verifyDrafts([1, 2], [[0]], [0, 0], { vocab: 2 }), () => verifyDrafts([1, 2], [[]], [], { vocab: 2 }),
  ].every((f) => throws(f, R)) && throws(() => M.forwardChunk([[1]], {}), TypeError) && throws(() => c.attend(0, new Float32Array(256), 4, 1, { scale: "1" }), TypeError) && c.freePages === 3;
  c.free();
  const gone = throws(() => c.handle, Error) && throws(() => c.reserve(1), Error) && throws(() => M.forwardChunk([[1], []], c), Error);
  M.release();
  return { ok: ok && gone };
});

for (const o of out) console.log(JSON.stringify(o));
process.exit(out.every((o) => o.ok) ? 0 : 1);
