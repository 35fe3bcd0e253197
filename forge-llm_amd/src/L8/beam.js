/**
 * L8 · beam search over a Transformer and its 4-bit cache, on the device: the choice
 * of the next beams over beams and vocabulary (fg_beam_select) and the beams'
 * caches following their parents in place (fg_kv4_reorder).  No counterpart in
 * forge-llm, whose sampling (src/L8/sampling.js) draws one token of one sequence.
 */
import { hip } from "../L2/device.js";
import { KV4Cache, checkEviction } from "../L5/attention.js";

/** The device arrays of a selection of `requests` x `beams`. */
class Beams {
  constructor(requests, beams) {
    const a = hip(), n = requests * beams;
    this.requests = requests; this.beams = beams; this.n = n;
    this._bufs = [];
    const alloc = () => { const h = a.alloc(n * 4); this._bufs.push(h); return h; };
    this.scores = [alloc(), alloc()]; this.done = [alloc(), alloc()];
    this.token = alloc(); this.parent = alloc();
    this.now = 0;  // which of the two holds the current beams
  }
  set(scores, done) {
    const a = hip();
    a.h2d(this.scores[this.now], Float32Array.from(scores));
    a.h2d(this.done[this.now], Int32Array.from(done));
  }
  /** Picks from logits [requests beams][vocab] on the device; the picked beams become the current ones. */
  select(logits, vocab, eos) {
    const a = hip(), was = this.now, is = 1 - was, stop = eos >= 0;
    a.beamSelect(this.scores[is], this.token, this.parent, stop ? this.done[is] : null, logits, vocab, this.scores[was],
                 stop ? this.done[was] : null, eos, this.requests, this.beams, vocab);
    this.now = is;
  }
  read(h, out) { hip().d2h(h, out); return out; }
  free() { for (const h of this._bufs) hip().free(h); this._bufs = []; }
}

/**
 * The next beams of `requests` requests from host arrays: logits [requests beams][vocab],
 * scores [requests beams] and, with `eos`, done flags.  Returns {scores, tokens, parents,
 * done}, each request's beams best first; parents count inside the request.
 */
export function beamSelect(logits, scores, { beams, vocab, requests = 1, done = null, eos = -1 }) {
  for (const [k, v] of [["beams", beams], ["vocab", vocab], ["requests", requests]])
    if (!Number.isInteger(v) || v <= 0) throw new RangeError(`beamSelect: ${k} must be a positive integer, got ${v}`);
  const n = requests * beams;
  if (!logits || logits.length < n * vocab) throw new RangeError(`beamSelect: ${n} x ${vocab} logits expected`);
  if (!scores || scores.length < n || (done && done.length < n)) throw new RangeError(`beamSelect: ${n} scores and flags expected`);
  if (!Number.isInteger(eos) || eos >= vocab) throw new RangeError(`beamSelect: eos ${eos}`);
  if (done && eos < 0) throw new RangeError("beamSelect: done needs eos");
  const a = hip(), b = new Beams(requests, beams), x = a.alloc(n * vocab * 4);
  try {
    a.h2d(x, Float32Array.from(logits.subarray ? logits.subarray(0, n * vocab) : logits.slice(0, n * vocab)));
    b.set(Array.prototype.slice.call(scores, 0, n), done ? Array.prototype.slice.call(done, 0, n) : new Int32Array(n));
    b.select(x, vocab, eos);
    return {
      scores: b.read(b.scores[b.now], new Float32Array(n)), tokens: b.read(b.token, new Int32Array(n)),
      parents: b.read(b.parent, new Int32Array(n)), done: eos >= 0 ? b.read(b.done[b.now], new Int32Array(n)) : new Int32Array(n),
    };
  } finally {
    a.free(x);
    b.free();
  }
}

/**
 * Beam search from `prompt` (token ids): `beams` continuations of up to `maxNew` tokens,
 * by the sum of their tokens' log probabilities, best first: [{tokens, score, done}].
 * A beam that takes `eos` (the Config's eosId; -1: none) is done and keeps its score.
 * With `budget` the cache holds that many tokens of every head, the newest `recent`
 * among them, and the others by accumulated attention.  The search ends at the Config's
 * maxSeq positions: its continuations are at most maxSeq - prompt.length + 1 tokens.
 */
export function beamSearch(transformer, prompt, { beams = 4, maxNew = 32, eos, budget = 0, recent = 0 } = {}) {
  const c = transformer.cfg, V = c.vocabSize;
  if (eos === undefined) eos = c.eosId < V ? c.eosId : -1;
  if (!prompt || prompt.length < 1) throw new RangeError("beamSearch: the prompt is empty");
  if (!Number.isInteger(beams) || beams < 1 || beams > 64 || beams > V) throw new RangeError(`beamSearch: ${beams} beams`);
  if (!Number.isInteger(maxNew) || maxNew < 1) throw new RangeError(`beamSearch: maxNew ${maxNew}`);
  if (!Number.isInteger(eos) || eos >= V) throw new RangeError(`beamSearch: eos ${eos}`);
  if (budget) checkEviction(budget, recent);
  if (prompt.length > c.maxSeq) throw new RangeError(`beamSearch: a prompt of ${prompt.length} tokens, the model has ${c.maxSeq} positions`);
  const most = Math.min(maxNew, c.maxSeq - prompt.length + 1);  // the last token taken is not run
  const room = budget ? budget + 1 : prompt.length + most;
  const cache = new KV4Cache(c.nLayers, room, c.nKvHeads, c.dHead, { sequences: beams, trackWeights: budget > 0 });
  const b = new Beams(1, beams);
  try {
    const idle = new Array(beams).fill(-1);
    let e;
    const step = (tokens) => {
      e = transformer._stepAll(tokens, cache);
      if (budget) cache.evict(budget, recent);
    };
    for (const t of prompt) {
      if (!(Number.isInteger(t) && t >= 0 && t < V)) throw new RangeError(`beamSearch: prompt token ${t}`);
      step([t].concat(idle.slice(1)));
    }
    cache.reorder(idle.map(() => 0));  // all beams go on from the prompt
    b.set(idle.map((_, i) => (i === 0 ? 0 : -Infinity)), new Int32Array(beams));
    let rows = idle.map(() => ({ tokens: [], done: false }));
    for (let n = 0; n < most; n++) {
      b.select(e.logits, V, eos);
      const tokens = b.read(b.token, new Int32Array(beams)), parents = b.read(b.parent, new Int32Array(beams));
      rows = rows.map((_, i) => {
        const p = rows[parents[i]];
        return p.done ? p : { tokens: p.tokens.concat(tokens[i]), done: tokens[i] === eos };
      });
      if (n + 1 === most || rows.every((r) => r.done)) break;
      hip().kv4Reorder(cache.handle, b.parent, beams);
      cache._follow(parents, beams);
      step(rows.map((r, i) => (r.done ? -1 : tokens[i])));
    }
    const scores = b.read(b.scores[b.now], new Float32Array(beams));
    return rows.map((r, i) => ({ tokens: r.tokens, score: scores[i], done: r.done }));
  } finally {
    b.free();
    transformer._dropKv4(cache);  // its graph and vectors belong to this cache
    cache.free();
  }
}
