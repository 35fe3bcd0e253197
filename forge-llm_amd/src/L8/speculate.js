/**
 * L8 · speculative decoding over paged caches: a small model drafts a few tokens, the
 * target model runs them in one step (Transformer.forwardChunk), and fg_draft_verify says on the
 * device how many stand and what comes after them.  What comes out is distributed as
 * the target model's own sampling (temperature 0: is its greedy decoding).  No
 * counterpart in forge-llm, whose sampling (src/L8/sampling.js:28-98) draws one token from one row.
 */
import { RNG } from "../L0/numeric.js";
import { hip } from "../L2/device.js";
import { PagedKVCache } from "../L5/paged.js";

function checkTemperature(t, fn) {
  if (!(t === 0 || (t >= 1e-30 && t < Infinity))) throw new RangeError(`${fn}: temperature ${t}`);
}

/**
 * Verification from host arrays: logits [sequences][D + 1][vocab] of the target model, drafts [sequences][D]
 * (arrays), u [sequences][D + 1] uniform in [0, 1), and what the drafts were drawn from, draftLogits
 * [sequences][D][vocab] (left out: they were certain).  `drafted`: how many drafts each sequence has (below 0: it
 * takes no part).  Returns {tokens, counts}: of each sequence the drafts that stand and the token after them.
 */
export function verifyDrafts(logits, drafts, u, { vocab, draftLogits = null, drafted = null, temperature = 1 }) {
  const S = drafts.length, D = S ? drafts[0].length : 0, V = vocab;
  if (!Number.isInteger(V) || V <= 0) throw new RangeError(`verifyDrafts: vocab ${V}`);
  if (!S || !drafts.every((d) => d.length === D)) throw new RangeError("verifyDrafts: drafts must be rows of one length");
  checkTemperature(temperature, "verifyDrafts");
  const need = (x, n, what) => { if (!x || x.length < n) throw new RangeError(`verifyDrafts: ${n} ${what} expected`); return x; };
  need(logits, S * (D + 1) * V, "logits");
  if (temperature > 0) need(u, S * (D + 1), "random numbers");
  if (draftLogits) need(draftLogits, S * D * V, "logits of the drafts");
  if (drafted) need(drafted, S, "numbers of drafts");
  // (an Int32Array would take 2^32 + 1 as 1)
  const whole = (x, what) => { for (const v of x) if (v !== (v | 0)) throw new RangeError(`verifyDrafts: ${what} ${v}`); };
  for (const d of drafts) whole(d, "draft");
  if (drafted) whole(Array.prototype.slice.call(drafted, 0, S), "number of drafts");
  const a = hip(), held = [];
  const up = (x) => { const h = a.alloc(Math.max(4, x.byteLength)); held.push(h); if (x.length) a.h2d(h, x); return h; };
  const f32 = (x, n) => (x instanceof Float32Array ? x.subarray(0, n) : Float32Array.from(Array.prototype.slice.call(x, 0, n)));
  try {
    const x = up(f32(logits, S * (D + 1) * V)), y = draftLogits && D ? up(f32(draftLogits, S * D * V)) : null;
    const d = up(Int32Array.from([].concat(...drafts.map((r) => Array.from(r))))), n = drafted ? up(Int32Array.from(Array.prototype.slice.call(drafted, 0, S))) : null;
    const r = temperature > 0 ? up(f32(u, S * (D + 1))) : null;
    const token = new Int32Array(S * (D + 1)), count = new Int32Array(S), bt = up(token), bc = up(count);
    a.draftVerify(bt, bc, x, V, y, V, d, n, r, temperature, S, D, V);
    a.d2h(bt, token); a.d2h(bc, count);
    return { tokens: Array.from(count, (c, s) => Array.from(token.subarray(s * (D + 1), s * (D + 1) + c))), counts: Array.from(count) };
  } finally {
    for (const h of held) a.free(h);
  }
}

/**
 * Up to `maxNew` tokens after `prompt` (token ids) by `target`, drafted by `draft` (Transformers of one vocabulary),
 * `drafts` at a time; ends with `eos` (the target Config's eosId; -1: none) or at the last position of either
 * model.  window and sinks bound what the target's tokens see.  Returns {tokens, steps, drafted, accepted}:
 * the target's steps, and how many drafts there were and stood.
 */
export function speculate(target, draft, prompt, opts = {}) {
  const pick = (k, d) => (opts[k] === undefined ? d : opts[k]);
  const c = target.cfg, V = c.vocabSize, maxNew = pick("maxNew", 32), drafts = pick("drafts", 4), temperature = pick("temperature", 1);
  const window = pick("window", 0), sinks = pick("sinks", 0), pageSize = pick("pageSize", 16), type = pick("type", "f32");
  const eos = pick("eos", c.eosId < V ? c.eosId : -1), rng = new RNG(pick("seed", 1));
  if (draft.cfg.vocabSize !== V) throw new RangeError(`speculate: vocabularies of ${V} and ${draft.cfg.vocabSize} tokens`);
  if (!prompt || prompt.length < 1) throw new RangeError("speculate: the prompt is empty");
  for (const t of prompt) if (!(Number.isInteger(t) && t >= 0 && t < V)) throw new RangeError(`speculate: prompt token ${t}`);
  if (!Number.isInteger(maxNew) || maxNew < 1) throw new RangeError(`speculate: maxNew ${maxNew}`);
  if (!Number.isInteger(drafts) || drafts < 0 || drafts > 1023) throw new RangeError(`speculate: ${drafts} drafts`);
  if (!Number.isInteger(eos) || eos >= V) throw new RangeError(`speculate: eos ${eos}`);
  checkTemperature(temperature, "speculate");
  const positions = Math.min(c.maxSeq, draft.cfg.maxSeq);
  if (prompt.length > positions) throw new RangeError(`speculate: a prompt of ${prompt.length} tokens, the models have ${positions} positions`);
  const most = Math.min(maxNew, positions - prompt.length + 1);  // the last token taken is not run
  const pages = Math.ceil(Math.min(positions, prompt.length + most) / pageSize);
  const a = hip(), held = [], result = { tokens: [], steps: 0, drafted: 0, accepted: 0 };
  const alloc = (n) => { const h = a.alloc(Math.max(1, n) * 4); held.push(h); return h; };
  const cacheOf = (cfg) => new PagedKVCache(cfg.nLayers, pages, cfg.nKvHeads, cfg.dHead, { pageSize, type });
  let mine = null, theirs = null;
  try {
    mine = cacheOf(c);
    theirs = cacheOf(draft.cfg);
    const rows = alloc(drafts * V), chosen = alloc(drafts), u = alloc(drafts + 1), token = alloc(drafts + 1), count = alloc(1);
    const uniform = (n) => { const x = new Float32Array(n); for (let i = 0; i < n; i++) x[i] = Math.min(rng.next(), 1 - 2 ** -24); a.h2d(u, x); };
    const known = Array.from(prompt.slice(0, prompt.length - 1));
    for (let t = 0; t < known.length; t += 64) {
      target._chunk([known.slice(t, t + 64)], mine, { window, sinks });
      draft._chunk([known.slice(t, t + 64)], theirs);
    }
    let fed = [prompt[prompt.length - 1]];  // what the drafting model has not seen yet, the newest token last
    while (result.tokens.length < most) {
      const base = mine.len, newest = fed[fed.length - 1], left = most - result.tokens.length;
      const D = Math.min(drafts, left - 1, positions - base - 1), picked = [];
      for (let t = 0; t < D; t++) {
        const feed = t === 0 ? fed : [picked[t - 1]], e = draft._chunk([feed], theirs);
        const row = a.view(e.logits, (feed.length - 1) * V * 4, V * 4), got = new Int32Array(1);
        a.d2d(a.view(rows, t * V * 4, V * 4), row, V * 4);
        uniform(1);
        a.draftVerify(token, count, row, V, null, V, null, null, u, temperature, 1, 0, V);
        a.d2h(token, got);
        if (got[0] < 0) throw new Error("speculate: the drafting model's logits are not numbers");
        picked.push(got[0]);
      }
      const e = target._chunk([[newest].concat(picked)], mine, { window, sinks, commit: false });
      if (D) a.h2d(chosen, Int32Array.from(picked));
      uniform(D + 1);
      a.draftVerify(token, count, e.logits, V, D ? rows : null, V, D ? chosen : null, null, u, temperature, 1, D, V);
      a.pagedCommit(mine.handle, D + 1, count);
      const got = new Int32Array(D + 1), n = new Int32Array(1);
      a.d2h(token, got); a.d2h(count, n);
      mine._advance(n);
      const stood = n[0] - 1, next = got[stood];
      if (next < 0) throw new Error("speculate: the model's logits are not numbers");
      result.steps++; result.drafted += D; result.accepted += stood;
      for (let t = 0; t <= stood; t++) {
        result.tokens.push(got[t]);
        if (got[t] === eos) return result;
      }
      // The drafting model has run the newest token and all drafts but the last; it goes on after those that stood.
      if (stood < D) theirs.truncate(0, base + 1 + stood);
      fed = D === 0 ? fed.concat(next) : stood === D ? [picked[D - 1], next] : [next];
    }
    return result;
  } finally {
    for (const h of held) a.free(h);
    for (const [m, cache] of [[target, mine], [draft, theirs]])
      if (cache) {
        m._dropPaged(cache);
        cache.free();
      }
  }
}
