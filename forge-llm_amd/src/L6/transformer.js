/**
 * L6 · model hyper-parameters and the inference model.  Config has the same
 * fields, defaults and derived dimensions as forge-llm's Config
 * (src/L6/transformer.js:29-53), including the GQA divisibility check;
 * Transformer is its inference forward (:69-184) on the device.
 */
import { hip } from "../L2/device.js";
import { KVCache, KV4Cache } from "../L5/attention.js";
import { PagedKVCache } from "../L5/paged.js";
import { info, rowBytes } from "../L3/quant.js";

function pick(o, k, d) { return o[k] === undefined || o[k] === null ? d : o[k]; }

export class Config {
  constructor(o = {}) {
    this.dim = pick(o, "dim", 288);
    this.hidden = pick(o, "hidden", 768);
    this.nLayers = pick(o, "nLayers", 6);
    this.nHeads = pick(o, "nHeads", 6);
    this.nKvHeads = pick(o, "nKvHeads", 6);
    this.vocabSize = pick(o, "vocabSize", 32000);
    this.maxSeq = pick(o, "maxSeq", 1024);
    this.normEps = pick(o, "normEps", 1e-5);
    this.ropeTheta = pick(o, "ropeTheta", 10000);
    this.bosId = pick(o, "bosId", 1);
    this.eosId = pick(o, "eosId", 2);
    this._derive();
  }
  _derive() {
    if (this.nHeads % this.nKvHeads !== 0) {
      throw new Error(`GQA needs nHeads (${this.nHeads}) divisible by nKvHeads (${this.nKvHeads})`);
    }
    this.dHead = Math.floor(this.dim / this.nHeads);
    this.kvDim = this.nKvHeads * this.dHead;
    this.qkvOut = (this.nHeads + 2 * this.nKvHeads) * this.dHead;
    this.groupSize = this.nHeads / this.nKvHeads;
  }
}

// ── inference forward (transformer.js:69-184) ───────────────────────────────

/** fp32 RoPE table of the inference path (special.js:116-127): angles in
 *  fp64, cos/sin rounded to fp32. */
function ropeTableF32(maxPos, dim, theta) {
  const half = dim / 2;
  const cos = new Float32Array(maxPos * half), sin = new Float32Array(maxPos * half);
  for (let p = 0; p < maxPos; p++) {
    for (let i = 0; i < dim; i += 2) {
      const freq = 1 / Math.pow(theta, i / dim);
      const ang = p * freq;
      cos[p * half + i / 2] = Math.cos(ang);
      sin[p * half + i / 2] = Math.sin(ang);
    }
  }
  return { cos, sin };
}

/** f32 vectors (norm weights): a Float32Array / array, or a QuantLinear of
 *  type 0. */
function f32Weights(w, n, what) {
  if (w && typeof w === "object" && !ArrayBuffer.isView(w) && !Array.isArray(w) && "type" in w) {
    if (w.type !== 0) throw new Error(`Transformer.loadWeights: ${what} must be f32, got type ${w.type}`);
    w = w.bytes;
  }
  if (!w || w.length !== n) throw new RangeError(`Transformer.loadWeights: ${what} needs ${n} values, got ${w ? w.length : 0}`);
  return w instanceof Float32Array ? w : Float32Array.from(w);
}

/** A weight matrix [N, K]: f32 values, or a QuantLinear ({type, bytes, N, K},
 *  nn.js:19-40) of any type the decode kernels read (asQuantLinear,
 *  transformer.js:66-70).  Returns {type, data} with data the bytes to upload. */
function matWeights(w, N, K, what) {
  if (w && typeof w === "object" && !ArrayBuffer.isView(w) && !Array.isArray(w) && "type" in w) {
    if ((w.N !== undefined && w.N !== N) || (w.K !== undefined && w.K !== K))
      throw new RangeError(`Transformer.loadWeights: ${what} is [${w.N}, ${w.K}], [${N}, ${K}] expected`);
    if (w.type === 0) return { type: 0, data: f32Weights(w.bytes, N * K, what) };
    if (!DEVICE_TYPES.has(w.type)) throw new Error(`Transformer.loadWeights: ${what} has ggml type ${w.type}, which the device decode does not read`);
    const bs = info(w.type).blockSize;
    if (K % bs !== 0) throw new RangeError(`Transformer.loadWeights: ${what}: rows of ${K} are not whole ${bs}-element blocks`);
    const need = rowBytes(w.type, K) * N;
    const b = w.bytes instanceof Uint8Array ? w.bytes : new Uint8Array(w.bytes.buffer, w.bytes.byteOffset, w.bytes.byteLength);
    if (b.byteLength < need) throw new RangeError(`Transformer.loadWeights: ${what} holds ${b.byteLength} bytes, ${need} needed`);
    return { type: w.type, data: b.subarray(0, need) };
  }
  return { type: 0, data: f32Weights(w, N * K, what) };
}
const DEVICE_TYPES = new Set([0, 1, 2, 6, 8, 12, 13, 14]);

const GRAPHS_KEPT = 4;
// Vectors of a paged cache's steps are kept from one to the next up to this many bytes; what a long chunk took beyond it
// (8192 rows of 32000 logits: 1 GB) goes back when the chunk is done.
const VECTORS_KEPT = 64 << 20;

/**
 * Inference model (transformer.js:69-184) on the device: `loadWeights(w)`
 * uploads the weights once; `forward(token, pos, cache)` runs one decode step
 * (fg_decode_step: embed, per layer RMSNorm → QKV → RoPE → KV write →
 * attention → Wo + residual → RMSNorm → SwiGLU FFN + residual, final norm,
 * LM head: 5 launches per layer + 1) and returns the logits as a host Float32Array (the same array
 * every call, like the reference's `this.logits`).  The first step with a
 * cache runs op by op; the second is recorded as a HIP graph that later
 * steps with that cache replay (token and position are read from device
 * memory); `opts.graph = false` issues every step op by op.  `cache` must be
 * this package's device KVCache, or its KV4Cache: `forward` takes one of one
 * sequence, at the sequence's next position, `forwardAll(tokens, cache)` one token
 * of every sequence (fg_decode_step_kv4).  Recorded steps are kept for the last four
 * caches of each kind.  `forwardChunk(tokens, cache)` takes several tokens of every
 * sequence of a PagedKVCache in one step (fg_decode_step_paged), op by op; `forward` takes
 * one of one sequence, at the sequence's next position.
 */
export class Transformer {
  constructor(config, opts = {}) {
    this.cfg = config instanceof Config ? config : new Config(config);
    this._graphOn = !(opts && opts.graph === false);
    const c = this.cfg;
    if (c.dim % c.nHeads !== 0) throw new Error(`Transformer: dim ${c.dim} must be a multiple of nHeads ${c.nHeads}`);
    this.logits = new Float32Array(c.vocabSize);
    this._w = null; this._model = null; this._graphs = []; this._kv4 = []; this._paged = [];
  }

  loadWeights(w) {
    const c = this.cfg, a = hip();
    this.release();
    const D = c.dim, H = c.hidden, V = c.vocabSize;
    const bufs = [];
    const up = (arr) => { const h = a.alloc(Math.max(1, arr.byteLength)); a.h2d(h, arr); bufs.push(h); return h; };
    const mat = (x, N, K, what) => { const m = matWeights(x, N, K, what); return { type: m.type, h: up(m.data) }; };
    const tok = mat(w.tok_emb, V, D, "tok_emb");
    const wcls = w.wcls ? mat(w.wcls, V, D, "wcls") : tok;
    const layers = [];
    for (let l = 0; l < c.nLayers; l++) {
      const L = w[`layer.${l}`];
      if (!L) throw new Error(`Transformer.loadWeights: layer.${l} missing`);
      const qkv = mat(L.wqkv, c.qkvOut, D, `layer.${l}.wqkv`), wo = mat(L.wo, D, D, `layer.${l}.wo`);
      const g = mat(L.ffn_gate, H, D, `layer.${l}.ffn_gate`), u = mat(L.ffn_up, H, D, `layer.${l}.ffn_up`);
      const dn = mat(L.ffn_down, D, H, `layer.${l}.ffn_down`);
      if (g.type !== u.type)
        throw new Error(`Transformer.loadWeights: layer.${l} ffn_gate (type ${g.type}) and ffn_up (type ${u.type}) must share a type on the device`);
      layers.push({
        ln1: up(f32Weights(L.ln1, D, `layer.${l}.ln1`)), ln2: up(f32Weights(L.ln2, D, `layer.${l}.ln2`)),
        wqkv: qkv.h, wo: wo.h, gate: g.h, up: u.h, down: dn.h,
        wqkv_type: qkv.type, wo_type: wo.type, gate_type: g.type, up_type: u.type, down_type: dn.type,
      });
    }
    const rt = ropeTableF32(c.maxSeq, c.dHead, c.ropeTheta);
    const scratch = (n) => { const h = a.alloc(Math.max(1, n) * 4); bufs.push(h); return h; };
    this._w = {
      bufs, tok: tok.h, wcls: wcls.h, emb_type: tok.type, cls_type: wcls.type, layers,
      ln_f: up(f32Weights(w.ln_f, D, "ln_f")), rope_cos: up(rt.cos), rope_sin: up(rt.sin),
      x: scratch(D), q: scratch(c.nHeads * c.dHead), h: scratch(H), logits: scratch(V),
      state: a.alloc(8), stateHost: new Int32Array(2), part: null, partSeq: 0,
    };
    bufs.push(this._w.state);
    return this;
  }

  _modelFor(cache) {
    const c = this.cfg, W = this._w, a = hip();
    if (W.partSeq < cache.maxSeq || this._model === null || this._modelSeq !== cache.maxSeq) {
      this._dropGraphs();
      if (W.partSeq < cache.maxSeq) {
        if (W.part) a.free(W.part);
        W.part = a.alloc(a.decodePartLen(c.nHeads, c.dHead, cache.maxSeq) * 8);
        W.partSeq = cache.maxSeq;
      }
      this._model = a.decodeModel({
        dim: c.dim, hidden: c.hidden, nLayers: c.nLayers, nHeads: c.nHeads, nKvHeads: c.nKvHeads,
        vocab: c.vocabSize, maxSeq: cache.maxSeq, normEps: c.normEps, tok_emb: W.tok, ln_f: W.ln_f, wcls: W.wcls,
        emb_type: W.emb_type, cls_type: W.cls_type,
        rope_cos: W.rope_cos, rope_sin: W.rope_sin, x: W.x, q: W.q, h: W.h, attn_part: W.part,
        layers: W.layers,
      });
      this._modelSeq = cache.maxSeq;
    }
    return this._model;
  }

  // The model over vectors of every sequence of a 4-bit cache, and its recorded step,
  // kept for the last GRAPHS_KEPT caches used.
  _kv4For(cache) {
    const c = this.cfg, W = this._w, a = hip();
    const known = this._kv4.findIndex((e) => e.cache === cache);
    if (known >= 0) {
      this._kv4.push(this._kv4.splice(known, 1)[0]);
      return this._kv4[this._kv4.length - 1];
    }
    for (const e of this._kv4.slice()) if (e.cache.freed) this._dropKv4(e.cache);
    while (this._kv4.length >= GRAPHS_KEPT) this._dropKv4(this._kv4[0].cache);
    const N = cache.sequences, bufs = [];
    const scratch = (n) => { const h = a.alloc(n * 4); bufs.push(h); return h; };
    try {
      const x = scratch(N * c.dim);
      const model = a.decodeModel({
        dim: c.dim, hidden: c.hidden, nLayers: c.nLayers, nHeads: c.nHeads, nKvHeads: c.nKvHeads,
        vocab: c.vocabSize, maxSeq: c.maxSeq, normEps: c.normEps, tok_emb: W.tok, ln_f: W.ln_f, wcls: W.wcls,
        emb_type: W.emb_type, cls_type: W.cls_type,
        rope_cos: W.rope_cos, rope_sin: W.rope_sin, x, q: scratch(N * c.dim), h: scratch(N * c.hidden), attn_part: x,
        layers: W.layers,
      });
      const e = { cache, model, bufs, tokens: scratch(N), logits: scratch(N * c.vocabSize), graph: null, steps: 0 };
      this._kv4.push(e);
      return e;
    } catch (err) {
      for (const h of bufs) a.free(h);
      throw err;
    }
  }
  // Of one cache, or of all.
  _dropKv4(cache) {
    const a = hip();
    for (const e of this._kv4) {
      if (cache && e.cache !== cache) continue;
      if (e.graph) a.graphDestroy(e.graph);
      for (const h of e.bufs) a.free(h);
    }
    this._kv4 = this._kv4.filter((e) => cache && e.cache !== cache);
  }

  // The model over the vectors of `rows` tokens for a paged cache, kept for the last GRAPHS_KEPT caches used.
  _pagedFor(cache, rows) {
    const c = this.cfg, W = this._w, a = hip();
    const known = this._paged.findIndex((e) => e.cache === cache);
    if (known >= 0 && this._paged[known].rows >= rows) {
      this._paged.push(this._paged.splice(known, 1)[0]);
      return this._paged[this._paged.length - 1];
    }
    this._dropPaged(cache);
    for (const e of this._paged.slice()) if (e.cache.freed) this._dropPaged(e.cache);
    while (this._paged.length >= GRAPHS_KEPT) this._dropPaged(this._paged[0].cache);
    const bufs = [];
    const scratch = (n) => { const h = a.alloc(n * 4); bufs.push(h); return h; };
    try {
      const x = scratch(rows * c.dim);
      const model = a.decodeModel({
        dim: c.dim, hidden: c.hidden, nLayers: c.nLayers, nHeads: c.nHeads, nKvHeads: c.nKvHeads,
        vocab: c.vocabSize, maxSeq: c.maxSeq, normEps: c.normEps, tok_emb: W.tok, ln_f: W.ln_f, wcls: W.wcls,
        emb_type: W.emb_type, cls_type: W.cls_type,
        rope_cos: W.rope_cos, rope_sin: W.rope_sin, x, q: scratch(rows * c.dim), h: scratch(rows * c.hidden), attn_part: x,
        layers: W.layers,
      });
      const e = { cache, rows, model, bufs, tokens: scratch(rows), count: scratch(cache.sequences), logits: scratch(rows * c.vocabSize) };
      this._paged.push(e);
      return e;
    } catch (err) {
      for (const h of bufs) a.free(h);
      throw err;
    }
  }
  // Of one cache, or of all.
  _dropPaged(cache) {
    const a = hip();
    for (const e of this._paged)
      if (!cache || e.cache === cache) for (const h of e.bufs) a.free(h);
    this._paged = this._paged.filter((e) => cache && e.cache !== cache);
  }

  /** Queues tokens[s] (arrays) of every sequence of a paged cache; rows [sequences][T] of logits stay in device
   *  memory (`logits` of what it returns), T being the most tokens of a sequence. */
  _chunk(tokens, cache, opts = {}) {
    const c = this.cfg, a = hip(), { window = 0, sinks = 0, commit = true } = opts;
    if (!this._w) throw new Error("Transformer.forwardChunk: call loadWeights first");
    if (!(cache instanceof PagedKVCache)) throw new TypeError("Transformer.forwardChunk: cache must be a PagedKVCache");
    const handle = cache.handle, S = cache.sequences;
    if (cache.nLayers !== c.nLayers || cache.nKvHeads !== c.nKvHeads || cache.dHead !== c.dHead)
      throw new RangeError("Transformer.forwardChunk: cache shape does not match the Config");
    if (!tokens || tokens.length !== S || !Array.from(tokens).every((t) => t && t.length !== undefined))
      throw new RangeError(`Transformer.forwardChunk: tokens of ${S} sequences expected`);
    for (const [k, v] of [["window", window], ["sinks", sinks]])
      if (!Number.isInteger(v) || v < 0 || v > 0x7FFFFFFF) throw new RangeError(`Transformer.forwardChunk: ${k} ${v}`);
    const counts = Int32Array.from(tokens, (t) => t.length), T = Math.max.apply(null, Array.from(counts));
    if (T < 1 || S * T > 65535) throw new RangeError(`Transformer.forwardChunk: ${S} sequences of ${T} tokens`);
    const ids = new Int32Array(S * T).fill(-1);
    for (let s = 0; s < S; s++) {
      for (let t = 0; t < counts[s]; t++) {
        const id = tokens[s][t];
        if (!(Number.isInteger(id) && id >= 0 && id < c.vocabSize)) throw new RangeError(`Transformer.forwardChunk: token ${id}`);
        ids[s * T + t] = id;
      }
      if (cache.lens[s] + counts[s] > c.maxSeq) throw new RangeError(`Transformer.forwardChunk: sequence ${s} runs past position ${c.maxSeq}`);
    }
    cache.reserve(counts);
    const e = this._pagedFor(cache, S * T);
    a.h2d(e.tokens, ids); a.h2d(e.count, counts);
    a.decodeStepPaged(e.model, handle, e.tokens, T, e.count, window, sinks, commit ? 1 : 0, e.logits);
    if (commit) cache._advance(counts);
    return e;
  }

  /** Several tokens of every sequence of a PagedKVCache (tokens[s]: an array, empty for none): logits
   *  [sequences][T][vocabSize], T being the most tokens of a sequence, NaN for rows behind a sequence's tokens.
   *  opts.window: the tokens see the last so many positions alone, and the first opts.sinks; opts.commit false: they
   *  are stored, but do not count until cache.commit takes as many of them as stand. */
  forwardChunk(tokens, cache, opts = {}) {
    const e = this._chunk(tokens, cache, opts), T = Math.max.apply(null, Array.from(tokens, (t) => t.length));
    const out = new Float32Array(cache.sequences * T * this.cfg.vocabSize);
    hip().d2h(e.logits, out);
    if (e.rows * (2 * this.cfg.dim + this.cfg.hidden + this.cfg.vocabSize) * 4 > VECTORS_KEPT) this._dropPaged(cache);
    return out;
  }

  /** Queues one token of every sequence of a 4-bit cache (logits stay in device
   *  memory, `logits` of what it returns); a token outside the vocabulary leaves its sequence idle. */
  _stepAll(tokens, cache) {
    const c = this.cfg, a = hip();
    if (!this._w) throw new Error("Transformer.forward: call loadWeights first");
    if (!(cache instanceof KV4Cache)) throw new TypeError("Transformer.forwardAll: cache must be a KV4Cache");
    const handle = cache.handle;
    if (cache.nLayers !== c.nLayers || cache.nKvHeads !== c.nKvHeads || cache.dHead !== c.dHead)
      throw new RangeError("Transformer.forwardAll: cache shape does not match the Config");
    if (!tokens || tokens.length !== cache.sequences) throw new RangeError(`Transformer.forwardAll: ${cache.sequences} tokens expected`);
    const ids = Int32Array.from(tokens, (t) => (Number.isInteger(t) && t >= 0 && t < c.vocabSize ? t : -1));
    ids.forEach((t, s) => {
      if (t < 0) return;
      if (cache.lens[s] >= cache.maxSeq) throw new RangeError(`Transformer.forwardAll: sequence ${s} fills the cache (${cache.maxSeq})`);
      if (cache.nexts[s] >= c.maxSeq) throw new RangeError(`Transformer.forwardAll: sequence ${s} is at position ${cache.nexts[s]} of ${c.maxSeq}`);
    });
    const e = this._kv4For(cache);
    const step = () => a.decodeStepKv4(e.model, handle, e.tokens, e.logits);
    a.h2d(e.tokens, ids);
    if (this._graphOn && e.steps > 0 && !e.graph) {
      a.graphBegin();
      try {
        step();
        e.graph = a.graphEnd();
      } catch (err) {
        a.graphAbort();
        throw err;
      }
    }
    if (e.graph) a.graphLaunch(e.graph);
    else step();
    e.steps++;
    cache._advance(ids.map((t) => (t >= 0 ? 1 : 0)));
    return e;
  }

  /** One token of every sequence of a KV4Cache: logits [sequences][vocabSize] (NaN
   *  for idle sequences, whose token is outside the vocabulary). */
  forwardAll(tokens, cache) {
    const e = this._stepAll(tokens, cache);
    const out = new Float32Array(cache.sequences * this.cfg.vocabSize);
    hip().d2h(e.logits, out);
    return out;
  }

  /** One decode step: logits of `token` at position `pos`, K/V appended to `cache`. */
  forward(token, pos, cache) {
    if (cache instanceof KV4Cache) {
      if (cache.sequences !== 1) throw new TypeError("Transformer.forward: a cache of several sequences goes to forwardAll");
      if (pos !== cache.nexts[0]) throw new RangeError(`Transformer.forward: position ${pos}, the 4-bit cache is at ${cache.nexts[0]}`);
      hip().d2h(this._stepAll([token], cache).logits, this.logits);
      return this.logits;
    }
    if (cache instanceof PagedKVCache) {
      if (cache.sequences !== 1) throw new TypeError("Transformer.forward: a cache of several sequences goes to forwardChunk");
      if (pos !== cache.len) throw new RangeError(`Transformer.forward: position ${pos}, the cache is at ${cache.len}`);
      hip().d2h(this._chunk([[token]], cache).logits, this.logits);
      return this.logits;
    }
    this._step(token, pos, cache);
    hip().d2h(this._w.logits, this.logits);
    return this.logits;
  }

  /** Queues one decode step (logits stay in device memory, `_w.logits`). */
  _step(token, pos, cache) {
    const c = this.cfg, W = this._w, a = hip();
    if (!W) throw new Error("Transformer.forward: call loadWeights first");
    if (!(cache instanceof KVCache)) throw new TypeError("Transformer.forward: cache must be a device KVCache");
    if (!cache.kd) throw new Error("Transformer.forward: the cache has been freed");
    if (cache.nLayers !== c.nLayers || cache.kvDim !== c.kvDim) throw new RangeError("Transformer.forward: cache shape does not match the Config");
    if (!Number.isInteger(pos) || pos < 0 || pos >= Math.min(cache.maxSeq, c.maxSeq))
      throw new RangeError(`Transformer.forward: position ${pos} outside [0, ${Math.min(cache.maxSeq, c.maxSeq)})`);
    const model = this._modelFor(cache);
    W.stateHost[0] = Number.isInteger(token) && token >= 0 && token < c.vocabSize ? token : -1;
    W.stateHost[1] = pos;
    a.h2d(W.state, W.stateHost);
    let g = this._graphOn ? this._graphs.find((e) => e.cache === cache) : null;
    if (!this._graphOn) {
      a.decodeStep(model, cache.kd, cache.vd, W.state, W.logits);
    } else if (g && g.graph) {
      a.graphLaunch(g.graph);
    } else if (g) {
      a.graphBegin();
      try {
        a.decodeStep(model, cache.kd, cache.vd, W.state, W.logits);
        g.graph = a.graphEnd();
      } catch (e) {
        a.graphAbort();
        throw e;
      }
      a.graphLaunch(g.graph);
    } else {
      a.decodeStep(model, cache.kd, cache.vd, W.state, W.logits);
      this._graphs.push({ cache, graph: null });
      if (this._graphs.length > GRAPHS_KEPT) {
        const old = this._graphs.shift();
        if (old.graph) a.graphDestroy(old.graph);
      }
    }
    if (pos + 1 > cache.len) cache.len = pos + 1;
  }

  _dropGraphs() {
    const a = hip();
    for (const e of this._graphs) if (e.graph) a.graphDestroy(e.graph);
    this._graphs = [];
  }

  /** Frees the device weights, scratch and recorded graphs. */
  release() {
    if (!this._w) return;
    const a = hip();
    this._dropGraphs();
    this._dropKv4();
    this._dropPaged();
    for (const h of this._w.bufs) a.free(h);
    if (this._w.part) a.free(this._w.part);
    this._w = null; this._model = null;
  }
}
