/**
 * L5 · KV cache of the inference forward, resident in device memory.
 *
 * Same interface as forge-llm's contiguous KVCache (src/L5/attention.js:
 * 128-156): nLayers × maxSeq × kvDim keys and values, `put`, `kView`/`vView`,
 * `sliceK`/`sliceV`, `reset`, `bytes`, `len`.  The arrays live in HBM, where
 * Transformer.forward's kernels write each position's K and V; `k` / `v` and
 * the views download a copy on access (writing into that copy does not
 * change the cache — use `put`).  The reference's single-row attention
 * helpers over host arrays (attentionDecode, attentionNaive, flashAttention)
 * are kept with their signatures and compute on the device; the model's own
 * decode attention runs inside Transformer.forward.
 */
import { hip } from "../L2/device.js";

export class KVCache {
  constructor(nLayers, maxSeq, kvDim) {
    for (const [k, v] of [["nLayers", nLayers], ["maxSeq", maxSeq], ["kvDim", kvDim]])
      if (!Number.isInteger(v) || v <= 0) throw new RangeError(`KVCache: ${k} must be a positive integer, got ${v}`);
    this.nLayers = nLayers; this.maxSeq = maxSeq; this.kvDim = kvDim;
    const a = hip();
    const bytes = nLayers * maxSeq * kvDim * 4;
    this.kd = a.alloc(bytes); this.vd = a.alloc(bytes);
    a.zero(this.kd, bytes); a.zero(this.vd, bytes);
    this.len = 0;
  }
  _off(layer, pos) {
    if (!Number.isInteger(layer) || layer < 0 || layer >= this.nLayers) throw new RangeError(`KVCache: layer ${layer} out of range`);
    if (!Number.isInteger(pos) || pos < 0 || pos > this.maxSeq) throw new RangeError(`KVCache: position ${pos} out of range`);
    return (layer * this.maxSeq + pos) * this.kvDim;
  }
  _read(h, off, n) {
    const out = new Float32Array(n);
    if (n > 0) hip().d2h(h, out, off * 4);
    return out;
  }
  put(layer, pos, k, v) {
    const o = this._off(layer, pos);
    if (pos >= this.maxSeq) throw new RangeError(`KVCache: position ${pos} out of range`);
    const a = hip();
    a.h2d(this.kd, Float32Array.from(k.subarray ? k.subarray(0, this.kvDim) : k.slice(0, this.kvDim)), o * 4);
    a.h2d(this.vd, Float32Array.from(v.subarray ? v.subarray(0, this.kvDim) : v.slice(0, this.kvDim)), o * 4);
    if (pos + 1 > this.len) this.len = pos + 1;
  }
  get k() { return this._read(this.kd, 0, this.nLayers * this.maxSeq * this.kvDim); }
  get v() { return this._read(this.vd, 0, this.nLayers * this.maxSeq * this.kvDim); }
  kView(layer, upto) { return this._read(this.kd, this._off(layer, 0), upto * this.kvDim); }
  vView(layer, upto) { return this._read(this.vd, this._off(layer, 0), upto * this.kvDim); }
  sliceK(layer, pos) { return this._read(this.kd, this._off(layer, pos), this.kvDim); }
  sliceV(layer, pos) { return this._read(this.vd, this._off(layer, pos), this.kvDim); }
  reset() { this.len = 0; }
  bytes() { return 2 * this.nLayers * this.maxSeq * this.kvDim * 4; }
  /** Frees the device arrays (the cache is unusable afterwards). */
  free() {
    const a = hip();
    if (this.kd) { a.free(this.kd); a.free(this.vd); this.kd = null; this.vd = null; }
  }
}

/** What KV4Cache.evict takes: whole numbers of 32 bits, which the device's call holds. */
export function checkEviction(budget, recent) {
  if (!Number.isInteger(budget) || budget < 1 || budget > 0x7FFFFFFF) throw new RangeError(`KV4Cache.evict: budget ${budget}`);
  if (!Number.isInteger(recent) || recent < 0 || recent > budget) throw new RangeError(`KV4Cache.evict: recent ${recent} outside [0, ${budget}]`);
}

/**
 * A KV cache in 4-bit blocks (Q4_0: 32 values on one fp16 step, 4.5 bits a
 * value), for one or several sequences: 7.1 times the context of KVCache in the
 * same memory.  No counterpart in forge-llm.  `Transformer.forward` takes it for
 * one sequence, `forwardAll` for several.  With `trackWeights` every cached token's
 * attention is added up, and `evict(budget, recent)` keeps, head by head, the
 * newest `recent` tokens and those of most attention; evicted caches run on past
 * maxSeq.  `reorder(parents)` lets the sequences go on from one another (beam
 * search).  Head sizes 32, 64, 96, 128 and 256.
 *
 * `lens` / `nexts` hold each sequence's cached tokens and the position of its next;
 * the device keeps its own, which every call here moves alike.
 */
export class KV4Cache {
  constructor(nLayers, maxSeq, nKvHeads, dHead, opts = {}) {
    const sequences = opts.sequences === undefined ? 1 : opts.sequences;
    for (const [k, v] of [["nLayers", nLayers], ["maxSeq", maxSeq], ["nKvHeads", nKvHeads], ["dHead", dHead], ["sequences", sequences]])
      if (!Number.isInteger(v) || v <= 0) throw new RangeError(`KV4Cache: ${k} must be a positive integer, got ${v}`);
    if (![32, 64, 96, 128, 256].includes(dHead))
      throw new RangeError(`KV4Cache: head size ${dHead} is not one of 32, 64, 96, 128, 256`);
    Object.assign(this, { nLayers, maxSeq, nKvHeads, dHead, sequences, kvDim: nKvHeads * dHead, trackWeights: !!opts.trackWeights });
    const a = hip(), slots = nLayers * sequences * nKvHeads * maxSeq;
    this._bufs = [];
    const alloc = (bytes) => { const h = a.alloc(bytes); a.zero(h, bytes); this._bufs.push(h); return h; };
    const [k, v] = [alloc(slots * dHead / 2), alloc(slots * dHead / 2)];
    const [kd, vd] = [alloc(slots * dHead / 16), alloc(slots * dHead / 16)];
    this._len = alloc(sequences * 4); this._next = alloc(sequences * 4);
    this._weight = this.trackWeights ? alloc(slots * 4) : null;
    this._pos = this.trackWeights ? alloc(slots * 4) : null;
    this._handle = a.kv4Cache(nLayers, sequences, nKvHeads, dHead, maxSeq, k, v, kd, vd, this._len, this._next, this._weight, this._pos);
    this.lens = new Int32Array(sequences); this.nexts = new Int32Array(sequences);
  }
  get len() { return this.lens[0]; }
  get freed() { return !this._bufs; }
  /** The device handle (throws once the cache has been freed). */
  get handle() {
    if (!this._bufs) throw new Error("KV4Cache: the cache has been freed");
    return this._handle;
  }
  _layer(layer) {
    if (!Number.isInteger(layer) || layer < 0 || layer >= this.nLayers) throw new RangeError(`KV4Cache: layer ${layer} out of range`);
  }
  _room(T) {
    if (!Number.isInteger(T) || T < 0) throw new RangeError(`KV4Cache: ${T} tokens`);
    for (const n of this.lens) if (n + T > this.maxSeq) throw new RangeError(`KV4Cache: ${n} + ${T} tokens exceed ${this.maxSeq}`);
  }
  _withBuffers(sizes, fn) {
    const a = hip(), held = [];
    try {
      for (const n of sizes) held.push(a.alloc(Math.max(1, n) * 4));
      return fn(a, held);
    } finally {
      for (const h of held) a.free(h);
    }
  }
  /** Stores T tokens of every sequence in a layer: rows [sequences][T][kvDim] of k and v. */
  append(layer, k, v, T = 1) {
    this._layer(layer); this._room(T);
    const n = this.sequences * T * this.kvDim, h = this.handle;
    const kh = f32Slice(k, 0, n, "KV4Cache.append k"), vh = f32Slice(v, 0, n, "KV4Cache.append v");
    if (n === 0) return;
    this._withBuffers([n, n], (a, [bk, bv]) => {
      a.h2d(bk, kh); a.h2d(bv, vh);
      a.kv4Append(h, layer, bk, bv, this.kvDim, T, null);
    });
  }
  /** Attention of one query token a sequence over the cached tokens and T not yet
   *  committed ones: q [sequences][nHeads][dHead], the same shape returned. */
  attend(layer, q, nHeads, T = 0, scale = 1 / Math.sqrt(this.dHead)) {
    this._layer(layer); this._room(T);
    if (!Number.isInteger(nHeads) || nHeads <= 0 || nHeads % this.nKvHeads !== 0)
      throw new RangeError(`KV4Cache.attend: ${nHeads} query heads for ${this.nKvHeads} kv heads`);
    if (typeof scale !== "number") throw new TypeError(`KV4Cache.attend: scale ${scale}`);
    const n = this.sequences * nHeads * this.dHead, h = this.handle;
    const qh = f32Slice(q, 0, n, "KV4Cache.attend q"), out = new Float32Array(n);
    this._withBuffers([n, n], (a, [bq, bo]) => {
      a.h2d(bq, qh);
      a.kv4Attn(h, layer, bo, bq, nHeads, scale, T, null);
      a.d2h(bo, out);
    });
    return out;
  }
  /** Ends a step of T tokens a sequence. */
  commit(T = 1) {
    this._room(T);
    hip().kv4Commit(this.handle, T, null);
    this._advance(this.lens.map(() => T));
  }
  _advance(counts) {
    for (let s = 0; s < this.sequences; s++) { this.lens[s] += counts[s]; this.nexts[s] += counts[s]; }
  }
  /** Keeps `budget` tokens of every head of the sequences that have more: the
   *  newest `recent` and those of most accumulated attention. */
  evict(budget, recent = 0) {
    if (!this.trackWeights) throw new Error("KV4Cache.evict: the cache was made without trackWeights");
    checkEviction(budget, recent);
    hip().kv4Evict(this.handle, budget, recent);
    for (let s = 0; s < this.sequences; s++) this.lens[s] = Math.min(this.lens[s], budget);
  }
  /** Sequence i goes on from what sequence parents[i] of its group holds (groups of
   *  `width` sequences, parents counted inside each). */
  reorder(parents, width = this.sequences) {
    if (!parents || parents.length !== this.sequences) throw new RangeError(`KV4Cache.reorder: ${this.sequences} parents expected`);
    if (!Number.isInteger(width) || width <= 0 || this.sequences % width !== 0) throw new RangeError(`KV4Cache.reorder: groups of ${width}`);
    for (const p of parents) if (!Number.isInteger(p) || p < 0 || p >= width) throw new RangeError(`KV4Cache.reorder: parent ${p} outside [0, ${width})`);
    const h = this.handle;
    this._withBuffers([this.sequences], (a, [bp]) => {
      a.h2d(bp, Int32Array.from(parents));
      a.kv4Reorder(h, bp, width);
    });
    this._follow(parents, width);
  }
  _follow(parents, width) {
    const from = (s) => s - s % width + parents[s];
    const [l, n] = [this.lens.slice(), this.nexts.slice()];
    for (let s = 0; s < this.sequences; s++) { this.lens[s] = l[from(s)]; this.nexts[s] = n[from(s)]; }
  }
  _view(layer, upto, seq, which) {
    this._layer(layer);
    if (!Number.isInteger(upto) || upto < 0 || upto > this.maxSeq) throw new RangeError(`KV4Cache: ${upto} positions`);
    if (!Number.isInteger(seq) || seq < 0 || seq >= this.sequences) throw new RangeError(`KV4Cache: sequence ${seq} out of range`);
    const n = upto * this.kvDim, out = new Float32Array(n), h = this.handle;
    if (n === 0) return out;
    this._withBuffers([this.sequences * n, this.sequences * n], (a, bufs) => {
      a.kv4Read(h, layer, bufs[0], bufs[1], this.kvDim, 0, upto);
      a.d2h(bufs[which], out, seq * n * 4);
    });
    return out;
  }
  /** The values that the first `upto` slots of a sequence stand for, rows of kvDim. */
  kView(layer, upto, seq = 0) { return this._view(layer, upto, seq, 0); }
  vView(layer, upto, seq = 0) { return this._view(layer, upto, seq, 1); }
  _perSlot(buf, Type, layer, seq, head) {
    this._layer(layer);
    if (!buf) throw new Error("KV4Cache: the cache was made without trackWeights");
    if (!Number.isInteger(seq) || seq < 0 || seq >= this.sequences || !Number.isInteger(head) || head < 0 || head >= this.nKvHeads)
      throw new RangeError(`KV4Cache: sequence ${seq}, head ${head}`);
    const out = new Type(this.lens[seq]);
    this.handle;
    if (out.length) hip().d2h(buf, out, (((layer * this.sequences + seq) * this.nKvHeads + head) * this.maxSeq) * 4);
    return out;
  }
  /** Accumulated attention, and position, of a head's cached tokens, slot by slot. */
  weights(layer, seq = 0, head = 0) { return this._perSlot(this._weight, Float32Array, layer, seq, head); }
  positions(layer, seq = 0, head = 0) { return this._perSlot(this._pos, Int32Array, layer, seq, head); }
  reset() {
    const a = hip();
    this.handle;
    a.zero(this._len, this.sequences * 4); a.zero(this._next, this.sequences * 4);
    this.lens.fill(0); this.nexts.fill(0);
  }
  bytes() {
    const slots = this.nLayers * this.sequences * this.nKvHeads * this.maxSeq;
    return slots * (this.dHead + this.dHead / 8) + (this.trackWeights ? slots * 8 : 0);
  }
  /** Frees the device arrays (the cache is unusable afterwards). */
  free() {
    const a = hip();
    if (this._bufs) { for (const h of this._bufs) a.free(h); this._bufs = null; this._handle = null; }
  }
}

// ── single-query-row attention over host arrays (attention.js:31-126) ──
// out[0..d) = Σ_j softmax_j(scale · q·K_j) V_j over keys j < n (rows of d
// floats at K[kOff + j d], V[kOff + j d]); with causal, keys j > qOff are
// masked.  The operands are copied to the device, fg_row_attention computes
// the row there with the variant's own order of operations (mode 0: the
// two-pass decode loop, 1: softmax then Σ p V, 2: blocks of `block` keys with
// the online rescale), and the d results are written into `out`.
function f32Slice(x, off, len, what) {
  if (len === 0) return new Float32Array(0);
  if (!x || typeof x.length !== "number" || x.length < off + len)
    throw new RangeError(`${what}: needs ${off + len} elements, has ${x ? x.length : 0}`);
  if (x instanceof Float32Array) return x.subarray(off, off + len);
  return Float32Array.from(Array.prototype.slice.call(x, off, off + len));
}

function rowAttention(name, mode, out, q, K, V, n, d, scale, causal, qOff, kOff, block, scores) {
  if (!Number.isInteger(n) || n < 0) throw new RangeError(`${name}: n must be a non-negative integer, got ${n}`);
  if (!Number.isInteger(d) || d <= 0) throw new RangeError(`${name}: d must be a positive integer, got ${d}`);
  if (!Number.isInteger(qOff)) throw new RangeError(`${name}: qOff must be an integer, got ${qOff}`);
  if (!Number.isInteger(kOff) || kOff < 0) throw new RangeError(`${name}: kOff must be a non-negative integer, got ${kOff}`);
  if (!Number.isInteger(block) || block <= 0) throw new RangeError(`${name}: block must be a positive integer, got ${block}`);
  if (typeof scale !== "number") throw new TypeError(`${name}: scale must be a number`);
  if (!out || out.length < d) throw new RangeError(`${name}: out needs ${d} elements`);
  const qh = f32Slice(q, 0, d, `${name} q`);
  const kh = f32Slice(K, kOff, n * d, `${name} K`);
  const vh = f32Slice(V, kOff, n * d, `${name} V`);
  const a = hip();
  const held = [];
  const alloc = (bytes) => { const h = a.alloc(bytes); held.push(h); return h; };
  try {
    const bq = alloc(d * 4), bk = alloc(Math.max(1, n * d) * 4), bv = alloc(Math.max(1, n * d) * 4);
    const bo = alloc(d * 4);
    const bs = scores ? alloc(Math.max(1, n) * 4) : null;
    a.h2d(bq, qh);
    if (n > 0) { a.h2d(bk, kh); a.h2d(bv, vh); }
    a.rowAttention(bo, bq, bk, bv, n, d, scale, causal ? 1 : 0, qOff, mode, block, bs);
    const r = new Float32Array(d);
    a.d2h(bo, r);
    for (let i = 0; i < d; i++) out[i] = r[i];
    if (scores && n > 0) {
      const sc = new Float32Array(n);
      a.d2h(bs, sc);
      for (let j = 0; j < n; j++) scores[j] = sc[j];
    }
  } finally {
    for (const h of held) a.free(h);
  }
  return out;
}

/** Two-pass single-row attention (attention.js:31-57); `s` (length >= n),
 *  when given, receives the scores as the reference leaves them. */
export function attentionDecode(out, q, K, V, n, d, scale, causal = true, qOff = 0, kOff = 0, s = null) {
  return rowAttention("attentionDecode", 0, out, q, K, V, n, d, scale, causal, qOff, kOff, 1,
                      s && s.length >= n ? s : null);
}
/** Reference single-row attention: softmax of the scores, then Σ p V (attention.js:63-79). */
export function attentionNaive(out, q, K, V, n, d, scale, causal = true, qOff = 0, kOff = 0) {
  return rowAttention("attentionNaive", 1, out, q, K, V, n, d, scale, causal, qOff, kOff, 1, null);
}
/** Online-softmax single-row attention over blocks of `block` keys (attention.js:89-126). */
export function flashAttention(out, q, K, V, n, d, scale, causal = true, qOff = 0, kOff = 0, block = 64) {
  return rowAttention("flashAttention", 2, out, q, K, V, n, d, scale, causal, qOff, kOff, block, null);
}
