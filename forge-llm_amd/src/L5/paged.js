/**
 * L5 · A key-value cache in pages, for one or several sequences that share one pool
 * (fg_paged_*), the counterpart of forge-llm's PagedKVCache (src/L5/attention.js:157-187).
 * Several new tokens of a sequence may be stored and attended to before they are committed,
 * and fewer committed than were stored (drafted tokens that did not stand).
 *
 * `lens` holds each sequence's committed tokens; the device keeps its own, which every
 * call here moves alike.  Pages are handed out by `reserve` (which `append` and
 * Transformer.forwardChunk call) and come back with `truncate`, `forget` and `free`.
 */
import { hip } from "../L2/device.js";

const TYPES = { f32: 0, f16: 1 };

function whole(v, what, least) {
  if (!Number.isInteger(v) || v < least || v > 0x7FFFFFFF) throw new RangeError(`PagedKVCache: ${what} ${v}`);
  return v;
}
function rowsOf(x, n, what) {
  if (!x || x.length < n) throw new RangeError(`${what}: ${n} values expected, got ${x ? x.length : x}`);
  return x instanceof Float32Array ? x.subarray(0, n) : Float32Array.from(x.slice(0, n));
}

export class PagedKVCache {
  /** opts: sequences (1), pageSize (16: a power of two from 4 to 1024), maxPages of one sequence (all), type "f32" or "f16". */
  constructor(nLayers, pages, nKvHeads, dHead, opts = {}) {
    const pick = (k, d) => (opts[k] === undefined ? d : opts[k]);
    const sequences = pick("sequences", 1), pageSize = pick("pageSize", 16), maxPages = pick("maxPages", pages), type = pick("type", "f32");
    for (const [k, v] of [["nLayers", nLayers], ["pages", pages], ["nKvHeads", nKvHeads], ["dHead", dHead], ["sequences", sequences], ["maxPages", maxPages]])
      whole(v, k, 1);
    if (![32, 64, 96, 128, 256].includes(dHead)) throw new RangeError(`PagedKVCache: head size ${dHead} is not one of 32, 64, 96, 128, 256`);
    if (!Number.isInteger(pageSize) || pageSize < 4 || pageSize > 1024 || (pageSize & (pageSize - 1)) !== 0)
      throw new RangeError(`PagedKVCache: page size ${pageSize} is not a power of two from 4 to 1024`);
    if (maxPages * pageSize > 2 ** 30) throw new RangeError(`PagedKVCache: ${maxPages} pages of ${pageSize} slots a sequence are above 2^30`);
    if (!Object.prototype.hasOwnProperty.call(TYPES, type)) throw new RangeError(`PagedKVCache: type ${type} is neither f32 nor f16`);
    Object.assign(this, { nLayers, pages, nKvHeads, dHead, sequences, pageSize, maxPages, type, kvDim: nKvHeads * dHead, maxSeq: maxPages * pageSize });
    const a = hip(), bytes = this.bytes() / 2;
    this._bufs = [];
    const alloc = (n) => { const h = a.alloc(n); a.zero(h, n); this._bufs.push(h); return h; };
    try {
      const k = alloc(bytes), v = alloc(bytes);
      this._table = alloc(sequences * maxPages * 4); this._len = alloc(sequences * 4); this._count = alloc(sequences * 4);
      this._handle = a.pagedCache(nLayers, sequences, nKvHeads, dHead, pageSize, pages, maxPages, TYPES[type], k, v, this._table, this._len);
      this.table = new Int32Array(sequences * maxPages).fill(-1); this.lens = new Int32Array(sequences);
      this._least = new Int32Array(sequences);  // the shortest that truncate may leave, after forget
      this._free = Array.from({ length: pages }, (_, i) => pages - 1 - i);  // the next one last
      this._rope = null;
      a.h2d(this._table, this.table);
    } catch (e) {
      this.free();
      throw e;
    }
  }
  get len() { return this.lens[0]; }
  get freed() { return !this._bufs; }
  get freePages() { return this._free.length; }
  /** The device handle (throws once the cache has been freed). */
  get handle() {
    if (!this._bufs) throw new Error("PagedKVCache: the cache has been freed");
    return this._handle;
  }
  bytes() { return 2 * this.nLayers * this.pages * this.nKvHeads * this.pageSize * this.dHead * (this.type === "f32" ? 4 : 2); }
  _layer(layer) {
    if (!Number.isInteger(layer) || layer < 0 || layer >= this.nLayers) throw new RangeError(`PagedKVCache: layer ${layer} out of range`);
  }
  _seq(seq) {
    if (!Number.isInteger(seq) || seq < 0 || seq >= this.sequences) throw new RangeError(`PagedKVCache: sequence ${seq} out of range`);
  }
  // New tokens of every sequence, T at most: a number for all of them, or one each.
  _counts(counts, T) {
    if (counts === undefined || counts === null) return new Int32Array(this.sequences).fill(T);
    if (counts.length !== this.sequences) throw new RangeError(`PagedKVCache: ${this.sequences} numbers of tokens expected`);
    for (const n of counts) if (!Number.isInteger(n) || n < 0 || n > T) throw new RangeError(`PagedKVCache: ${n} tokens of ${T}`);
    return Int32Array.from(counts);
  }
  /** Gives every sequence the pages of `counts` more tokens (a number, or one each); throws, and changes nothing, where there are none left. */
  reserve(counts) {
    this.handle;
    counts = counts && counts.length !== undefined ? this._counts(counts, 0x7FFFFFFF) : new Int32Array(this.sequences).fill(whole(counts, "tokens", 0));
    const want = [];
    counts.forEach((n, s) => {
      const end = this.lens[s] + n;
      if (end > this.maxSeq) throw new RangeError(`PagedKVCache: ${this.lens[s]} + ${n} tokens of sequence ${s} exceed ${this.maxSeq}`);
      for (let p = Math.floor(this.lens[s] / this.pageSize); p * this.pageSize < end; p++)
        if (this.table[s * this.maxPages + p] < 0) want.push(s * this.maxPages + p);
    });
    if (want.length > this._free.length) throw new RangeError(`PagedKVCache: ${want.length} pages wanted, ${this._free.length} of ${this.pages} left`);
    if (want.length === 0) return;
    for (const at of want) this.table[at] = this._free.pop();
    hip().h2d(this._table, this.table);
  }
  _giveBack(which) {  // which(s, p): page p of sequence s
    let some = false;
    for (let s = 0; s < this.sequences; s++)
      for (let p = 0; p < this.maxPages; p++) {
        const at = s * this.maxPages + p;
        if (this.table[at] >= 0 && which(s, p)) { this._free.push(this.table[at]); this.table[at] = -1; some = true; }
      }
    if (some) hip().h2d(this._table, this.table);
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
  // cos and sin of the positions below npos, on the device (theta, dims as in ropeRows).
  _angles(theta, dims, npos) {
    const a = hip(), r = this._rope;
    if (r && r.theta === theta && r.dims === dims && r.npos >= npos) return r;
    const n = Math.max(npos, Math.min(this.maxSeq, 2 * npos)), size = n * dims / 2;
    const cos = new Float64Array(size), sin = new Float64Array(size);
    a.ropeTable(cos, sin, n, dims, theta);
    if (r) { a.free(r.cos); a.free(r.sin); this._rope = null; }
    const c = a.alloc(cos.byteLength);
    let s;
    try {
      s = a.alloc(sin.byteLength);
    } catch (e) {
      a.free(c);
      throw e;
    }
    a.h2d(c, cos); a.h2d(s, sin);
    this._rope = { theta, dims, npos: n, cos: c, sin: s };
    return this._rope;
  }
  /**
   * Stores up to T tokens of every sequence in a layer: rows [sequences][T][kvDim] of k and v (opts.counts: how many of
   * each).  With opts.rope = {theta, dims, half} the first `dims` values (dHead) of every head turn by their
   * positions' angles, pairs being neighbours or, with `half`, dims / 2 apart, and opts.q, rows
   * [sequences][T][nHeads][dHead] (opts.nHeads), comes back turned.
   */
  append(layer, k, v, T = 1, opts = {}) {
    this._layer(layer); whole(T, "tokens", 0);
    const counts = this._counts(opts.counts, T), rows = this.sequences * T, n = rows * this.kvDim, h = this.handle;
    const kh = rowsOf(k, n, "PagedKVCache.append k"), vh = rowsOf(v, n, "PagedKVCache.append v"), { rope, q } = opts;
    const nHeads = q ? whole(opts.nHeads, "query heads", 1) : 0, nq = rows * nHeads * this.dHead;
    const qh = q ? rowsOf(q, nq, "PagedKVCache.append q") : null, out = q ? new Float32Array(nq) : undefined;
    let dims = 0, angles = null;
    if (rope) {
      dims = rope.dims === undefined ? this.dHead : rope.dims;
      if (!Number.isInteger(dims) || dims <= 0 || dims > this.dHead || dims % 2) throw new RangeError(`PagedKVCache.append: ${dims} rotated values of ${this.dHead}`);
      if (!(rope.theta > 0)) throw new RangeError(`PagedKVCache.append: theta ${rope.theta}`);
    }
    if (rows === 0) return out;
    this.reserve(counts);
    if (rope) angles = this._angles(rope.theta, dims, Math.max.apply(null, Array.from(this.lens, (l, s) => l + counts[s])) || 1);
    // one row stride for all three: queries apart go in with rows of their own width
    const wide = Math.max(this.kvDim, nHeads * this.dHead);
    const spread = (x, w) => {
      if (w === wide) return x;
      const y = new Float32Array(rows * wide);
      for (let r = 0; r < rows; r++) y.set(x.subarray(r * w, (r + 1) * w), r * wide);
      return y;
    };
    this._withBuffers([rows * wide, rows * wide, q ? rows * wide : 0, nq], (a, [bk, bv, bq, bo]) => {
      a.h2d(bk, spread(kh, this.kvDim)); a.h2d(bv, spread(vh, this.kvDim)); a.h2d(this._count, counts);
      if (q) { a.h2d(bq, spread(qh, nHeads * this.dHead)); a.zero(bo, nq * 4); }
      a.pagedAppend(h, layer, q ? bo : null, q ? bq : null, bk, bv, wide, nHeads, T, this._count, angles ? angles.cos : null,
                    angles ? angles.sin : null, angles ? angles.npos : 0, dims, rope && rope.half ? 1 : 0);
      if (q) a.d2h(bo, out);
    });
    return out;
  }
  /** Causal attention of T stored, not yet committed tokens a sequence (opts.counts) over the cache: q
   *  [sequences][T][nHeads][dHead], the same shape returned, zeros for rows behind a sequence's tokens.
   *  opts.window: the last so many slots alone, and the first opts.sinks. */
  attend(layer, q, nHeads, T = 1, opts = {}) {
    this._layer(layer); whole(T, "tokens", 0);
    if (!Number.isInteger(nHeads) || nHeads <= 0 || nHeads % this.nKvHeads !== 0)
      throw new RangeError(`PagedKVCache.attend: ${nHeads} query heads for ${this.nKvHeads} kv heads`);
    const window = opts.window === undefined ? 0 : whole(opts.window, "window", 0), sinks = opts.sinks === undefined ? 0 : whole(opts.sinks, "sinks", 0);
    const scale = opts.scale === undefined ? 1 / Math.sqrt(this.dHead) : opts.scale;
    if (typeof scale !== "number") throw new TypeError(`PagedKVCache.attend: scale ${scale}`);
    const counts = this._counts(opts.counts, T), n = this.sequences * T * nHeads * this.dHead, h = this.handle;
    const qh = rowsOf(q, n, "PagedKVCache.attend q"), out = new Float32Array(n);
    if (n === 0) return out;
    this._withBuffers([n, n], (a, [bq, bo]) => {
      a.h2d(bq, qh); a.h2d(this._count, counts); a.zero(bo, n * 4);
      a.pagedAttn(h, layer, bo, bq, nHeads, scale, T, this._count, window, sinks);
      a.d2h(bo, out);
    });
    return out;
  }
  /** Ends a step: T more tokens of every sequence count, or counts[s] of each. */
  commit(counts = 1) {
    const each = counts && counts.length !== undefined;
    const T = each ? Math.max.apply(null, [0].concat(Array.from(counts))) : whole(counts, "tokens", 0), n = this._counts(each ? counts : null, T);
    n.forEach((m, s) => { if (this.lens[s] + m > this.maxSeq) throw new RangeError(`PagedKVCache: ${this.lens[s]} + ${m} tokens exceed ${this.maxSeq}`); });
    const h = this.handle, a = hip();
    a.h2d(this._count, n);
    a.pagedCommit(h, T, this._count);
    this._advance(n);
  }
  _advance(counts) { for (let s = 0; s < this.sequences; s++) this.lens[s] += counts[s]; }
  /** Keeps the first `length` tokens of a sequence; the pages behind them come back.  After `forget`, a length whose
   *  window reaches back to what was forgotten throws (0, a new start, does not). */
  truncate(seq, length) {
    this._seq(seq);
    if (!Number.isInteger(length) || length < 0 || length > this.lens[seq]) throw new RangeError(`PagedKVCache.truncate: ${length} of ${this.lens[seq]} tokens`);
    if (length > 0 && length < this._least[seq])
      throw new RangeError(`PagedKVCache.truncate: ${length} tokens, of which the window needs forgotten ones (${this._least[seq]} at least, or 0)`);
    this.handle;
    this.lens[seq] = length;
    if (length === 0) this._least[seq] = 0;
    hip().h2d(this._len, this.lens);
    this._giveBack((s, p) => s === seq && p * this.pageSize >= length);
  }
  /** Takes back the pages that a window of the last `window` tokens and the first `sinks` leaves unseen for good. */
  forget(window, sinks = 0) {
    whole(window, "window", 1); whole(sinks, "sinks", 0);
    this.handle;
    this._giveBack((s, p) => {
      const end = (p + 1) * this.pageSize, unseen = p * this.pageSize >= sinks && end <= this.lens[s] + 1 - window;
      if (unseen) this._least[s] = Math.max(this._least[s], end - 1 + window);
      return unseen;
    });
  }
  _view(layer, upto, seq, which) {
    this._layer(layer); this._seq(seq);
    if (!Number.isInteger(upto) || upto < 0 || upto > this.maxSeq) throw new RangeError(`PagedKVCache: ${upto} positions`);
    const n = upto * this.kvDim, out = new Float32Array(n), h = this.handle;
    if (n === 0) return out;
    this._withBuffers([this.sequences * n, this.sequences * n], (a, bufs) => {
      a.pagedRead(h, layer, bufs[0], bufs[1], this.kvDim, 0, upto);
      a.d2h(bufs[which], out, seq * n * 4);
    });
    return out;
  }
  /** The values of the first `upto` slots of a sequence, rows of kvDim (zeros where it has no page). */
  kView(layer, upto, seq = 0) { return this._view(layer, upto, seq, 0); }
  vView(layer, upto, seq = 0) { return this._view(layer, upto, seq, 1); }
  /** Frees the device arrays (the cache is unusable afterwards). */
  free() {
    const a = hip();
    if (this._rope) { a.free(this._rope.cos); a.free(this._rope.sin); this._rope = null; }
    if (this._bufs) { for (const h of this._bufs) a.free(h); this._bufs = null; this._handle = null; }
  }
}
