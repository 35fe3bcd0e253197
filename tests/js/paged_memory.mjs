// Device memory that steps over a paged cache hold when they are done.  Prints one JSON line per case.
import { Config, Transformer, PagedKVCache, initWeights, hip } from "../../forge-llm_amd/src/index.js";

const cfg = new Config({ dim: 64, hidden: 96, nLayers: 1, nHeads: 2, nKvHeads: 1, vocabSize: 40000, maxSeq: 1024, normEps: 1e-5 });
const w = initWeights(cfg, 3), t = { tok_emb: w.tok_emb, ln_f: w.ln_f, wcls: null, "layer.0": w["layer.0"] };
const ids = Array.from({ length: 600 }, (_, i) => (i * 7919) % cfg.vocabSize);
const same = (x, y) => x.length === y.length && x.every((v, i) => Object.is(v, y[i]));
const M = new Transformer(cfg).loadWeights(t), V = cfg.vocabSize, used = () => hip().memStats()[0];
const a = new PagedKVCache(1, 64, 1, 32), b = new PagedKVCache(1, 64, 1, 32);

const before = used();
const all = M.forwardChunk([ids], a), held = used() - before;
const next = Float32Array.from(M.forward(5, 600, a));
for (let at = 0; at < 600; at += 50) M.forwardChunk([ids.slice(at, at + 50)], b);
const small = used() - before;
const ok = {
  "a chunk's vectors go back": held < (64 << 20) && all.length === 600 * V,
  "the next step goes on": same(next, M.forward(5, 600, b)),
  "small ones are kept": small > 50 * V * 4 && small < 2 * (64 << 20),
};
a.free(); b.free(); M.release();
for (const [test, r] of Object.entries(ok)) console.log(JSON.stringify({ test, ok: r, held, small }));
process.exit(Object.values(ok).every((x) => x) ? 0 : 1);
