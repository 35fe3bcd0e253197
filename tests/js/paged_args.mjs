// Arguments of the paged cache and of verifyDrafts that are refused.  Prints one JSON line per case.
import { PagedKVCache, verifyDrafts } from "../../forge-llm_amd/src/index.js";

const out = [];
const rec = (test, fn) => { try { out.push({ test, ok: fn() }); } catch (e) { out.push({ test, ok: false, error: String(e && e.stack || e) }); } };
const refused = (fns) => fns.every((f) => { try { f(); return false; } catch (e) { return e instanceof RangeError; } });

rec("reserve: a number for every sequence, whole and not below zero", () => {
  const c = new PagedKVCache(1, 4, 1, 32, { sequences: 2, pageSize: 4 });
  let ok = refused([() => c.reserve([1]), () => c.reserve([1, 1, 9]), () => c.reserve([1.5, 0]), () => c.reserve([-1, 1]), () => c.reserve([NaN, 1]),
                    () => c.reserve([]), () => c.reserve("12"), () => c.reserve(undefined), () => c.reserve(0.5)]);
  ok = ok && c.freePages === 4;
  c.reserve([5, 1]);
  ok = ok && c.freePages === 1;
  c.reserve(Int32Array.of(0, 4));
  ok = ok && c.freePages === 1;
  c.free();
  return ok;
});

rec("verifyDrafts: drafts and their numbers are whole and fit 32 bits", () => {
  const p = [0.5, 0.25, 0.25, 0.1, 0.1, 0.8].map(Math.log), go = (d, n) => verifyDrafts(p, [[d]], [0, 0.5], { vocab: 3, drafted: n });
  return refused([2 ** 32 + 1, 0.5, NaN, "1", undefined].map((d) => () => go(d, null)).concat([[2 ** 32], [0.5], [NaN]].map((n) => () => go(0, n)))) &&
    go(0, [1]).counts[0] === 2 && go(-1, null).counts[0] === 1 && go(2 ** 31 - 1, null).counts[0] === 1 && go(0, Int32Array.of(-1, 7)).counts[0] === 0;
});

for (const o of out) console.log(JSON.stringify(o));
process.exit(out.every((o) => o.ok) ? 0 : 1);
