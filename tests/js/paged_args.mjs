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

for (const o of out) console.log(JSON.stringify(o));
process.exit(out.every((o) => o.ok) ? 0 : 1);
