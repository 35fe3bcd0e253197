"""The serving cache in four bits and what goes with it, as timed cases.

store    keys and values of new tokens into a 4-bit cache (Q4_0 blocks of 32 values), and back as the values they stand for
attend   one token's attention over that cache, for a batch of sequences of their own lengths, with or without the
         accumulated weight of every cached token
budget   one step of a generation whose cache is bounded: store a token, attend, and evict the token of least weight
evict    the choice of what a bounded cache keeps, by accumulated weight, for all layers and heads at once
select   a beam search's next beams over beams and vocabulary
reorder  the beams' cached states following their parents, in place

Tensors are torch's; the library works on a stream of its own.  The cache's layout is that of fg_kv4_cache:
codes [layer][sequence][kv head][slot][dH / 2], steps fp16 [layer][sequence][kv head][slot][dH / 32]; with nb = dH / 32,
byte n nb + b of a slot's codes (n < 16, b < nb) holds values 32 b + n (low four bits) and 32 b + 16 + n (high four).
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

BLOCK = 32


def listed():
    return [
        # one new token of four short conversations of the small decode model: launches and latency
        {"name": "store-token", "kind": "store", "seqs": 4, "T": 1, "nKV": 4, "dH": 32, "cap": 256},
        # the prompts of a batch, heads of Llama-3-8B
        {"name": "store-8b", "kind": "store", "seqs": 4, "T": 4096, "nKV": 8, "dH": 128, "cap": 4096},
        # a token of the small decode benchmark's model at position 200
        {"name": "attend-small", "kind": "attend", "seqs": 1, "nH": 8, "nKV": 4, "dH": 32, "cap": 512, "len": 201, "weights": False},
        # a batch of conversations of the 125M model, weights kept for eviction
        {"name": "attend-125m", "kind": "attend", "seqs": 8, "nH": 12, "nKV": 12, "dH": 64, "cap": 1024, "len": 1023, "weights": True},
        # one long document, heads of Llama-3-8B
        {"name": "attend-8b-long", "kind": "attend", "seqs": 1, "nH": 32, "nKV": 8, "dH": 128, "cap": 131072, "len": 130001, "weights": False},
        # a serving batch of sequences of all lengths, one slot of it empty
        {"name": "attend-8b-batch", "kind": "attend", "seqs": 32, "nH": 32, "nKV": 8, "dH": 128, "cap": 8192, "len": 8192, "weights": False},
        # a token of a generation held to 2048 cached tokens
        {"name": "budget-8b", "kind": "budget", "seqs": 1, "nH": 32, "nKV": 8, "dH": 128, "budget": 2048, "T": 1, "recent": 256},
        # what remains of 16384 cached tokens in 4096 slots, 32 layers of 8 heads
        {"name": "evict-8b", "kind": "evict", "layers": 32, "seqs": 1, "nKV": 8, "cap": 16384, "len": 16384, "budget": 4096, "recent": 512},
        # four beams of the small decode model
        {"name": "select-small", "kind": "select", "reqs": 1, "W": 4, "V": 4096},
        # eight requests of eight beams over Llama-3-8B's vocabulary
        {"name": "select-8b", "kind": "select", "reqs": 8, "W": 8, "V": 128256},
        # four beams of the small decode model, f32 states
        {"name": "reorder-small", "kind": "reorder", "layers": 4, "reqs": 1, "W": 4, "kvD": 128, "cap": 512, "len": 200},
        # eight beams of the 125M model, f32 states
        {"name": "reorder-125m", "kind": "reorder", "layers": 12, "reqs": 1, "W": 8, "kvD": 768, "cap": 1024, "len": 1000},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "budget", "evict", "select", "select", "reorder"])
    dH, nKV = rng.choice([32, 64, 64, 96, 128, 128, 256]), rng.choice([1, 2, 3, 4, 5, 8, 12])
    if kind == "store":
        while True:
            c = {"kind": kind, "seqs": _log(rng, 1, 16), "T": _log(rng, 1, 4096), "nKV": nKV, "dH": dH, "cap": 0}
            c["cap"] = c["T"] + rng.randint(0, 300)
            if c["seqs"] * c["T"] * nKV * dH <= 16e6:
                return c
    if kind == "attend":
        group = rng.choice([1, 2, 3, 4, 4, 6, 8, 12])
        while True:
            seqs, length = _log(rng, 1, 48), _log(rng, 1, 131072)
            if seqs * length * nKV * dH <= 2.6e8 and seqs * length * nKV * dH * group <= 1.2e9:
                return {"kind": kind, "seqs": seqs, "nH": nKV * group, "nKV": nKV, "dH": dH, "cap": length + rng.randint(0, 300),
                        "len": length, "weights": rng.random() < 0.4}
    if kind == "budget":
        group = rng.choice([1, 2, 4, 4, 8])
        while True:
            budget, seqs = _log(rng, 64, 8192), _log(rng, 1, 8)
            if seqs * budget * nKV * dH <= 8.4e6:
                return {"kind": kind, "seqs": seqs, "nH": nKV * group, "nKV": nKV, "dH": dH, "budget": budget,
                        "T": _log(rng, 1, 64), "recent": rng.randint(0, budget // 2)}
    if kind == "evict":
        while True:
            cap, layers, seqs = _log(rng, 64, 65536), _log(rng, 1, 32), _log(rng, 1, 8)
            length = rng.randint(cap // 2, cap)
            if layers * seqs * nKV * cap <= 4.2e6:
                budget = rng.randint(1, cap - 1)
                return {"kind": kind, "layers": layers, "seqs": seqs, "nKV": nKV, "cap": cap, "len": length, "budget": budget,
                        "recent": rng.randint(0, budget)}
    if kind == "select":
        while True:
            c = {"kind": kind, "reqs": _log(rng, 1, 16), "W": _log(rng, 1, 32), "V": _log(rng, 31, 128256)}
            if c["reqs"] * c["W"] * c["V"] <= 8.2e6:
                return c
    while True:
        c = {"kind": kind, "layers": _log(rng, 1, 24), "reqs": _log(rng, 1, 4), "W": _log(rng, 2, 32), "kvD": nKV * dH,
             "cap": _log(rng, 16, 4096), "len": 0}
        c["len"] = rng.randint(max(1, c["cap"] // 3), c["cap"])
        if c["layers"] * c["reqs"] * c["W"] * c["kvD"] * c["cap"] <= 7.5e7:
            return c


# ── inputs ────────────────────────────────────────────────────────────────
def _lens(c):
    """The sequences' lengths: the case's own for the first, others spread below it, one slot of a larger batch empty."""
    n = c["seqs"]
    got = [max(1, c["len"] * (n - i) // n - 3 * i) for i in range(n)]
    if n >= 4:
        got[n // 2] = 0
    return got


def _parents(c):
    """Which beam each goes on from: some go on themselves, a good beam is taken more than once."""
    rng = random.Random(c["W"] * 131 + c["reqs"])
    return [[b if rng.random() < 0.3 else rng.randrange(max(1, (c["W"] + 1) // 2)) for b in range(c["W"])] for _ in range(c["reqs"])]


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std)


def _kv(g, *shape):
    """Keys or values as projections give them: channels of their own size and offset."""
    nKV, dH = shape[-2:]
    return _randn(g, *shape).mul_(_randn(g, nKV, dH, std=0.4).exp_()).add_(_randn(g, nKV, dH, std=0.5))


def _codes(x):
    """Q4_0 codes (0..15) and fp16 steps of x [..., dH], block by block of 32."""
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    a = b.abs()
    first = (a == a.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1, keepdim=True)
    step = (b.gather(-1, first) / -8.0).to(torch.float16)
    wide = step.double()
    code = torch.where(wide == 0, 8.0, torch.floor(b.double() / wide + 8.5).clamp_(0, 15)).to(torch.uint8)
    return code, step.squeeze(-1)


def _pack(code):
    """Codes [..., dH / 32, 32] as a cache slot's bytes [..., dH / 2]."""
    low, high = code[..., :16], code[..., 16:]
    return (low | (high << 4)).transpose(-1, -2).reshape(*code.shape[:-2], -1).contiguous()


def _values(bytes_, step):
    """The values [..., dH] that a cache's bytes and steps stand for, in 32 bits."""
    nb = step.shape[-1]
    b = bytes_.reshape(*bytes_.shape[:-1], 16, nb).transpose(-1, -2)
    code = torch.cat([b & 15, b >> 4], -1).float() - 8.0
    return (code * step.float().unsqueeze(-1)).flatten(-2)


def _cache(g, c, seqs, cap):
    code, step = _codes(_kv(g, 1, seqs, cap, c["nKV"], c["dH"]).transpose(2, 3))
    return _pack(code), step.contiguous()


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = {"c": c, "kind": c["kind"]}
    kind = c["kind"]
    if kind in ("store", "attend", "budget"):
        n, nKV, dH = c["seqs"], c["nKV"], c["dH"]
        cap = c["budget"] + c["T"] if kind == "budget" else c["cap"]
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        s["next"] = i32([5 + cap] * n)
        if kind == "store":
            s["new_k"], s["new_v"] = _kv(g, n, c["T"], nKV, dH), _kv(g, n, c["T"], nKV, dH)
            s["k"], s["v"] = (torch.zeros(1, n, nKV, cap, dH // 2, dtype=torch.uint8, device="cuda") for _ in range(2))
            s["kd"], s["vd"] = (torch.zeros(1, n, nKV, cap, dH // BLOCK, dtype=torch.float16, device="cuda") for _ in range(2))
            s["len"] = i32([0] * n)
            s["out_k"], s["out_v"] = torch.empty_like(s["new_k"]), torch.empty_like(s["new_v"])
            return s
        s["k"], s["kd"] = _cache(g, c, n, cap)
        s["v"], s["vd"] = _cache(g, c, n, cap)
        s["q"] = _randn(g, n, c["nH"], dH, std=1.2)
        s["out"] = torch.empty_like(s["q"])
        s["len"] = i32(_lens(c) if kind == "attend" else [c["budget"]] * n)
        if kind == "budget" or c["weights"]:
            s["weight"] = _randn(g, 1, n, nKV, cap, std=2.0).exp_().mul_(1e-2)
            # the positions of a cache whose slots have been filled out of order
            order = torch.rand(1, n, nKV, cap, generator=g, device="cuda").argsort(-1)
            s["pos"] = (order + 5).to(torch.int32)
        if kind == "budget":
            s["next"] = i32([5 + cap] * n)
            s["new_k"], s["new_v"] = _kv(g, n, c["T"], nKV, dH), _kv(g, n, c["T"], nKV, dH)
            s["out_k"], s["out_v"] = (torch.empty(n, cap, nKV, dH, device="cuda") for _ in range(2))
        return s
    if kind == "evict":
        shape = (c["layers"], c["seqs"], c["nKV"], c["cap"])
        w = _randn(g, *shape, std=2.0).exp_()
        s["weight"] = torch.where(torch.rand(*shape, generator=g, device="cuda") < 0.1, 0.0, w)  # tokens that nothing attended to
        s["pos"] = (torch.rand(*shape, generator=g, device="cuda").argsort(-1)).to(torch.int32)
        s["len"] = torch.tensor(_lens(c), dtype=torch.int32, device="cuda")
        s["next"] = torch.full((c["seqs"],), c["cap"], dtype=torch.int32, device="cuda")
        most = max(1, min(c["budget"], c["cap"] - c["budget"]))
        s["holes"], s["movers"] = (torch.empty(*shape[:3], most, dtype=torch.int32, device="cuda") for _ in range(2))
        s["moves"] = torch.empty(*shape[:3], dtype=torch.int32, device="cuda")
        return s
    if kind == "select":
        n = c["reqs"] * c["W"]
        s["logits"] = (_randn(g, n, c["V"], std=2.5) * 64).round_().div_(64)  # ties, as a head of coarse weights has them
        s["scores"] = -(_randn(g, n, std=4.0).abs() + 10.0)
        s["done"] = (torch.rand(n, generator=g, device="cuda") < 0.1).to(torch.int32)
        s["out"] = {"scores": torch.empty(n, device="cuda"), **{k: torch.empty(n, dtype=torch.int32, device="cuda") for k in ("token", "parent", "done")}}
        return s
    n = c["reqs"] * c["W"]
    s["k"], s["v"] = (_randn(g, c["layers"], n, c["cap"], c["kvD"]) for _ in range(2))
    s["parent"] = torch.tensor(_parents(c), dtype=torch.int32, device="cuda").reshape(-1)
    s["len"] = torch.full((n,), c["len"], dtype=torch.int32, device="cuda")
    return s


# ── the framework's calls ─────────────────────────────────────────────────
_lib = None


def _forge():
    global _lib
    if _lib is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "forge-llm_amd"))
        import forge_hip
        torch.cuda.init()
        forge_hip.init(0)
        _lib = forge_hip
    return _lib


def _at(t):
    return None if t is None else t.data_ptr()


def _handle(s, fh):
    """What a program builds once for its cache or states and keeps."""
    if "handle" not in s:
        c = s["c"]
        if s["kind"] == "reorder":
            row, n = 4 * c["kvD"], c["reqs"] * c["W"]
            s["handle"] = (fh.BeamState * 2)(*[fh.BeamState(t.data_ptr(), c["cap"] * row, c["layers"], n * c["cap"] * row, 1, 0, row, c["cap"])
                                               for t in (s["k"], s["v"])])
        else:
            s["handle"] = fh.Kv4Cache(1, c["seqs"], c["nKV"], c["dH"], s["k"].shape[3], _at(s["k"]), _at(s["v"]), _at(s["kd"]), _at(s["vd"]),
                                      _at(s["len"]), _at(s["next"]), _at(s.get("weight")), _at(s.get("pos")))
    return s["handle"]


def _own(s):
    fh, c, kind = _forge(), s["c"], s["kind"]
    if kind in ("store", "attend", "budget"):
        cache, ld, scale = fh.ref(_handle(s, fh)), c["nKV"] * c["dH"], 1.0 / math.sqrt(c["dH"])
        if kind == "store":
            fh.call("kv4_append", cache, 0, _at(s["new_k"]), _at(s["new_v"]), ld, c["T"], None)
            fh.call("kv4_read", cache, 0, _at(s["out_k"]), _at(s["out_v"]), ld, 0, c["T"])
            return {"k": s["out_k"], "v": s["out_v"]}
        if kind == "attend":
            fh.call("kv4_attn", cache, 0, _at(s["out"]), _at(s["q"]), c["nH"], scale, 0, None)
            return {"out": s["out"], **({"weight": s["weight"]} if c["weights"] else {})}
        fh.call("kv4_append", cache, 0, _at(s["new_k"]), _at(s["new_v"]), ld, c["T"], None)
        fh.call("kv4_attn", cache, 0, _at(s["out"]), _at(s["q"]), c["nH"], scale, c["T"], None)
        fh.call("kv4_commit", cache, c["T"], None)
        fh.call("kv4_evict", cache, c["budget"], c["recent"])
        fh.call("kv4_read", cache, 0, _at(s["out_k"]), _at(s["out_v"]), ld, 0, c["budget"] + c["T"])
        return {"out": s["out"], "weight": s["weight"], "pos": s["pos"], "len": s["len"], "next": s["next"], "k": s["out_k"], "v": s["out_v"]}
    if kind == "evict":
        fh.call("kv_evict_select", _at(s["holes"]), _at(s["movers"]), _at(s["moves"]), _at(s["weight"]), _at(s["pos"]), _at(s["len"]),
                _at(s["next"]), c["layers"], c["seqs"], c["nKV"], c["cap"], c["budget"], c["recent"])
        return {"holes": s["holes"], "movers": s["movers"], "moves": s["moves"]}
    if kind == "select":
        o = s["out"]
        fh.call("beam_select", _at(o["scores"]), _at(o["token"]), _at(o["parent"]), _at(o["done"]), _at(s["logits"]), c["V"], _at(s["scores"]),
                _at(s["done"]), 2, c["reqs"], c["W"], c["V"])
        return o
    fh.call("beam_reorder", fh.ref(_handle(s, fh)), 2, _at(s["parent"]), _at(s["len"]), c["reqs"], c["W"])
    return {"k": s["k"], "v": s["v"]}


# ── the plain forms ───────────────────────────────────────────────────────
def _store(s, at):
    """New rows [seqs, T, nKV, dH] into the slots from `at` on."""
    T = s["c"]["T"]
    for_k, for_v = _codes(s["new_k"].transpose(1, 2)), _codes(s["new_v"].transpose(1, 2))
    s["k"][0, :, :, at:at + T], s["kd"][0, :, :, at:at + T] = _pack(for_k[0]), for_k[1]
    s["v"][0, :, :, at:at + T], s["vd"][0, :, :, at:at + T] = _pack(for_v[0]), for_v[1]


def _attend(s, n):
    """Softmax attention of q over the first n [seqs] slots, in 32 bits; the weights are added to s["weight"] if it is there."""
    c = s["c"]
    N, nH, dH = s["q"].shape
    q = s["q"].reshape(N, c["nKV"], nH // c["nKV"], dH).transpose(-1, -2).contiguous()
    score = torch.matmul(_values(s["k"][0], s["kd"][0]), q) / math.sqrt(dH)  # [seq, kv head, slot, head of the group]
    there = (torch.arange(score.shape[2], device="cuda") < n[:, None])[:, None, :, None]
    score = torch.where(there, score, -math.inf)
    top = score.amax(2, keepdim=True)
    p = torch.where(there, torch.exp(score - top), 0.0)
    total = p.sum(2, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    if "weight" in s:
        s["weight"][0] += p.sum(-1)
    out = torch.matmul(p.transpose(-1, -2).contiguous(), _values(s["v"][0], s["vd"][0]))
    return out.reshape(N, nH, dH)


def _keep(weight, pos, length, nxt, budget, recent):
    """For every head: which slots move where.  Lists of slots, holes and movers first, and the number of moves."""
    slot = torch.arange(weight.shape[-1], device="cuda")
    there = slot < length[:, None, None]
    safe = there & (pos >= (nxt - recent)[:, None, None])
    worth = torch.where(safe, math.inf, torch.where(there, weight, -math.inf))
    rank = torch.sort(worth, dim=-1, descending=True, stable=True).indices.argsort(-1)
    kept = there & ((rank < budget) | (length <= budget)[:, None, None])
    hole, mover = there & ~kept & (slot < budget), kept & (slot >= budget) & (length > budget)[:, None, None]
    first = lambda m: torch.sort((~m).to(torch.uint8), dim=-1, stable=True).indices  # noqa: E731
    return first(hole), first(mover), hole.sum(-1)


def _budget(s):
    c = s["c"]
    T, B = c["T"], c["budget"]
    _store(s, B)
    s["weight"][..., B:] = 0.0
    s["pos"][..., B:] = (s["next"][:, None] + torch.arange(T, device="cuda")).to(torch.int32)[None, :, None, :]
    out = _attend(s, s["len"] + T)
    s["next"] += T
    hole, mover, moves = _keep(s["weight"], s["pos"], s["len"] + T, s["next"], B, c["recent"])
    source = torch.where(torch.arange(B + T, device="cuda") < moves[..., None], mover, hole)
    source = torch.empty_like(hole).scatter_(-1, hole, source)
    s["weight"], s["pos"] = s["weight"].gather(-1, source), s["pos"].gather(-1, source)
    move = lambda t: t.gather(3, source[..., None].expand(-1, -1, -1, -1, t.shape[-1]))  # noqa: E731
    s["k"], s["v"], s["kd"], s["vd"] = move(s["k"]), move(s["v"]), move(s["kd"]), move(s["vd"])
    read = lambda b, d: _values(b[0], d[0]).transpose(1, 2).contiguous()  # noqa: E731
    return {"out": out, "weight": s["weight"], "pos": s["pos"], "len": s["len"], "next": s["next"], "k": read(s["k"], s["kd"]), "v": read(s["v"], s["vd"])}


def _select(s):
    c = s["c"]
    x, V, W = s["logits"].double(), c["V"], c["W"]
    top = x.amax(-1, keepdim=True)
    score = s["scores"].double()[:, None] - (top + torch.exp(x - top).sum(-1, keepdim=True).log()) + x
    only = torch.where(torch.arange(V, device="cuda") == 2, s["scores"].double()[:, None], -math.inf)
    score = torch.where(s["done"][:, None] != 0, only, score).reshape(c["reqs"], W * V)
    best, at = torch.sort(score, dim=-1, descending=True, stable=True)
    best, at = best[:, :W], at[:, :W]
    parent, token = at // V, at % V
    done = (s["done"].reshape(-1, W).gather(1, parent) != 0) | (token == 2)
    flat = lambda t, k: t.reshape(-1).to(k)  # noqa: E731
    return {"scores": flat(best, torch.float32), "token": flat(token, torch.int32), "parent": flat(parent, torch.int32), "done": flat(done, torch.int32)}


def run(s):
    if own:
        return _own(s)
    c, kind = s["c"], s["kind"]
    if kind == "store":
        _store(s, 0)
        T = c["T"]
        read = lambda b, d: _values(s[b][0, :, :, :T], s[d][0, :, :, :T]).transpose(1, 2).contiguous()  # noqa: E731
        return {"k": read("k", "kd"), "v": read("v", "vd")}
    if kind == "attend":
        out = _attend(s, s["len"])
        return {"out": out, **({"weight": s["weight"]} if c["weights"] else {})}
    if kind == "budget":
        return _budget(s)
    if kind == "evict":
        hole, mover, moves = _keep(s["weight"], s["pos"], s["len"], s["next"], c["budget"], c["recent"])
        most = s["holes"].shape[-1]
        used = torch.arange(most, device="cuda") < moves[..., None]
        cut = lambda t: torch.where(used, t[..., :most], -1).to(torch.int32)  # noqa: E731
        return {"holes": cut(hole), "movers": cut(mover), "moves": moves.to(torch.int32)}
    if kind == "select":
        return _select(s)
    W, n = c["W"], c["reqs"] * c["W"]
    source = (torch.arange(n, device="cuda") // W * W + s["parent"]).long()
    moved = (torch.arange(c["cap"], device="cuda") < s["len"][source][:, None])[None, :, :, None]
    s["k"], s["v"] = torch.where(moved, s["k"][:, source], s["k"]), torch.where(moved, s["v"][:, source], s["v"])
    return {"k": s["k"], "v": s["v"]}


def work(c):
    kind = c["kind"]
    if kind in ("store", "attend", "budget"):
        row = c["nKV"] * (c["dH"] + 4 * (c["dH"] // BLOCK))  # bytes of a token's K and V
        wide = 8 * c["nKV"] * c["dH"]
    if kind == "store":
        rows = c["seqs"] * c["T"]
        return {"bytes": rows * (2 * wide + 2 * row), "flops": 4 * rows * c["nKV"] * c["dH"]}
    if kind == "attend":
        rows = sum(_lens(c))
        per = row + (8 * c["nKV"] if c["weights"] else 0)
        return {"bytes": rows * per + 8 * c["seqs"] * c["nH"] * c["dH"], "flops": 4 * rows * c["nH"] * c["dH"]}
    if kind == "budget":
        n, T = c["budget"] + c["T"], c["T"]
        per = T * (wide + row) + n * (row + 8 * c["nKV"]) + 8 * n * c["nKV"] + 2 * T * (row + 8 * c["nKV"]) + n * (row + wide)
        return {"bytes": c["seqs"] * (per + 8 * c["nH"] * c["dH"]), "flops": 4 * c["seqs"] * n * c["nH"] * c["dH"]}
    if kind == "evict":
        heads = c["layers"] * c["nKV"]
        most = max(1, min(c["budget"], c["cap"] - c["budget"]))
        return {"bytes": heads * (8 * sum(_lens(c)) + 8 * c["seqs"] * most), "flops": heads * sum(_lens(c))}
    if kind == "select":
        n = c["reqs"] * c["W"]
        return {"bytes": 4 * n * c["V"] + 24 * n, "flops": 4 * n * c["V"]}
    moved = sum(len({p for b, p in enumerate(ps) if p != b}) + sum(p != b for b, p in enumerate(ps)) for ps in _parents(c))
    return {"bytes": max(16, moved * c["layers"] * c["len"] * c["kvD"] * 8), "flops": 0}


# ── the definitions in 64 bits ────────────────────────────────────────────
def _exact_values(x):
    """What 4-bit blocks of x [..., dH] stand for: the step of 1/-8 of the farthest value, rounded to fp16, the nearest of 16 multiples of it."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for b in range(0, x.shape[-1], BLOCK):
        v = x[..., b:b + BLOCK].double()
        lo, hi = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
        far = torch.where(hi > -lo, hi, lo)
        tie = (hi == -lo) & (hi > 0)
        if bool(tie.any()):
            where = torch.arange(v.shape[-1], device=x.device)
            at_hi = torch.where(v == hi, where, BLOCK).amin(-1, keepdim=True)
            at_lo = torch.where(v == lo, where, BLOCK).amin(-1, keepdim=True)
            far = torch.where(tie & (at_hi < at_lo), hi, far)
        step = (-0.125 * far).float().half().double()
        units = torch.floor(v / torch.where(step == 0, 1.0, step) + 0.5).clamp(-8, 7)
        out[..., b:b + BLOCK] = units * step
    return out


def _exact_rows(s, which, i, h, n):
    """Sequence i, kv head h: the cache's first n rows, taken apart byte by byte in 64 bits."""
    raw, step = s[which][0, i, h, :n], s[which + "d"][0, i, h, :n].double()
    nb = step.shape[-1]
    out = torch.empty(n, nb * BLOCK, dtype=torch.float64, device=raw.device)
    for b in range(nb):
        column = raw[:, b::nb].double()
        high = torch.floor(column / 16)
        out[:, BLOCK * b:BLOCK * b + 16] = (column - 16 * high - 8) * step[:, b:b + 1]
        out[:, BLOCK * b + 16:BLOCK * b + 32] = (high - 8) * step[:, b:b + 1]
    return out


def exact(c, seed):
    s = prepare(c, seed)
    kind = c["kind"]
    if kind == "store":
        return {"k": _exact_values(s["new_k"]), "v": _exact_values(s["new_v"])}
    if kind in ("attend", "budget"):
        N, nH, dH = s["q"].shape
        group = nH // c["nKV"]
        out = torch.zeros(N, nH, dH, dtype=torch.float64, device="cuda")
        weight = s["weight"].double() if "weight" in s else None
        if kind == "budget":
            weight[..., c["budget"]:] = 0
        for i, n in enumerate(s["len"].tolist()):
            for h in range(c["nKV"]):
                K, V = _exact_rows(s, "k", i, h, n), _exact_rows(s, "v", i, h, n)
                if kind == "budget":
                    K, V = (torch.cat([a, _exact_values(s[b][i, :, h])]) for a, b in ((K, "new_k"), (V, "new_v")))
                if not len(K):
                    continue
                for z in range(h * group, (h + 1) * group):
                    p = torch.softmax((K * s["q"][i, z].double()).sum(-1) / math.sqrt(dH), 0)
                    out[i, z] = (p[:, None] * V).sum(0)
                    if weight is not None:
                        weight[0, i, h, :len(p)] += p
        if kind == "attend":
            return {"out": out, **({"weight": weight} if weight is not None else {})}
        # the moved state follows whole numbers: only what does not depend on them is given here
        return {"out": out, "weight": None, "pos": None, "len": None, "next": None, "k": None, "v": None}
    if kind == "select":
        x, W, V = s["logits"].double().cpu().numpy(), c["W"], c["V"]
        scores, done = s["scores"].double().cpu().numpy(), s["done"].cpu().numpy()
        got = []
        for r in range(c["reqs"]):
            every = []
            for b in range(r * W, r * W + W):
                if done[b]:
                    every.append(scores[b:b + 1])
                else:
                    m = x[b].max()
                    every.append(np.sort(scores[b] + x[b] - (m + math.log(math.fsum(np.exp(x[b] - m)))))[::-1][:W])
            got.append(np.sort(np.concatenate(every))[::-1][:W])
        return {"scores": torch.from_numpy(np.concatenate(got).copy()), "token": None, "parent": None, "done": None}
    return None
