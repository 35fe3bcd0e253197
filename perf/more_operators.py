"""A key-value cache in pages and the steps of speculative decoding over it, as timed cases.

append   keys and values of new tokens into the pages, the positions' rotation applied on the way, queries rotated beside them
attend   causal attention of the new tokens (one, a few drafted ones, a chunk of a prompt) over the pages, with or
         without a sliding window and first tokens that stay visible
verify   drafted tokens against the target's probabilities: how many stand, and the token that comes after them

Tensors are torch's; the library works on a stream of its own.  The cache's layout is that of fg_paged_cache: pages
[layer][page][kv head][slot][dH] in fp32 or fp16, and a table of each sequence's pages, -1 where there is none.  Rows of
new tokens are [sequence][T], of which sequence s has count[s].
"""
import math
import os
import random
import sys

import torch

own = False


def listed():
    return [
        # one token of four conversations of the small decode model: launches and latency
        {"name": "append-token", "kind": "append", "seqs": 4, "T": 1, "ragged": False, "nH": 8, "nKV": 4, "dH": 32, "page": 16,
         "type": "f32", "len": 200, "rot": 32, "half": False},
        # drafted tokens of a serving batch, heads of Llama-3-8B, some sequences with fewer of them or none
        {"name": "append-draft-8b", "kind": "append", "seqs": 32, "T": 8, "ragged": True, "nH": 32, "nKV": 8, "dH": 128, "page": 16,
         "type": "f16", "len": 777, "rot": 128, "half": True},
        # a prompt, half of each head rotated
        {"name": "append-prompt-8b", "kind": "append", "seqs": 1, "T": 8191, "ragged": False, "nH": 32, "nKV": 8, "dH": 128, "page": 64,
         "type": "f16", "len": 0, "rot": 64, "half": False},
        # a token of four conversations of the small decode model
        {"name": "attend-small", "kind": "attend", "seqs": 4, "T": 1, "ragged": False, "nH": 8, "nKV": 4, "dH": 32, "page": 16,
         "type": "f32", "len": 200, "window": 0, "sinks": 0},
        # the chunk of a prompt of the 125M model's heads, for a batch, fp32 cache
        {"name": "attend-chunk-125m", "kind": "attend", "seqs": 4, "T": 256, "ragged": True, "nH": 12, "nKV": 12, "dH": 64, "page": 32,
         "type": "f32", "len": 768, "window": 0, "sinks": 0},
        # four drafted tokens and the one before them, for a serving batch of sequences of all lengths, one of them new
        {"name": "attend-draft-8b", "kind": "attend", "seqs": 16, "T": 5, "ragged": True, "nH": 32, "nKV": 8, "dH": 128, "page": 16,
         "type": "f16", "len": 8187, "window": 0, "sinks": 0},
        # a token after a long document
        {"name": "attend-long-8b", "kind": "attend", "seqs": 1, "T": 1, "ragged": False, "nH": 32, "nKV": 8, "dH": 128, "page": 64,
         "type": "f16", "len": 130001, "window": 0, "sinks": 0},
        # a chunk of a long prompt
        {"name": "attend-chunk-8b", "kind": "attend", "seqs": 1, "T": 512, "ragged": False, "nH": 32, "nKV": 8, "dH": 128, "page": 64,
         "type": "f16", "len": 8192, "window": 0, "sinks": 0},
        # tokens of endless conversations: the last 4096 and the first four are seen
        {"name": "attend-window-8b", "kind": "attend", "seqs": 8, "T": 1, "ragged": False, "nH": 32, "nKV": 8, "dH": 128, "page": 32,
         "type": "f16", "len": 32000, "window": 4096, "sinks": 4},
        # four drafts of the small decode model
        {"name": "verify-small", "kind": "verify", "seqs": 1, "D": 4, "V": 4096, "temperature": 0.8, "certain": False},
        # four drafts of each sequence of a serving batch, Llama-3-8B's vocabulary
        {"name": "verify-8b", "kind": "verify", "seqs": 16, "D": 4, "V": 128256, "temperature": 1.0, "certain": False},
        # drafts looked up in the text so far, which have no probabilities, the 125M model's vocabulary
        {"name": "verify-lookup", "kind": "verify", "seqs": 7, "D": 9, "V": 32000, "temperature": 0.7, "certain": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "verify", "verify"])
    if kind == "verify":
        while True:
            c = {"kind": kind, "seqs": _log(rng, 1, 32), "D": rng.randint(0, 9), "V": _log(rng, 31, 128256),
                 "temperature": rng.choice([0.0, 0.5, 0.7, 1.0, 1.0, 1.3]), "certain": rng.random() < 0.3}
            if c["seqs"] * (c["D"] + 1) * c["V"] <= 1.0e7:
                return c
    dH, nKV, group = rng.choice([32, 64, 64, 96, 128, 128, 256]), rng.choice([1, 2, 3, 4, 5, 8, 12]), rng.choice([1, 2, 3, 4, 4, 6, 8])
    c = {"kind": kind, "seqs": 1, "T": 1, "ragged": rng.random() < 0.5, "nH": nKV * group, "nKV": nKV, "dH": dH,
         "page": rng.choice([8, 16, 16, 32, 64, 128]), "type": rng.choice(["f16", "f16", "f32"]), "len": 0}
    if kind == "append":
        c.update(rot=rng.choice([0, dH // 2, dH, dH]), half=rng.random() < 0.5)
        while True:
            c.update(seqs=_log(rng, 1, 48), T=_log(rng, 1, 8191), len=rng.randint(0, 300))
            if c["seqs"] * c["T"] * (c["nH"] + 2 * nKV) * dH <= 5.0e7:
                return c
    c.update(window=0, sinks=0)
    if rng.random() < 0.3:
        c.update(window=_log(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 4, 40]))
    while True:
        c.update(seqs=_log(rng, 1, 32), T=rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 1024)]), len=_log(rng, 1, 131072) - 1)
        pairs, slots = c["seqs"] * c["T"] * (c["len"] + c["T"]), c["seqs"] * (c["len"] + c["T"])
        if slots * nKV * dH <= 1.33e8 and pairs * c["nH"] <= 1.42e8 and pairs * c["nH"] * dH <= 1.8e10:
            return c


# ── inputs ────────────────────────────────────────────────────────────────
def _counts(c):
    """New tokens of every sequence: T for the first, where the batch is ragged anything from none to T for the others."""
    rng = random.Random(c["T"] * 131 + c["seqs"])
    return [c["T"] if i == 0 or not c["ragged"] else rng.randint(0, c["T"]) for i in range(c["seqs"])]


def _lens(c):
    """Cached tokens before the new ones: the case's own number for the first, others spread below it, the middle one of a larger batch new."""
    n = c["seqs"]
    got = [max(0, c["len"] * (n - i) // n - 3 * i) for i in range(n)]
    if n >= 4:
        got[n // 2] = 0
    return got


def _visible(c):
    """Of every sequence: the slots that a query of it sees, and pairs of a query and a slot that it sees."""
    slots, pairs = [], []
    for n, t in zip(_lens(c), _counts(c)):
        sees = seen = 0
        if t:
            if not c["window"]:
                sees, seen = t * n + t * (t + 1) // 2, n + t
            else:
                for p in range(n, n + t):
                    first = max(0, p + 1 - c["window"])
                    sees += p + 1 - first + min(c["sinks"], first)
                first = max(0, n + 1 - c["window"])
                seen = n + t - first + min(c["sinks"], first)
        slots.append(seen)
        pairs.append(sees)
    return slots, pairs


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std)


def _channels(g, nKV, dH):
    """Sizes and offsets of the channels of keys or values, as projections give them."""
    return _randn(g, nKV, dH, std=0.4).exp_(), _randn(g, nKV, dH, std=0.5)


def _angles(npos, rot):
    """cos and sin of p 10000^(-i / rot), i = 0, 2, .. < rot, in 64 bits."""
    f = torch.pow(torch.tensor(10000.0, dtype=torch.float64), -torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    a = torch.arange(npos, dtype=torch.float64)[:, None] * f
    return a.cos().contiguous().cuda(), a.sin().contiguous().cuda()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(c):
    """Every sequence's pages, shuffled; none where a window has left them behind.  The table, and the number of pages."""
    rng = random.Random(c["seqs"] * 8191 + c["len"] * 31 + c["page"])
    P, need = c["page"], []
    most = max(1, max(-(-(n + t) // P) for n, t in zip(_lens(c), _counts(c))))
    for n, t in zip(_lens(c), _counts(c)):
        behind = max(0, n + 1 - c["window"]) if c.get("window") else 0
        need.append([p * P < n + t and not (c.get("sinks", 0) <= p * P and p * P + P <= behind) for p in range(most)])
    total = sum(map(sum, need)) + 2
    pages = list(range(total))
    rng.shuffle(pages)
    return _i32([[pages.pop() if there else -1 for there in row] for row in need]), total


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = {"c": c, "kind": c["kind"]}
    if c["kind"] == "verify":
        n, D, V = c["seqs"], c["D"], c["V"]
        s["logits"] = _randn(g, n, D + 1, V, std=2.5)
        # a draft model of the same opinion, more or less; its tokens are drawn from it (the Gumbel way)
        s["draft_logits"] = s["logits"][:, :D] + _randn(g, n, D, V, std=0.7)
        noise = torch.rand(n, D, V, generator=g, device="cuda").clamp_(min=1e-12).log_().neg_().log_().neg_()
        heat = c["temperature"] if c["temperature"] else 0.01
        s["draft"] = (s["draft_logits"] / heat + noise).argmax(-1).to(torch.int32) if D else torch.empty(n, 0, dtype=torch.int32, device="cuda")
        if c["certain"]:
            s["draft_logits"] = None
        s["u"] = torch.rand(n, D + 1, generator=g, device="cuda")
        s["token"], s["count"] = torch.empty(n, D + 1, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
        return s
    N, T, nH, nKV, dH = c["seqs"], c["T"], c["nH"], c["nKV"], c["dH"]
    kind = {"f32": torch.float32, "f16": torch.float16}[c["type"]]
    s["table"], pages = _table(c)
    s["len"], s["count"] = _i32(_lens(c)), _i32(_counts(c))
    if c["kind"] == "append":
        size_k, size_v = _channels(g, nKV, dH), _channels(g, nKV, dH)
        # a fused projection's rows: queries, keys and values side by side
        qkv = _randn(g, N * T, nH + 2 * nKV, dH, std=1.2)
        qkv[:, nH:nH + nKV].mul_(size_k[0]).add_(size_k[1])
        qkv[:, nH + nKV:].mul_(size_v[0]).add_(size_v[1])
        s["qkv"] = qkv
        s["k"], s["v"] = (torch.zeros(1, pages, nKV, c["page"], dH, dtype=kind, device="cuda") for _ in range(2))
        s["q_out"] = torch.zeros(N, T, nH, dH, device="cuda")
        s["cos"], s["sin"] = _angles(max(_lens(c)) + T, c["rot"])
        return s
    for name in ("k", "v"):
        size, offset = _channels(g, nKV, dH)
        s[name] = _randn(g, 1, pages, nKV, c["page"], dH).mul_(size[:, None]).add_(offset[:, None]).to(kind)
    s["q"] = _randn(g, N, T, nH, dH, std=1.2)
    s["out"] = torch.zeros_like(s["q"])
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


def _own(s):
    fh, c = _forge(), s["c"]
    if c["kind"] == "verify":
        fh.call("draft_verify", _at(s["token"]), _at(s["count"]), _at(s["logits"]), c["V"], _at(s["draft_logits"]), c["V"], _at(s["draft"]), None,
                _at(s["u"]), c["temperature"], c["seqs"], c["D"], c["V"])
        return {"token": s["token"], "count": s["count"]}
    if "handle" not in s:  # what a program builds once for its cache
        s["handle"] = fh.PagedCache(1, c["seqs"], c["nKV"], c["dH"], c["page"], s["k"].shape[1], s["table"].shape[1],
                                    {"f32": 0, "f16": 1}[c["type"]], _at(s["k"]), _at(s["v"]), _at(s["table"]), _at(s["len"]))
    cache = fh.ref(s["handle"])
    if c["kind"] == "append":
        nH, nKV, dH = c["nH"], c["nKV"], c["dH"]
        at = s["qkv"].data_ptr()
        fh.call("paged_append", cache, 0, _at(s["q_out"]), at, at + 4 * nH * dH, at + 4 * (nH + nKV) * dH, (nH + 2 * nKV) * dH, nH, c["T"],
                _at(s["count"]), _at(s["cos"]), _at(s["sin"]), s["cos"].shape[0], c["rot"], int(c["half"]))
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    fh.call("paged_attn", cache, 0, _at(s["out"]), _at(s["q"]), c["nH"], 1.0 / math.sqrt(c["dH"]), c["T"], _at(s["count"]), c["window"], c["sinks"])
    return {"out": s["out"]}


# ── the plain forms ───────────────────────────────────────────────────────
def _rotate(x, cos, sin, rot, half):
    """x [..., heads, dH] of rows whose angles are cos and sin [..., rot / 2]: the first rot values in pairs, neighbours or half of rot apart."""
    wide = x[..., :rot].double()
    a, b = (wide[..., :rot // 2], wide[..., rot // 2:]) if half else (wide[..., 0::2], wide[..., 1::2])
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([a, b], -1) if half else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:].double()], -1)


def _append(s):
    c = s["c"]
    N, T, nH, nKV, P = c["seqs"], c["T"], c["nH"], c["nKV"], c["page"]
    t = torch.arange(T, device="cuda")
    there = t < s["count"][:, None]
    pos = torch.where(there, s["len"][:, None] + t, 0).long()
    rows = s["qkv"].reshape(N, T, nH + 2 * nKV, c["dH"])
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotate(rows[:, :, :nH], cos, sin, c["rot"], c["half"]).float()
    k = _rotate(rows[:, :, nH:nH + nKV], cos, sin, c["rot"], c["half"]).to(s["k"].dtype)
    s["q_out"] = torch.where(there[..., None, None], q, s["q_out"])
    page = s["table"].gather(1, pos // P)[there].long()
    slot = (pos % P)[there]
    s["k"][0, page, :, slot] = k[there]
    s["v"][0, page, :, slot] = rows[:, :, nH + nKV:][there].to(s["v"].dtype)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _attend(s):
    c = s["c"]
    N, T, nH, nKV, dH, P = c["seqs"], c["T"], c["nH"], c["nKV"], c["dH"], c["page"]
    group, n = nH // nKV, s["table"].shape[1] * P
    pages = s["table"].clamp(min=0).long()
    row = lambda b: s[b][0][pages].transpose(1, 2).reshape(N, nKV, n, dH).float()  # noqa: E731
    q = s["q"].reshape(N, T, nKV, group, dH).transpose(1, 2).reshape(N, nKV, T * group, dH)
    score = torch.matmul(q, row("k").transpose(-1, -2).contiguous()) / math.sqrt(dH)
    slot, t = torch.arange(n, device="cuda"), torch.arange(T, device="cuda")
    pos = s["len"][:, None] + t
    sees = slot <= pos[..., None]
    if c["window"]:
        sees = sees & ((slot > pos[..., None] - c["window"]) | (slot < c["sinks"]))
    sees = sees & (t < s["count"][:, None])[..., None] & (s["table"] >= 0).repeat_interleave(P, 1)[:, None]
    sees = sees[:, None, :, None].expand(-1, -1, -1, group, -1).reshape(N, 1, T * group, n)
    score = torch.where(sees, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.where(sees, torch.exp(score - top), 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    out = torch.matmul(p, row("v")).reshape(N, nKV, T, group, dH).transpose(1, 2).reshape(N, T, nH, dH)
    return {"out": torch.where((t < s["count"][:, None])[..., None, None], out, s["out"])}


def _verify(s):
    c = s["c"]
    D, V, heat = c["D"], c["V"], c["temperature"]
    n = torch.arange(c["seqs"], device="cuda")
    x, at = s["logits"], s["draft"].long().unsqueeze(-1)
    where = torch.arange(V, device="cuda")

    def chances(y):  # in 64 bits: a number next to a border decides for one token or the next
        e = torch.exp((y.double() - y.double().amax(-1, keepdim=True)) / heat)
        return e / e.sum(-1, keepdim=True)
    if heat == 0:
        best = torch.where(x == x.amax(-1, keepdim=True), where, V).amin(-1)
        stands = best[:, :D] == s["draft"]
    else:
        p = chances(x)
        q = (where == at).double() if c["certain"] else chances(s["draft_logits"])
        stands = s["u"][:, :D].double() * q.gather(-1, at).squeeze(-1) < p[:, :D].gather(-1, at).squeeze(-1)
    taken = torch.cumprod(stands.to(torch.int32), 1).sum(1) if D else torch.zeros_like(n)
    if heat == 0:
        last = best[n, taken]
    else:
        less = torch.cat([q, torch.zeros_like(p[:, :1])], 1)[n, taken]
        left = (p[n, taken] - less).clamp_(min=0.0)
        left = torch.where(left.sum(-1, keepdim=True) > 0, left, p[n, taken])
        reach = left.cumsum(-1)
        last = (reach <= s["u"][:, D:].double() * reach[:, -1:]).sum(-1).clamp_(max=V - 1)
    t = torch.arange(D + 1, device="cuda")
    drafts = torch.cat([s["draft"], torch.full_like(s["count"][:, None], -1)], 1)
    token = torch.where(t < taken[:, None], drafts, torch.where(t == taken[:, None], last[:, None], -1))
    return {"token": token.to(torch.int32), "count": (taken + 1).to(torch.int32)}


def run(s):
    if own:
        return _own(s)
    return {"append": _append, "attend": _attend, "verify": _verify}[s["kind"]](s)


def work(c):
    if c["kind"] == "verify":
        rows = c["seqs"] * (c["D"] + 1 + (0 if c["certain"] or not c["temperature"] else c["D"]))
        return {"bytes": 4 * rows * c["V"] + 16 * c["seqs"] * (c["D"] + 1), "flops": 4 * rows * c["V"]}
    one = {"f32": 4, "f16": 2}[c["type"]]
    if c["kind"] == "append":
        rows, kv = sum(_counts(c)), 2 * c["nKV"] * c["dH"]
        return {"bytes": rows * (8 * c["nH"] * c["dH"] + (4 + one) * kv) + 8 * c["T"] * c["rot"], "flops": 3 * rows * (c["nH"] + c["nKV"]) * c["rot"]}
    slots, pairs = _visible(c)
    return {"bytes": sum(slots) * 2 * c["nKV"] * c["dH"] * one + 8 * sum(_counts(c)) * c["nH"] * c["dH"], "flops": 4 * sum(pairs) * c["nH"] * c["dH"]}


# ── the definitions in 64 bits ────────────────────────────────────────────
def _exact_turn(x, pos, rot, half):
    """One row x [heads, dH] at position pos: each pair as a complex number times e^(i angle)."""
    y = x.double().clone()
    for i in range(rot // 2):
        a, b = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
        angle = pos * 10000.0 ** (-2.0 * i / rot)
        y[..., a] = x[..., a].double() * torch.cos(angle) - x[..., b].double() * torch.sin(angle)
        y[..., b] = x[..., a].double() * torch.sin(angle) + x[..., b].double() * torch.cos(angle)
    return y


def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "verify":
        return None  # whole numbers alone
    N, T, nH, nKV, dH, P = c["seqs"], c["T"], c["nH"], c["nKV"], c["dH"], c["page"]
    lens, counts, table = _lens(c), _counts(c), s["table"].cpu()
    if c["kind"] == "append":
        q, k, v = s["q_out"].double(), s["k"].double(), s["v"].double()
        rows = s["qkv"].reshape(N, T, nH + 2 * nKV, dH)
        for i in range(N):
            if not counts[i]:
                continue
            pos = torch.arange(lens[i], lens[i] + counts[i])
            at, slot, mine = table[i][pos // P].long().cuda(), (pos % P).cuda(), rows[i, :counts[i]]
            turn = pos.double().cuda()[:, None]
            q[i, :counts[i]] = _exact_turn(mine[:, :nH], turn, c["rot"], c["half"])
            k[0, at, :, slot] = _exact_turn(mine[:, nH:nH + nKV], turn, c["rot"], c["half"])
            v[0, at, :, slot] = mine[:, nH + nKV:].double()
        return {"q": q, "k": k, "v": v}
    out, group = s["out"].double(), nH // nKV
    for i in range(N):
        n = lens[i] + counts[i]
        if not counts[i]:
            continue
        slot = torch.tensor([j for j in range(n) if table[i][j // P] >= 0])
        at, within, slot = table[i][slot // P].long().cuda(), (slot % P).cuda(), slot.cuda()
        pos = torch.arange(lens[i], n, device="cuda")[:, None]
        hidden = slot > pos
        if c["window"]:
            hidden |= (pos - slot >= c["window"]) & (slot >= c["sinks"])
        for h in range(nKV):
            K, V = s["k"][0, at, h, within].double(), s["v"][0, at, h, within].double()
            for z in range(h * group, (h + 1) * group):
                score = torch.mm(s["q"][i, :counts[i], z].double(), K.t().contiguous()) * dH ** -0.5
                out[i, :counts[i], z] = torch.mm(torch.softmax(score.masked_fill(hidden, -math.inf), -1), V)
    return {"out": out}
