"""What is timed of the operators that serve a batch of conversations: keys and values in pages, attention that reads a
prefix shared by the whole batch once, and sampling of the next words.

Kinds of case:
  plan    block tables and slot maps from the lengths of the requests: page_plan
  put     head norms, rotation and the write of keys and values into their pages: page_put
  attn    attention of every request over the shared prefix and its own pages: page_attn
  sample  one word for each row of scores, by temperature, top-k, top-p and min-p and a given random number: sample

With `own` false the same results come from elementary torch operations. `exact` has them in 64 bits, request by request
and row by row.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decode step of 64 conversations: one new position each, a page opened now and then
        {"name": "plan_decode", "kind": "plan", "n": 64, "held": 1000, "add": 1, "page": 16, "spare": 0},
        # 500 conversations of which most join with a prompt, odd lengths throughout
        {"name": "plan_prompts", "kind": "plan", "n": 500, "held": 300, "add": 1999, "page": 64, "spare": 37},
        # the keys and values of a decode step of 64 conversations (32 / 8 heads of 64)
        {"name": "put_decode", "kind": "put", "rows": 64, "n_head": 32, "n_kv": 8, "dim": 64, "page": 64, "src": "f32", "type": "f16"},
        # prompts of 8191 positions together on the wide heads (16 / 4 of 128)
        {"name": "put_prompts", "kind": "put", "rows": 8191, "n_head": 16, "n_kv": 4, "dim": 128, "page": 32, "src": "f32", "type": "bf16"},
        # slot A and slot B behind one short instruction: the smallest batch, where launches count
        {"name": "attn_pair", "kind": "attn", "n": 2, "n_head": 32, "n_kv": 8, "dim": 64, "page": 16, "type": "f16", "prefix": 90, "own": 45,
         "rows": 1, "window": 0},
        # 48 conversations on the wide heads, each deep in a context of its own behind an instruction of odd length
        {"name": "attn_own_contexts", "kind": "attn", "n": 48, "n_head": 16, "n_kv": 4, "dim": 128, "page": 32, "type": "bf16", "prefix": 1001,
         "own": 4096, "rows": 1, "window": 0},
        # one conversation in a very long context, nothing shared
        {"name": "attn_long_single", "kind": "attn", "n": 1, "n_head": 32, "n_kv": 8, "dim": 64, "page": 128, "type": "f16", "prefix": 0,
         "own": 65521, "rows": 1, "window": 0},
        # prompts of up to 300 positions behind the shared prefix, in layers with a window of 256
        {"name": "attn_prompts_window", "kind": "attn", "n": 13, "n_head": 16, "n_kv": 4, "dim": 128, "page": 64, "type": "f16", "prefix": 500,
         "own": 700, "rows": 300, "window": 256},
        # the largest batch: 256 conversations share 8192 positions and hold up to 2048 each
        {"name": "attn_shared_256", "kind": "attn", "n": 256, "n_head": 32, "n_kv": 8, "dim": 64, "page": 64, "type": "f16", "prefix": 8192,
         "own": 2048, "rows": 1, "window": 0},
        # the next word of one conversation over the whole word table
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 97496, "type": "f32", "filters": "mixed"},
        # 61 rows of an odd word table in 16 bits, top-p alone
        {"name": "sample_top_p_odd", "kind": "sample", "rows": 61, "vocab": 32003, "type": "bf16", "filters": "top_p"},
        # the largest batch's next words
        {"name": "sample_256", "kind": "sample", "rows": 256, "vocab": 97496, "type": "f32", "filters": "mixed"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "put", "attn", "attn", "attn", "sample", "sample"])
    if kind == "plan":
        n = _log(rng, 1, 2048)
        return {"kind": kind, "n": n, "held": _log(rng, 1, 4096), "add": 1 if rng.random() < 0.4 else _log(rng, 2, max(2, min(4096, 900000 // n))),
                "page": rng.choice([16, 32, 64, 128, 256]), "spare": rng.randint(0, 100)}
    heads = rng.choice([(32, 8, 64), (16, 4, 128), (8, 2, 32), (12, 4, 64), (7, 1, 128), (6, 6, 64), (20, 1, 64)])
    layout = {"n_head": heads[0], "n_kv": heads[1], "dim": heads[2], "page": rng.choice([16, 32, 64, 128, 256])}
    if kind == "put":
        return {"kind": kind, "rows": _log(rng, 1, 8000), **layout, "src": rng.choice(["f32", "f16", "bf16"]), "type": rng.choice(["f16", "bf16"])}
    if kind == "attn":
        case = {"kind": kind, **layout, "type": rng.choice(["f16", "bf16"]), "window": rng.choice([0, 0, 0, _log(rng, 8, 4096)])}
        if rng.random() < 0.3:   # prompts
            n, prefix, held, rows = _log(rng, 1, 32), rng.choice([0, _log(rng, 1, 2048)]), _log(rng, 1, 1024), _log(rng, 2, 300)
        else:
            n, prefix, rows = _log(rng, 1, 256), rng.choice([0, _log(rng, 1, 8192), _log(rng, 64, 8192)]), 1
            held = _log(rng, 1, min(65536, 400000 // n))
        return {**case, "n": n, "prefix": prefix, "own": max(held, rows), "rows": rows}
    vocab = _log(rng, 200, 200000)
    return {"kind": kind, "rows": _log(rng, 1, max(1, min(512, 20000000 // vocab))), "vocab": vocab, "type": rng.choice(["f32", "f32", "f16", "bf16"]),
            "filters": rng.choice(["mixed", "none", "top_k", "top_p", "min_p"])}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _integers(g, low, high, *size):
    return torch.randint(low, high + 1, size, generator=g, device="cuda", dtype=torch.int32)


def _spread(g, most, n):
    """n lengths spread evenly over 0 .. most, the longest among them, in an order of the seed's: their sum is the case's own."""
    lengths = most - torch.arange(n, device="cuda") * (most + 1) // n
    return lengths[torch.randperm(n, generator=g, device="cuda")].to(torch.int32)


def _pages_of(lens, page, g, spare):
    """Tables of shuffled pages for requests of these lengths, and the pages nobody has (in the order they are given out)."""
    counts = ((lens + page - 1) // page).tolist()
    total = sum(counts)
    order = torch.randperm(total + spare, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(counts), max(max(counts), 1)), -1, dtype=torch.int32, device="cuda")
    flat = torch.arange(table.shape[1], device="cuda")[None, :] < torch.tensor(counts, device="cuda")[:, None]
    table[flat] = order[:total]
    return table, order[total:], total + spare


def _prepare_plan(case, seed):
    g = _generator(seed)
    n, page = case["n"], case["page"]
    held = _integers(g, 0, case["held"], n)
    add = torch.ones_like(held) if case["add"] == 1 else _spread(g, case["add"], n)
    more = int((((held + add + page - 1) // page) - ((held + page - 1) // page)).sum())
    have, free, _ = _pages_of(held, page, g, more + case["spare"])
    cols = (case["held"] + case["add"] + page - 1) // page
    table = torch.full((n, cols), -1, dtype=torch.int32, device="cuda")
    table[:, :have.shape[1]] = have[:, :cols]
    rows = int(add.sum())
    return {"held": held, "add": add, "free": torch.cat([free[:3], free]), "taken": torch.full((1,), 3, dtype=torch.int32, device="cuda"),
            "table": table, "page": page, "pos0": 17, "rows": rows,
            "out_len": torch.zeros_like(held), "cu": torch.zeros(n + 1, dtype=torch.int32, device="cuda"),
            "slots": torch.full((rows,), -1, dtype=torch.int64, device="cuda"), "pos": torch.zeros(rows, dtype=torch.int32, device="cuda"),
            "out_taken": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _prepare_put(case, seed):
    g = _generator(seed)
    H, K, D, page, R = case["n_head"], case["n_kv"], case["dim"], case["page"], case["rows"]
    pages = -(-(R + R // 8 + 1) // page)
    ld = (H + 2 * K) * D + H      # the head gates of the packed table's output ride behind q, k and v
    qkv = torch.randn(R, ld, generator=g, device="cuda").to(TYPES[case["src"]])
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:R].contiguous()
    if R > 1:
        slots[R // 2] = -1        # a row that has no place
    positions = 4096
    pos = _integers(g, 0, positions - 1, R)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) * 2 / D)
    caches = [torch.randn(pages, K, page, D, generator=g, device="cuda").to(TYPES[case["type"]]) for _ in range(2)]
    return {"qkv": qkv, "slots": slots, "pos": pos, "rope": torch.stack([angle.cos(), angle.sin()], -1).float().contiguous(),
            "q_norm": 1 + 0.1 * torch.randn(D, generator=g, device="cuda"), "k_norm": 1 + 0.1 * torch.randn(D, generator=g, device="cuda"),
            "kc": caches[0], "vc": caches[1], "q": torch.zeros(R, H, D, device="cuda", dtype=TYPES[case["type"]]), "eps": 1e-5}


def _prepare_attn(case, seed):
    g = _generator(seed)
    n, H, K, D, page = case["n"], case["n_head"], case["n_kv"], case["dim"], case["page"]
    kind = TYPES[case["type"]]
    if case["rows"] == 1:
        add, cu = None, None
        length = _integers(g, max(1, case["own"] // 8), case["own"], n)
        rows = n
    else:
        add = _spread(g, case["rows"], n)
        length = torch.maximum(add, _integers(g, 0, case["own"], n))
        cu = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
        cu[1:] = add.cumsum(0)
        rows = int(add.sum())
    table, spare, pages = _pages_of(length, page, g, -(-case["prefix"] // page) + 1)
    kc = torch.randn(pages, K, page, D, generator=g, device="cuda").to(kind)
    vc = torch.randn(pages, K, page, D, generator=g, device="cuda").to(kind)
    q = (2 * torch.randn(rows, H, D, generator=g, device="cuda")).to(kind)
    return {"q": q, "kc": kc, "vc": vc, "prefix": spare[:-(-case["prefix"] // page)].contiguous(), "prefix_len": case["prefix"], "table": table,
            "length": length, "cu": cu, "max_len": max(1, int(length.max())), "max_rows": case["rows"], "window": case["window"],
            "gate": torch.randn(rows, H, generator=g, device="cuda"), "out": torch.zeros_like(q),
            "lse": torch.zeros(rows, H, device="cuda")}


def _prepare_sample(case, seed):
    g = _generator(seed)
    R, V, what = case["rows"], case["vocab"], case["filters"]
    scores = 3 * torch.randn(R, V, generator=g, device="cuda")
    banned = torch.rand(V, generator=g, device="cuda") < 0.02
    scores[::2, banned] = -math.inf       # words that half of the rows may not say
    pick = torch.rand(R, 4, generator=g, device="cuda")
    temp = 0.5 + torch.rand(R, generator=g, device="cuda")
    top_k = torch.zeros(R, dtype=torch.int32, device="cuda")
    top_p, min_p = torch.ones(R, device="cuda"), torch.zeros(R, device="cuda")
    mixed = what == "mixed"
    if what == "top_k" or mixed:
        k = torch.exp(torch.rand(R, generator=g, device="cuda") * math.log(2000)).to(torch.int32)
        top_k = torch.where(pick[:, 0] < (0.6 if mixed else 2), k, top_k)
    if what == "top_p" or mixed:
        top_p = torch.where(pick[:, 1] < (0.6 if mixed else 2), 0.7 + 0.29 * torch.rand(R, generator=g, device="cuda"), top_p)
    if what == "min_p" or mixed:
        min_p = torch.where(pick[:, 2] < (0.4 if mixed else 2), 0.1 * torch.rand(R, generator=g, device="cuda"), min_p)
    if mixed and R > 1:
        temp = torch.where(pick[:, 3] < 0.1, torch.zeros_like(temp), temp)   # greedy rows among the others
    return {"scores": scores.to(TYPES[case["type"]]), "u": torch.rand(R, generator=g, device="cuda", dtype=torch.float64), "temp": temp,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "ids": torch.zeros(R, dtype=torch.int32, device="cuda"),
            "chance": torch.zeros(R, device="cuda")}


def prepare(case, seed):
    make = {"plan": _prepare_plan, "put": _prepare_put, "attn": _prepare_attn, "sample": _prepare_sample}[case["kind"]]
    return {"kind": case["kind"], **make(case, seed)}


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _plan(s):
    held, add, page, table = s["held"].long(), s["add"].long(), s["page"], s["table"]
    have, want = (held + page - 1) // page, (held + add + page - 1) // page
    need = want - have
    start = need.cumsum(0) - need
    taken = s["taken"].long()
    fits = (want <= table.shape[1]) & ((need == 0) | (taken + start + need <= s["free"].numel()))
    cu = torch.zeros(held.numel() + 1, dtype=torch.int64, device="cuda")
    cu[1:] = add.cumsum(0)
    col = torch.arange(table.shape[1], device="cuda")[None, :]
    fresh = (taken + start)[:, None] + col - have[:, None]
    opened = (col >= have[:, None]) & (col < want[:, None]) & fits[:, None]
    new_table = torch.where(opened, s["free"][fresh.clamp(0, s["free"].numel() - 1)], table)
    who = torch.repeat_interleave(torch.arange(held.numel(), device="cuda"), add, output_size=s["rows"])
    at = held[who] + torch.arange(s["rows"], device="cuda") - cu[who]
    slot = new_table[who, (at // page).clamp(max=table.shape[1] - 1)].long() * page + at % page
    return {"table": new_table, "len": (held + add * fits).int(), "cu": cu.int(), "slots": torch.where(fits[who], slot, -1),
            "pos": (at + s["pos0"]).int(), "taken": (taken + (need * fits).sum()).int()}


def _turned(x, w, eps, cs):
    """Heads [rows][heads][D] in 32 bits: norm over the head, then the rotation of the pairs (i, i + D / 2)."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w
    a, b = x.chunk(2, -1)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _put(s):
    R, H, D = s["q"].shape
    K, page = s["kc"].shape[1:3]
    x = s["qkv"].float()
    cs = s["rope"][s["pos"].long()]
    q = _turned(x[:, :H * D].view(R, H, D), s["q_norm"], s["eps"], cs)
    k = _turned(x[:, H * D:(H + K) * D].view(R, K, D), s["k_norm"], s["eps"], cs)
    v = x[:, (H + K) * D:(H + 2 * K) * D].view(R, K, D)
    there = s["slots"] >= 0
    slot = s["slots"][there]
    s["kc"][slot // page, :, slot % page] = k[there].to(s["kc"].dtype)
    s["vc"][slot // page, :, slot % page] = v[there].to(s["vc"].dtype)
    return {"q": q.to(s["q"].dtype), "k": s["kc"], "v": s["vc"]}


def _rows_of(pages, cache):
    """[n][pages] page ids -> keys or values [n][kv][positions][D] in 32 bits."""
    x = cache[pages.long().clamp(min=0)].float()
    n, P, K, page, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(n, K, P * page, D)


def _attn(s):
    R, H, D = s["q"].shape
    K, n, L0, m = s["kc"].shape[1], s["length"].numel(), s["prefix_len"], s["max_rows"]
    group, length = H // K, s["length"].long()
    if s["cu"] is None:
        who, nth, add = torch.arange(n, device="cuda"), torch.zeros(n, dtype=torch.int64, device="cuda"), torch.ones_like(length)
    else:
        cu = s["cu"].long()
        add = cu[1:] - cu[:-1]
        who = torch.repeat_interleave(torch.arange(n, device="cuda"), add, output_size=R)
        nth = torch.arange(R, device="cuda") - cu[who]
    q = torch.zeros(n, m, H, D, device="cuda")
    q[who, nth] = s["q"].float()
    q = q.view(n, m, K, group, D).permute(0, 2, 1, 3, 4).reshape(n, K, m * group, D)
    k, v = _rows_of(s["table"], s["kc"])[:, :, :s["max_len"]], _rows_of(s["table"], s["vc"])[:, :, :s["max_len"]]
    at = L0 + (length - add)[:, None] + torch.arange(m, device="cuda")          # [n][m] positions of the query rows
    at = at.repeat_interleave(group, 1)[:, None, :, None]
    key = L0 + torch.arange(k.shape[2], device="cuda")
    seen = (key <= at) & ((key > at - s["window"]) if s["window"] else True)
    score = (torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(D)).masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    if L0:
        k0, v0 = _rows_of(s["prefix"][None], s["kc"])[0, :, :L0], _rows_of(s["prefix"][None], s["vc"])[0, :, :L0]
        q0 = q.permute(1, 0, 2, 3).reshape(K, n * m * group, D)
        score0 = (torch.matmul(q0, k0.transpose(1, 2).contiguous()) / math.sqrt(D)).view(K, n, m * group, L0).permute(1, 0, 2, 3)
        if s["window"]:
            score0 = score0.masked_fill(torch.arange(L0, device="cuda") <= at - s["window"], -math.inf)
        top = torch.maximum(top, score0.amax(-1, keepdim=True))
    top = top.clamp(min=-3e38)
    p = torch.exp_(score.sub_(top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v)
    if L0:
        p0 = torch.exp(score0 - top)
        total = total + p0.sum(-1, keepdim=True)
        out = out + torch.matmul(p0.permute(1, 0, 2, 3).reshape(K, n * m * group, L0), v0).view(K, n, m * group, D).permute(1, 0, 2, 3)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + torch.log(total))[..., 0]

    def rows(x):   # [n][K][m * group][...] -> [rows][H][...]
        return x.view(n, K, m, group, -1).permute(0, 2, 1, 3, 4).reshape(n, m, H, -1)[who, nth]

    return {"out": (rows(out) * torch.sigmoid(s["gate"])[..., None]).to(s["q"].dtype), "lse": rows(lse)[..., 0]}


def _sample(s):
    x = s["scores"].double()
    R, V = x.shape
    top, first = x.max(1, keepdim=True)
    greedy = s["temp"] == 0
    temp = torch.where(greedy, torch.ones_like(s["temp"]), s["temp"]).double()[:, None]
    w = torch.exp((x - top) / temp)
    _, order = torch.sort(x, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    rank = torch.arange(V, device="cuda")[None, :]
    keep = (rank < torch.where(s["top_k"] > 0, s["top_k"], V)[:, None]) & (ws > 0)
    ws = ws * keep
    before = ws.cumsum(1) - ws
    top_p = s["top_p"].double()[:, None]
    keep &= (top_p >= 1) | (before < top_p * ws.sum(1, keepdim=True)) | (rank == 0)
    keep &= (ws >= s["min_p"].double().clamp(max=1)[:, None])
    w = torch.zeros_like(w).scatter_(1, order, ws * keep)
    cdf = w.cumsum(1)
    total = cdf[:, -1:]
    pick = (cdf <= s["u"][:, None] * total).sum(1, keepdim=True).clamp(max=V - 1)
    pick = torch.where(greedy[:, None], (x == top).int().argmax(1, keepdim=True), pick)
    chance = torch.where(greedy, torch.ones_like(s["u"]), (w.gather(1, pick) / total)[:, 0])
    return {"ids": pick[:, 0].int(), "chance": chance.float()}


# ---- the framework's calls -----------------------------------------------------------------------------------------

_contexts: dict = {}


def _context():
    """The program's context on the stream that its tensors are made on."""
    import nunchi_amd
    at = torch.cuda.current_stream().cuda_stream
    if at not in _contexts:
        _contexts[at] = nunchi_amd.Context(torch.cuda.current_device(), stream=at)
    return _contexts[at]


def _shape(s):
    """The layout of the pages that `s` holds, made once."""
    import nunchi_amd
    if "shape" not in s:
        pages, K, page, D = s["kc"].shape
        s["shape"] = nunchi_amd.PageShape(n_head=s["q"].shape[1], n_kv=K, head_dim=D, page=page, n_pages=pages,
                                          dtype="f16" if s["kc"].dtype == torch.float16 else "bf16", window=s.get("window", 0), eps=s.get("eps", 1e-5))
    return s["shape"]


def _own(s):
    import nunchi_amd
    ctx = _context()
    if s["kind"] == "plan":
        nunchi_amd.page_plan(ctx, s["held"], s["add"], s["free"], s["taken"], s["table"], s["page"], s["out_len"], s["cu"], s["slots"], s["pos"],
                             s["out_taken"], pos0=s["pos0"])
        return {"table": s["table"], "len": s["out_len"], "cu": s["cu"], "slots": s["slots"], "pos": s["pos"], "taken": s["out_taken"]}
    if s["kind"] == "put":
        nunchi_amd.page_put(ctx, _shape(s), s["qkv"], s["slots"], s["kc"], s["vc"], q=s["q"], pos=s["pos"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                            rope=s["rope"])
        return {"q": s["q"], "k": s["kc"], "v": s["vc"]}
    if s["kind"] == "attn":
        shape = _shape(s)
        if "work" not in s:
            size = nunchi_amd.page_attn_work(shape, s["length"].numel(), s["q"].shape[0], s["max_len"], max_rows=s["max_rows"], prefix_len=s["prefix_len"])
            s["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        nunchi_amd.page_attn(ctx, shape, s["q"], s["kc"], s["vc"], s["table"], s["length"], s["out"], s["work"], s["max_len"], cu=s["cu"],
                             max_rows=s["max_rows"], prefix=s["prefix"], prefix_len=s["prefix_len"], gate=s["gate"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if "work" not in s:
        s["work"] = torch.empty(nunchi_amd.sample_work(*s["scores"].shape), dtype=torch.uint8, device="cuda")
    nunchi_amd.sample(ctx, s["scores"], s["u"], s["ids"], s["work"], temp=s["temp"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                      chance=s["chance"])
    return {"ids": s["ids"], "chance": s["chance"]}


def run(s):
    if own:
        return _own(s)
    return {"plan": _plan, "put": _put, "attn": _attn, "sample": _sample}[s["kind"]](s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "plan":
        n, add = case["n"], 1 if case["add"] == 1 else case["add"] / 2
        opened = add / case["page"]
        return {"bytes": n * (8 + 8 + 8 * opened + 12 * add), "flops": n * add}
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if kind == "put":
        R, H, K, D = case["rows"], case["n_head"], case["n_kv"], case["dim"]
        return {"bytes": R * (H + 2 * K) * D * (size[case["src"]] + 2) + R * (12 + 4 * D), "flops": 10.0 * R * (H + K) * D}
    if kind == "attn":
        n, H, K, D, L0, m, win = case["n"], case["n_head"], case["n_kv"], case["dim"], case["prefix"], case["rows"], case["window"]
        if m == 1:
            held, rows = case["own"] * 9 / 16, n
        else:
            held, rows = max(case["own"], m) / 2 + m * m / (6 * max(case["own"], m)), n * m / 2
        seen0, seen = L0, held - (0 if m == 1 else m / 4)      # keys a row sees in the prefix, and of its own
        read0, read = L0, held                                 # positions that have to be read of the prefix, and of a request
        if win:
            read = min(read, win + m)
            seen = min(seen, win)
            seen0 = min(L0, max(0, win - seen))
            read0 = min(read0, max(0, win))
        return {"bytes": 4.0 * K * D * (read0 + n * read) + rows * H * (4 * D + 8), "flops": 4.0 * rows * H * D * (seen0 + seen)}
    return {"bytes": case["rows"] * (case["vocab"] * size[case["type"]] + 32), "flops": 4.0 * case["rows"] * case["vocab"]}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _exact_heads(x, w, eps, rope, pos, slots=None):
    """One row's heads [heads][D]: normed, and turned by complex multiplication."""
    half = x.shape[-1] // 2
    x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + eps) * w
    z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(rope[pos, :, 0], rope[pos, :, 1])[:, None]
    return torch.cat([z.real, z.imag], -1)


def _exact_put(s):
    R, H, D = s["q"].shape
    K, page = s["kc"].shape[1:3]
    pos, rope = s["pos"].long(), s["rope"].double()
    k, v = s["kc"].double(), s["vc"].double()
    q_in, k_in, v_in = torch.split(s["qkv"].double()[:, :(H + 2 * K) * D].reshape(R, -1, D), [H, K, K], 1)
    keys = _exact_heads(k_in, s["k_norm"].double(), s["eps"], rope, pos)
    for r, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            k[slot // page, :, slot % page], v[slot // page, :, slot % page] = keys[r], v_in[r]
    return {"q": _exact_heads(q_in, s["q_norm"].double(), s["eps"], rope, pos), "k": k, "v": v}


def _exact_attn(s):
    R, H, D = s["q"].shape
    K, L0 = s["kc"].shape[1], s["prefix_len"]
    out, lse = torch.zeros(R, H, D, dtype=torch.float64, device="cuda"), torch.zeros(R, H, dtype=torch.float64, device="cuda")
    starts = list(range(R + 1)) if s["cu"] is None else s["cu"].tolist()

    def gather(cache, i, held):
        page = cache.shape[2]
        ids = torch.cat([s["prefix"], s["table"][i, :-(-held // page)]]).long()
        x = cache[ids].double().transpose(1, 2).reshape(-1, K, D)
        return torch.cat([x[:L0], x[s["prefix"].numel() * page:][:held]])

    for i, held in enumerate(s["length"].tolist()):
        r0, r1 = starts[i], starts[i + 1]
        if r0 == r1:
            continue
        k, v = gather(s["kc"], i, held), gather(s["vc"], i, held)
        at = L0 + held - (r1 - r0) + torch.arange(r1 - r0, device="cuda")
        j = torch.arange(L0 + held, device="cuda")
        hide = (j[None] > at[:, None]) | ((at[:, None] - j[None] >= s["window"]) if s["window"] else False)
        for g in range(K):
            heads = slice(g * (H // K), (g + 1) * (H // K))
            q = s["q"][r0:r1, heads].double()
            z = (q.reshape(-1, D) @ k[:, g].T.contiguous()).view(r1 - r0, H // K, -1) / math.sqrt(D)
            z = z.masked_fill(hide[:, None], -math.inf)
            lse[r0:r1, heads] = torch.logsumexp(z, -1)
            out[r0:r1, heads] = (torch.softmax(z, -1).view(-1, L0 + held) @ v[:, g].contiguous()).view(r1 - r0, -1, D)
    return {"out": out / (1 + torch.exp(-s["gate"].double()))[..., None], "lse": lse}


def _exact_sample(s):
    ids, chance = [], []
    host = {k: s[k].double().cpu().numpy() for k in ("scores", "u", "temp", "top_k", "top_p", "min_p")}
    for x, u, temp, top_k, top_p, min_p in zip(*(host[k] for k in ("scores", "u", "temp", "top_k", "top_p", "min_p"))):
        if temp == 0:
            ids.append(int(np.argmax(x)))
            chance.append(1.0)
            continue
        words = np.argsort(-x, kind="stable")
        if top_k > 0:
            words = words[:int(top_k)]
        w = np.exp((x[words] - x[words[0]]) / temp)
        if top_p < 1:
            words = words[:1 + int(np.count_nonzero(np.cumsum(w)[:-1] < top_p * w.sum()))]
        words = np.sort(words[w[:len(words)] >= min(min_p, 1.0)])
        w = np.exp((x[words] - x.max()) / temp)
        sums = np.cumsum(w)
        at = min(int(np.searchsorted(sums, u * sums[-1], side="right")), len(words) - 1)
        ids.append(int(words[at]))
        chance.append(w[at] / sums[-1])
    return {"ids": np.array(ids, np.int32), "chance": np.array(chance)}


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    return {"put": _exact_put, "attn": _exact_attn, "sample": _exact_sample}[case["kind"]](prepare(case, seed))
