"""What is timed of the operators that let a batch of conversations try drafted words: every request gets a tree of drafted words
in one step, the model reads all of them at once, and the longest branch that it would have said itself is kept.

Kinds of case:
  plan   which drafted words each one follows, as bit masks, and their positions, from the parents: tree_plan
  attn   attention of every drafted word over the shared prefix, its request's pages and the drafted words it follows: tree_attn
  probs  log probabilities of given words, with the entropy and the likeliest words of each row of scores: word_probs
  take   the branch that the sampled words agree with, the new lengths and the pages that are free again: tree_take
  keep   keys and values of that branch moved to the positions they are kept at: page_keep

With `own` false the same results come from elementary torch operations. `exact` has those that are computed numbers in 64 bits,
request by request and row by row.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # slot A and slot B with a short draft each
        {"name": "plan_pair", "kind": "plan", "n": 2, "nodes": 8, "held": 300},
        # 256 conversations with up to 64 drafted words
        {"name": "plan_batch", "kind": "plan", "n": 256, "nodes": 64, "held": 2000},
        # slot A and slot B behind one short instruction, 12 drafted words: the smallest step, where launches count
        {"name": "attn_pair", "kind": "attn", "n": 2, "n_head": 32, "n_kv": 8, "dim": 64, "page": 16, "type": "f16", "prefix": 90, "own": 75,
         "nodes": 12, "window": 0},
        # one conversation in a long context of odd length on the wide heads, 33 drafted words
        {"name": "attn_long_single", "kind": "attn", "n": 1, "n_head": 16, "n_kv": 4, "dim": 128, "page": 64, "type": "bf16", "prefix": 0, "own": 32749,
         "nodes": 33, "window": 0},
        # the largest step: 64 conversations share 2048 positions, hold up to 2048 each and try up to 64 words
        {"name": "attn_batch", "kind": "attn", "n": 64, "n_head": 32, "n_kv": 8, "dim": 64, "page": 64, "type": "f16", "prefix": 2048, "own": 2048,
         "nodes": 64, "window": 0},
        # the word that one conversation says next, with five alternatives
        {"name": "probs_one", "kind": "probs", "rows": 1, "vocab": 97496, "type": "f32", "words": 1, "top": 5},
        # 61 drafted words over an odd word table in 16 bits: the probabilities of four children each, 20 alternatives
        {"name": "probs_nodes_odd", "kind": "probs", "rows": 61, "vocab": 32003, "type": "bf16", "words": 4, "top": 20},
        # the largest batch's words with eight alternatives
        {"name": "probs_256", "kind": "probs", "rows": 256, "vocab": 97496, "type": "f32", "words": 1, "top": 8},
        # what slot A and slot B keep of 8 drafted words
        {"name": "take_pair", "kind": "take", "n": 2, "nodes": 8, "held": 300, "page": 16},
        # what 256 conversations keep of up to 64
        {"name": "take_batch", "kind": "take", "n": 256, "nodes": 64, "held": 2000, "page": 64},
        # the moves of one layer for slot A and slot B
        {"name": "keep_pair", "kind": "keep", "n": 2, "n_kv": 8, "dim": 64, "page": 16, "type": "f16", "nodes": 12, "held": 45, "taken": 5},
        # the moves of one layer for 256 conversations on the wide heads that keep up to 15 of 64 words
        {"name": "keep_batch", "kind": "keep", "n": 256, "n_kv": 4, "dim": 128, "page": 32, "type": "bf16", "nodes": 64, "held": 301, "taken": 15},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    kind = rng.choice(["plan", "attn", "attn", "attn", "probs", "probs", "take", "keep"])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind in ("plan", "take"):
        n = _log(rng, 1, 1024)
        case = {"kind": kind, "n": n, "nodes": _log(rng, 1, max(1, min(256, 16384 // n))), "held": _log(rng, 1, 4096)}
        return case if kind == "plan" else {**case, "page": page}
    if kind == "probs":
        vocab = _log(rng, 200, 200000)
        return {"kind": kind, "rows": _log(rng, 1, max(1, min(2048, 24000000 // vocab))), "vocab": vocab, "type": rng.choice(["f32", "f32", "f16", "bf16"]),
                "words": rng.choice([0, 1, 1, rng.randint(2, 40)]), "top": rng.choice([0, 1, 5, 20, rng.randint(2, 64)])}
    H, K, D = rng.choice([(32, 8, 64), (16, 4, 128), (8, 2, 32), (12, 4, 64), (7, 1, 128), (6, 6, 64), (20, 1, 64)])
    if kind == "keep":
        nodes = _log(rng, 2, 256)
        return {"kind": kind, "n": _log(rng, 1, 256), "n_kv": K, "dim": D, "page": page, "type": rng.choice(["f16", "bf16"]), "nodes": nodes,
                "held": _log(rng, 1, 300), "taken": rng.randint(1, min(16, (nodes + 1) // 2))}
    n = _log(rng, 1, 64)
    nodes = _log(rng, 1, min(256, 4096 // n))
    return {"kind": kind, "n": n, "n_head": H, "n_kv": K, "dim": D, "page": page, "type": rng.choice(["f16", "bf16"]),
            "prefix": rng.choice([0, _log(rng, 1, 4096), _log(rng, 64, 4096)]), "own": nodes + _log(rng, 1, min(32768, 131072 // n)), "nodes": nodes,
            "window": rng.choice([0, 0, 0, _log(rng, 8, 4096)])}


def draw(rng):
    most = {}
    for case in listed():
        w = work(case)
        most[case["kind"]] = max(most.get(case["kind"], (0, 0)), (w["flops"], w["bytes"]))
    while True:
        case = _drawn(rng)
        w = work(case)
        if w["flops"] <= most[case["kind"]][0] and w["bytes"] <= most[case["kind"]][1]:
            return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _cuda(x, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(x, dtype)).cuda()


def _spread(rng, most, n):
    """n numbers spread evenly over 0 .. most, the largest among them, in an order of the seed's: their sum is the case's own."""
    return rng.permutation(most - np.arange(n) * (most + 1) // n)


def _trees(rng, sizes):
    """Parents of the words of requests of these sizes: chains, bushes and what lies between; the first word of a request has none."""
    parent = np.full(int(sizes.sum()), -1, np.int64)
    at = 0
    for m in sizes.tolist():
        bush = rng.choice([0.0, 0.2, 0.5, 1.0])
        j = np.arange(1, m)
        parent[at + 1:at + m] = np.minimum((rng.random(max(m - 1, 0)) ** bush * j).astype(np.int64), j - 1) if bush else j - 1
        at += m
    return parent


def _starts(sizes):
    return np.concatenate([[0], np.cumsum(sizes)])


def _masks(parent, sizes, most):
    """[rows][words] bit k of a row: it is, or follows, its request's word k."""
    words = (most + 31) // 32
    out = np.zeros((len(parent), words), np.uint32)
    r = 0
    for m in sizes.tolist():
        for j in range(m):
            if parent[r + j] >= 0:
                out[r + j] = out[r + parent[r + j]]
            out[r + j, j >> 5] |= np.uint32(1 << (j & 31))
        r += m
    return out.view(np.int32)


def _pages_of(rng, lens, page, spare=0, pool=0):
    """Tables of shuffled pages for requests of these lengths, and the pages that nobody has (`spare` of them, or what is left of a
    pool of `pool` pages)."""
    counts = (lens + page - 1) // page
    order = rng.permutation(pool or int(counts.sum()) + spare)
    table = np.full((len(lens), max(int(counts.max()), 1)), -1, np.int64)
    table[np.arange(table.shape[1])[None, :] < counts[:, None]] = order[:counts.sum()]
    return table, order[counts.sum():]


def _prepare_plan(case, seed):
    rng = np.random.default_rng(seed)
    sizes = _spread(rng, case["nodes"], case["n"])
    held = rng.integers(1, case["held"] + 1, case["n"])
    rows, words = int(sizes.sum()), (case["nodes"] + 31) // 32
    return {"cu": _cuda(_starts(sizes)), "parent": _cuda(_trees(rng, sizes)), "held": _cuda(held), "length": _cuda(held + sizes), "pos0": 17, "max_rows": case["nodes"],
            "mask": torch.zeros(rows, words, dtype=torch.int32, device="cuda"), "pos": torch.zeros(rows, dtype=torch.int32, device="cuda")}


def _prepare_attn(case, seed):
    rng, g = np.random.default_rng(seed), _generator(seed)
    n, H, K, D, page, L0 = case["n"], case["n_head"], case["n_kv"], case["dim"], case["page"], case["prefix"]
    kind = TYPES[case["type"]]
    sizes = _spread(rng, case["nodes"], n)
    length = np.maximum(sizes, rng.integers(max(1, case["own"] // 8), case["own"] + 1, n))
    table, left = _pages_of(rng, length, page, -(-L0 // page) + 1)
    pages = int((table >= 0).sum()) + len(left)
    rows = int(sizes.sum())
    cache = [torch.randn(pages, K, page, D, generator=g, device="cuda").to(kind) for _ in range(2)]
    q = (2 * torch.randn(rows, H, D, generator=g, device="cuda")).to(kind)
    return {"q": q, "kc": cache[0], "vc": cache[1], "prefix": _cuda(left[:-(-L0 // page)]), "prefix_len": L0, "table": _cuda(table), "length": _cuda(length),
            "cu": _cuda(_starts(sizes)), "mask": _cuda(_masks(_trees(rng, sizes), sizes, case["nodes"])), "max_len": int(length.max()), "max_rows": case["nodes"],
            "window": case["window"], "gate": torch.randn(rows, H, generator=g, device="cuda"), "out": torch.zeros_like(q),
            "lse": torch.zeros(rows, H, device="cuda")}


def _prepare_probs(case, seed):
    g = _generator(seed)
    R, V = case["rows"], case["vocab"]
    scores = 3 * torch.randn(R, V, generator=g, device="cuda")
    sure = torch.randint(0, V, (R, 1), generator=g, device="cuda")      # a word that the model is more or less sure of
    scores.scatter_add_(1, sure, 25 * torch.rand(R, 1, generator=g, device="cuda"))
    scores[::2, torch.rand(V, generator=g, device="cuda") < 0.02] = -math.inf       # words that half of the rows may not say
    temp = 0.5 + torch.rand(R, generator=g, device="cuda")
    if R > 1:
        temp = torch.where(torch.rand(R, generator=g, device="cuda") < 0.1, torch.zeros_like(temp), temp)   # greedy rows among the others
    words = torch.randint(0, V, (R, case["words"]), generator=g, device="cuda", dtype=torch.int32)
    words[:, :1] = torch.where(torch.rand(R, 1, generator=g, device="cuda") < 0.7, sure.int(), words[:, :1])
    return {"scores": scores.to(TYPES[case["type"]]), "temp": temp, "words": words, "logp": torch.zeros(R, case["words"], device="cuda"),
            "entropy": torch.zeros(R, device="cuda"), "top_words": torch.zeros(R, case["top"], dtype=torch.int32, device="cuda"),
            "top_logp": torch.zeros(R, case["top"], device="cuda")}


def _prepare_take(case, seed):
    rng = np.random.default_rng(seed)
    n, page = case["n"], case["page"]
    sizes = _spread(rng, case["nodes"], n)
    held = rng.integers(1, case["held"] + 1, n)
    starts, parent = _starts(sizes), _trees(rng, sizes)
    rows = int(sizes.sum())
    words, picks = rng.integers(0, 97496, rows), rng.integers(0, 97496, rows)
    child = np.flatnonzero((parent >= 0) & (rng.random(rows) < 0.75))      # the model would say three of four drafted words itself
    picks[np.repeat(starts[:-1], sizes)[child] + parent[child]] = words[child]
    table, left = _pages_of(rng, held + sizes, page, pool=n * -(-(case["held"] + case["nodes"]) // page) + 50)
    given = int((table >= 0).sum())
    return {"cu": _cuda(starts), "parent": _cuda(parent), "words": _cuda(words), "picks": _cuda(picks), "held": _cuda(held), "length": _cuda(held + sizes),
            "table": _cuda(table), "page": page, "free": _cuda(np.concatenate([rng.permutation(given), left])), "taken": _cuda([given]),
            "path": torch.zeros(rows, dtype=torch.int32, device="cuda"), "count": torch.zeros(n, dtype=torch.int32, device="cuda"),
            "next": torch.zeros(n, dtype=torch.int32, device="cuda"), "out_len": torch.zeros(n, dtype=torch.int32, device="cuda"),
            "out_taken": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _prepare_keep(case, seed):
    rng, g = np.random.default_rng(seed), _generator(seed)
    n, m, page = case["n"], case["nodes"], case["page"]
    length = rng.integers(1, case["held"] + 1, n) + m
    table, left = _pages_of(rng, length, page, pool=n * -(-(case["held"] + m) // page) + 3)
    path = np.full((n, m), -1)
    for i, c in enumerate(_spread(rng, case["taken"], n).tolist()):
        path[i, :min(c, 1)] = 0             # the first word, then words that no kept one is moved onto: a pass may be repeated
        path[i, 1:c] = np.sort(rng.choice(np.arange(c, m), max(c - 1, 0), replace=False))
    shape = (int((table >= 0).sum()) + len(left), case["n_kv"], page, case["dim"])
    cache = [torch.randn(shape, generator=g, device="cuda").to(TYPES[case["type"]]) for _ in range(2)]
    return {"cu": _cuda(np.arange(n + 1) * m), "path": _cuda(path.reshape(-1)), "length": _cuda(length), "table": _cuda(table), "kc": cache[0], "vc": cache[1]}


def prepare(case, seed):
    make = {"plan": _prepare_plan, "attn": _prepare_attn, "probs": _prepare_probs, "take": _prepare_take, "keep": _prepare_keep}[case["kind"]]
    return {"kind": case["kind"], **make(case, seed)}


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _requests(s, rows):
    """(request, place among the request's rows) of each row, and rows of each request."""
    cu = s["cu"].long()
    sizes = cu[1:] - cu[:-1]
    who = torch.repeat_interleave(torch.arange(sizes.numel(), device="cuda"), sizes, output_size=rows)
    return who, torch.arange(rows, device="cuda") - cu[who], sizes


def _plan(s):
    rows, words = s["mask"].shape
    who, nth, _ = _requests(s, rows)
    parent = s["parent"].long()
    up = torch.where(parent >= 0, parent + s["cu"].long()[who], -1)
    seen = torch.arange(32 * words, device="cuda") == nth[:, None]
    steps = 1
    while steps < s["max_rows"]:            # each turn doubles the words that a row knows it follows
        seen = seen | (seen[up.clamp(min=0)] & (up >= 0)[:, None])
        up = torch.where(up >= 0, up[up.clamp(min=0)], -1)
        steps *= 2
    mask = (seen.view(rows, words, 32).long() << torch.arange(32, device="cuda")).sum(-1)
    return {"mask": torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).int(), "pos": (s["pos0"] + s["held"].long()[who] + seen.sum(1) - 1).int()}


def _rows_of(pages, cache):
    """[n][pages] page ids -> keys or values [n][kv][positions][D] in 32 bits."""
    x = cache[pages.long().clamp(min=0)].float()
    n, P, K, page, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(n, K, P * page, D)


def _attn(s):
    R, H, D = s["q"].shape
    K, n, L0, m, window = s["kc"].shape[1], s["length"].numel(), s["prefix_len"], s["max_rows"], s["window"]
    group, length = H // K, s["length"].long()
    who, nth, sizes = _requests(s, R)
    base = length - sizes
    bits = (s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32) & 1).reshape(R, -1) == 1
    q = torch.zeros(n, m, H, D, device="cuda")
    q[who, nth] = s["q"].float()
    q = q.view(n, m, K, group, D).permute(0, 2, 1, 3, 4).reshape(n, K, m * group, D)
    k, v = _rows_of(s["table"], s["kc"])[:, :, :s["max_len"]], _rows_of(s["table"], s["vc"])[:, :, :s["max_len"]]
    tree = torch.zeros(n, m, bits.shape[1], dtype=torch.bool, device="cuda")
    tree[who, nth] = bits
    depth = tree.sum(-1) - 1
    at = base[:, None] + depth                                                  # [n][m] the rows' own positions
    key = torch.arange(k.shape[2], device="cuda")
    node = key - base[:, None]                                                  # [n][keys] which drafted word a key is
    seen = (node < 0)[:, None] & ((key > at[..., None] - window) if window else torch.ones_like(at, dtype=torch.bool)[..., None])
    drafted = tree.gather(2, node.clamp(0, tree.shape[2] - 1)[:, None].expand(n, m, -1)) & ((node >= 0) & (node < sizes[:, None]))[:, None]
    if window:
        depths = torch.zeros(n, tree.shape[2], dtype=torch.int64, device="cuda")
        depths[:, :m] = depth
        drafted &= (depths.gather(1, node.clamp(0, tree.shape[2] - 1))[:, None] > depth[..., None] - window)
    seen = (seen | drafted).repeat_interleave(group, 1)[:, None]
    score = (torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(D)).masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    if L0:
        k0, v0 = _rows_of(s["prefix"][None], s["kc"])[0, :, :L0], _rows_of(s["prefix"][None], s["vc"])[0, :, :L0]
        q0 = q.permute(1, 0, 2, 3).reshape(K, n * m * group, D)
        score0 = (torch.matmul(q0, k0.transpose(1, 2).contiguous()) / math.sqrt(D)).view(K, n, m * group, L0).permute(1, 0, 2, 3)
        if window:
            left = torch.arange(L0, device="cuda") <= L0 + at[..., None] - window
            score0 = score0.masked_fill(left.repeat_interleave(group, 1)[:, None], -math.inf)
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


def _probs(s):
    x = s["scores"].double()
    greedy = (s["temp"] == 0)[:, None]
    first = x.max(1, keepdim=True).values == x
    first &= first.cumsum(1) == 1                                               # greedy rows: the first of the largest has all
    z = x / torch.where(greedy, torch.ones_like(s["temp"])[:, None], s["temp"][:, None]).double()
    z = torch.where(greedy, torch.where(first, 0.0, -math.inf), z)
    top = z.amax(1, keepdim=True)
    w = torch.exp(z - top)
    total = w.sum(1, keepdim=True)
    logp = z - top - torch.log(total)
    entropy = -(w / total * logp.masked_fill(w == 0, 0.0)).sum(1)
    k = s["top_words"].shape[1]
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    return {"logp": logp.gather(1, s["words"].long()).float(), "entropy": entropy.float(), "top_words": order.int(), "top_logp": logp.gather(1, order).float()}


def _take(s):
    rows, n, page = s["path"].numel(), s["count"].numel(), s["page"]
    who, nth, sizes = _requests(s, rows)
    cu = s["cu"].long()
    there = sizes > 0
    path = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    count = there.long()
    at = torch.zeros(n, dtype=torch.int64, device="cuda")
    row = torch.where(there, cu[:-1], 0)
    if rows:
        path[row[there]] = 0
        going = there
        while going.any():
            child = (s["parent"].long() == at[who]) & (s["words"] == s["picks"][row][who]) & going[who]
            found = torch.full((n,), rows, dtype=torch.int64, device="cuda").scatter_reduce_(0, who, torch.where(child, nth, rows), "amin")
            going = found < rows
            at = torch.where(going, found, at)
            row = torch.where(going, cu[:-1] + at, row)
            path[(cu[:-1] + count)[going]] = at[going]
            count = count + going
    length, out_len = s["length"].long(), s["held"].long() + count
    have, want = (length + page - 1) // page, (out_len + page - 1) // page
    col = torch.arange(s["table"].shape[1], device="cuda")[None, :]
    back = s["table"][(col >= want[:, None]) & (col < have[:, None])]
    taken = s["taken"].long() - back.numel()
    free = s["free"].clone()
    free[taken + torch.arange(back.numel(), device="cuda")] = back
    pick = s["picks"][row] if rows else torch.zeros_like(s["next"])
    return {"path": path.int(), "count": count.int(), "next": torch.where(there, pick, -1).int(), "len": out_len.int(), "free": free, "taken": taken.int()}


def _keep(s):
    rows = s["path"].numel()
    who, nth, sizes = _requests(s, rows)
    page, path = s["kc"].shape[2], s["path"].long()
    moved = path > nth
    base = (s["length"].long() - sizes)[who[moved]]
    source, to = base + path[moved], base + nth[moved]
    table = s["table"].long()
    for cache in (s["kc"], s["vc"]):
        cache[table[who[moved], to // page], :, to % page] = cache[table[who[moved], source // page], :, source % page]
    return {"k": s["kc"], "v": s["vc"]}


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
        s["shape"] = nunchi_amd.PageShape(n_head=s["q"].shape[1] if "q" in s else K, n_kv=K, head_dim=D, page=page, n_pages=pages,
                                          dtype="f16" if s["kc"].dtype == torch.float16 else "bf16", window=s.get("window", 0))
    return s["shape"]


def _own(s):
    import nunchi_amd
    ctx = _context()
    if s["kind"] == "plan":
        nunchi_amd.tree_plan(ctx, s["cu"], s["parent"], s["held"], s["length"], s["mask"], s["pos"], s["max_rows"], pos0=s["pos0"])
        return {"mask": s["mask"], "pos": s["pos"]}
    if s["kind"] == "attn":
        shape = _shape(s)
        if "work" not in s:
            size = nunchi_amd.tree_attn_work(shape, s["length"].numel(), s["q"].shape[0], s["max_len"], s["max_rows"], prefix_len=s["prefix_len"])
            s["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        nunchi_amd.tree_attn(ctx, shape, s["q"], s["kc"], s["vc"], s["table"], s["length"], s["cu"], s["mask"], s["out"], s["work"], s["max_len"],
                             s["max_rows"], prefix=s["prefix"], prefix_len=s["prefix_len"], gate=s["gate"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if s["kind"] == "probs":
        top = s["top_words"].shape[1]
        if "work" not in s:
            s["work"] = torch.empty(nunchi_amd.word_probs_work(*s["scores"].shape, top), dtype=torch.uint8, device="cuda")
        nunchi_amd.word_probs(ctx, s["scores"], s["work"], temp=s["temp"], words=s["words"] if s["words"].shape[1] else None,
                              logp=s["logp"] if s["words"].shape[1] else None, entropy=s["entropy"], top_words=s["top_words"] if top else None,
                              top_logp=s["top_logp"] if top else None)
        return {"logp": s["logp"], "entropy": s["entropy"], "top_words": s["top_words"], "top_logp": s["top_logp"]}
    if s["kind"] == "take":
        nunchi_amd.tree_take(ctx, s["cu"], s["parent"], s["words"], s["picks"], s["held"], s["length"], s["path"], s["count"], s["next"], s["out_len"],
                             table=s["table"], page=s["page"], free=s["free"], taken=s["taken"], taken_out=s["out_taken"])
        return {"path": s["path"], "count": s["count"], "next": s["next"], "len": s["out_len"], "free": s["free"], "taken": s["out_taken"]}
    nunchi_amd.page_keep(ctx, _shape(s), s["cu"], s["path"], s["length"], s["table"], s["kc"], s["vc"])
    return {"k": s["kc"], "v": s["vc"]}


def run(s):
    if own:
        return _own(s)
    return {"plan": _plan, "attn": _attn, "probs": _probs, "take": _take, "keep": _keep}[s["kind"]](s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------


def _rows(case):
    """The sum of _spread's numbers."""
    n, most = case["n"], case["nodes"]
    return sum(most - i * (most + 1) // n for i in range(n))


def work(case):
    kind = case["kind"]
    if kind == "plan":
        rows, words = _rows(case), (case["nodes"] + 31) // 32
        return {"bytes": 12 * case["n"] + rows * (8 + 4 * words), "flops": rows}
    if kind == "attn":
        H, K, D, L0, win = case["n_head"], case["n_kv"], case["dim"], case["prefix"], case["window"]
        rows, held = _rows(case), case["own"] * 9 / 16
        seen0, seen, read0, read = L0, max(1, held - case["nodes"] / 4), L0, held
        if win:
            seen, read = min(seen, win), min(read, win + case["nodes"])
            seen0 = read0 = min(L0, max(0, win - seen))
        return {"bytes": 4.0 * K * D * (read0 + case["n"] * read) + rows * (H * (4 * D + 8) + 4 * ((case["nodes"] + 31) // 32)),
                "flops": 4.0 * rows * H * D * (seen0 + seen)}
    if kind == "probs":
        return {"bytes": case["rows"] * (case["vocab"] * SIZE[case["type"]] + 8 + 8 * case["words"] + 8 * case["top"]), "flops": 5.0 * case["rows"] * case["vocab"]}
    if kind == "take":
        rows = _rows(case)
        return {"bytes": 28 * case["n"] + 16 * rows, "flops": rows}
    n, c = case["n"], case["taken"]
    moved = sum(max(0, c - i * (c + 1) // n - 1) for i in range(n))
    return {"bytes": 8.0 * moved * case["n_kv"] * case["dim"] + 8 * n + 4 * n * case["nodes"], "flops": moved}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _exact_attn(s):
    R, H, D = s["q"].shape
    K, L0, window = s["kc"].shape[1], s["prefix_len"], s["window"]
    out, lse = torch.zeros(R, H, D, dtype=torch.float64), torch.zeros(R, H, dtype=torch.float64)
    out, lse = out.cuda(), lse.cuda()
    starts, words = s["cu"].tolist(), s["mask"].cpu().numpy().view(np.uint8)
    page = s["kc"].shape[2]

    def gather(cache, i, held):
        ids = torch.cat([s["prefix"], s["table"][i, :-(-held // page)]]).long()
        x = cache[ids].double().transpose(1, 2).reshape(-1, K, D)
        return torch.cat([x[:L0], x[s["prefix"].numel() * page:][:held]])

    for i, held in enumerate(s["length"].tolist()):
        r0, r1 = starts[i], starts[i + 1]
        m = r1 - r0
        if m == 0:
            continue
        k, v = gather(s["kc"], i, held), gather(s["vc"], i, held)
        follows = np.unpackbits(words[r0:r1], axis=1, bitorder="little")[:, :m].astype(bool)
        depth = follows.sum(1) - 1
        before = L0 + held - m
        where = np.concatenate([np.arange(before), before + depth])             # the position of each key
        see = np.concatenate([np.ones((m, before), bool), follows], 1)
        if window:
            see &= where[None] > (before + depth)[:, None] - window
        see = torch.from_numpy(see).cuda()
        for g in range(K):
            heads = slice(g * (H // K), (g + 1) * (H // K))
            q = s["q"][r0:r1, heads].double()
            z = (q.reshape(-1, D) @ k[:, g].T.contiguous()).view(m, H // K, -1) / math.sqrt(D)
            z = z.masked_fill(~see[:, None], -math.inf)
            lse[r0:r1, heads] = torch.logsumexp(z, -1)
            out[r0:r1, heads] = (torch.softmax(z, -1).view(-1, L0 + held) @ v[:, g].contiguous()).view(m, -1, D)
    return {"out": out / (1 + torch.exp(-s["gate"].double()))[..., None], "lse": lse}


def _exact_probs(s):
    logp, entropy, best, best_logp = [], [], [], []
    k = s["top_words"].shape[1]
    for x, temp, words in zip(s["scores"].double().cpu().numpy(), s["temp"].double().cpu().numpy(), s["words"].cpu().numpy()):
        order = np.argsort(-x, kind="stable")
        if temp == 0:
            lp = np.full(len(x), -np.inf)
            lp[order[0]] = 0.0
            entropy.append(0.0)
        else:
            z = (x - x[order[0]]) / temp
            rest = np.exp(z[order[1:]])[::-1].sum()                             # all but the likeliest word's 1
            lp = z - np.log1p(rest)
            p = np.exp(lp)
            entropy.append(np.log1p(rest) - (p[p > 0] * z[p > 0]).sum())
        logp.append(lp[words])
        best.append(order[:k])
        best_logp.append(lp[order[:k]])
    return {"logp": np.stack(logp), "entropy": np.array(entropy), "top_words": np.stack(best).astype(np.int32), "top_logp": np.stack(best_logp)}


def exact(case, seed):
    """None for what is whole numbers or copies."""
    if case["kind"] not in ("attn", "probs"):
        return None
    return {"attn": _exact_attn, "probs": _exact_probs}[case["kind"]](prepare(case, seed))
