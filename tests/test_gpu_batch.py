"""The operators that serve a batch of conversations (sh_page_plan, sh_page_put, sh_page_attn, sh_sample) against plain
implementations in 64 bits on the CPU.

Tolerances count roundings. HALF is half a step of a 16-bit type relative to the value; single precision rounds by 2^-24.
 put:  one rounding to the type, on top of single precision norms (the sum of D squares D / 16 + 4 roundings deep, halved
       by the root; root, division and two products) and rotations (two products and a sum, each on values below sqrt(2)
       times the head's largest): below 20 roundings of 2^-24 on sqrt(2) times the largest, under 2^-19 of it.
 attn: weights are rounded to the type (HALF of each, so HALF of the largest visible value at most), fp16 weights below
       2^-14 to 2^-25 against a largest one of at least 1 (2^-25 per key), the output once more (HALF); the scores' error
       in single precision (below) moves the weights by as much twice (once in the sum).
 lse:  a score is a sum of D products in single precision (D 2^-24 of the sum of their sizes at most, 16-bit products are
       exact in it), scaled (2^-24) and, in powers of two, held to 2^-24 of its size; the sum of n weights adds n / 128 + 16
       roundings (eight keys a lane at a time, joined in order), each 2^-24, the two hardware exponentials and the logarithm
       2^-22 each.
 sample: ids are equal; the chance is a weight (2^-23) over an exact sum of such weights (2^-23 at most), rounded once.
"""
import math
import threading

import numpy as np
import pytest

import nunchi_amd
from conftest import ROOT  # noqa: F401  (the repository's root in sys.path)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def ctx():
    return nunchi_amd.Context(0, stream=torch.cuda.current_stream().cuda_stream)


def dev(x, dtype=None):
    return torch.as_tensor(x, dtype=dtype).cuda()


def i32(x):
    return dev(np.asarray(x, np.int32))


# ---------------------------------------------------------------- block tables and slot maps


def plan_reference(held, add, page, table, free, taken, rows, pos0):
    n, cols = table.shape
    table = table.copy()
    taken, start, cu = max(int(taken), 0), 0, 0
    out_taken = taken
    length, starts = [], [0]
    slots, pos = np.full(rows, -7, np.int64), np.full(rows, -7, np.int64)
    for i in range(n):
        h, a = int(held[i]), int(add[i])
        more = max(a, 0)
        ok = h >= 0 and a >= 0 and -(-(h + a) // page) <= cols and h + a < 2 ** 31
        need = -(-(h + a) // page) - -(-h // page) if ok else 0
        fits = ok and cu + more <= rows and (need == 0 or taken + start + need <= len(free))
        if fits and need:
            have = -(-h // page)
            table[i, have:have + need] = free[taken + start:taken + start + need]
            out_taken = taken + start + need
        for t in range(more):
            if cu + t >= rows:
                break
            p = h + t
            slots[cu + t] = table[i, p // page] * page + p % page if fits and table[i, p // page] >= 0 else -1
            pos[cu + t] = min(pos0 + p, 2 ** 31 - 1)
        length.append(h + a if fits else h)
        start += need
        cu += more
        starts.append(min(cu, 2 ** 31 - 1))
    return {"table": table, "len": length, "cu": starts, "slots": slots, "pos": pos, "taken": [out_taken]}


def run_plan(ctx, held, add, page, table, free, taken, rows, pos0=0):
    n = len(held)
    t = {"table": i32(table), "len": i32(np.full(n, -7)), "cu": i32(np.full(n + 1, -7)), "taken": i32([-7]),
         "slots": dev(np.full(rows, -7, np.int64)), "pos": i32(np.full(rows, -7))}
    nunchi_amd.page_plan(ctx, i32(held), i32(add), i32(free), i32([taken]), t["table"], page, t["len"], t["cu"], t["slots"], t["pos"], t["taken"], pos0=pos0)
    torch.cuda.synchronize()
    return t


def check_plan(ctx, held, add, page, table, free, taken, rows, pos0=0):
    want = plan_reference(held, add, page, table, free, taken, rows, pos0)
    got = run_plan(ctx, held, add, page, table, free, taken, rows, pos0)
    for k, v in want.items():
        assert np.array_equal(got[k].cpu().numpy(), np.asarray(v)), k


def plan_case(seed, n, page, most_held, most_add, spare=0):
    rng = np.random.default_rng(seed)
    held, add = rng.integers(0, most_held + 1, n), rng.integers(0, most_add + 1, n)
    have, want = -(-held // page), -(-(held + add) // page)
    cols = max(1, int(want.max()))
    ids = rng.permutation(int(want.sum()) + 5 + spare)
    table = np.full((n, cols), -1)
    at = 0
    for i in range(n):
        table[i, :have[i]] = ids[at:at + have[i]]
        at += have[i]
    return held, add, table, ids[at:]


@pytest.mark.parametrize("n,page,held,add", [(1, 16, 0, 1), (1, 16, 40, 0), (2, 16, 15, 1), (3, 32, 31, 33), (64, 64, 300, 1), (255, 16, 100, 5),
                                             (256, 16, 100, 70), (3, 16, 40, 5), (5, 16, 100, 27), (2, 16, 3, 9000), (257, 128, 1000, 300), (1000, 256, 700, 3), (4096, 16, 60, 9)])
def test_plan(ctx, n, page, held, add):
    h, a, table, free = plan_case(n * page, n, page, held, add)
    check_plan(ctx, h, a, page, table, free, 2, int(a.sum()), pos0=11)


def test_plan_boundaries(ctx):
    """Lengths on, one before and one behind a page's end; requests that add nothing; a first request without rows."""
    held = np.array([0, 0, 15, 16, 17, 31, 32, 16, 0])
    add = np.array([0, 16, 1, 1, 15, 1, 0, 17, 1])
    table = np.arange(9 * 4).reshape(9, 4)
    check_plan(ctx, held, add, 16, table, np.arange(100, 120), 0, int(add.sum()))


def test_plan_refuses_requests_one_by_one(ctx):
    """Negative lengths, too many pages, too few free pages, too few rows, and entries of -1 in a table."""
    held = np.array([3, -1, 5, 4, 60, 0, 2 ** 31 - 1, 10])
    add = np.array([14, 4, -2, 2 ** 30, 5, 0, 1, 20])
    table = np.full((8, 4), -1)
    table[[0, 3, 4, 7], 0] = [7, 8, 9, 6]
    for rows in (0, 3, 14, 18, 60):
        for taken in (-4, 0, 9, 10, 11, 400):
            check_plan(ctx, held[:3], add[:3], 16, table[:3], np.arange(50, 61), taken, rows)
            check_plan(ctx, held[[0, 1, 2, 4, 5, 7]], add[[0, 1, 2, 4, 5, 7]], 16, table[[0, 1, 2, 4, 5, 7]], np.arange(50, 61), taken, rows, pos0=2 ** 31 - 5)


def test_plan_row_sums_past_32_bits(ctx):
    """Two requests of 2^30 and one of 2^31 - 1 rows: refused, the sums stay at the largest 32-bit number; the rows that are
    there have no slots."""
    add = [5, 2 ** 30, 2 ** 30, 2 ** 31 - 1, 3]
    got = run_plan(ctx, [0] * 5, add, 16, np.zeros((5, 4)), np.arange(9), 0, 40)
    assert got["cu"].tolist() == [0, 5, 5 + 2 ** 30, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]
    assert got["len"].tolist() == [5, 0, 0, 0, 0]
    assert got["slots"].tolist() == [0, 1, 2, 3, 4] + [-1] * 35
    assert got["taken"].tolist() == [1]


def test_plan_slots_pass_32_bits(ctx):
    got = run_plan(ctx, [256], [3], 256, np.array([[2 ** 31 - 1, -1]]), [2 ** 31 - 2], 0, 3)
    assert got["slots"].tolist() == [(2 ** 31 - 2) * 256 + k for k in range(3)]


def test_plan_leaves_what_is_behind(ctx):
    got = run_plan(ctx, [0, 4], [2, 1], 16, np.array([[3, 3], [4, 4]]), [9], 0, 7)
    assert got["slots"].tolist() == [144, 145, 68, -7, -7, -7, -7] and got["pos"].tolist() == [0, 1, 4, -7, -7, -7, -7]
    assert got["table"].tolist() == [[9, 3], [4, 4]]


# ---------------------------------------------------------------- the write of a step's positions


def heads_reference(x, w, eps, cs):
    """[rows][heads][D] in 64 bits."""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if cs is None:
        return x
    a, b = x.chunk(2, -1)
    c, s = cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def put_case(seed, rows, H, K, D, page, src, kind, extra=0, skew=0, positions=50):
    g = torch.Generator().manual_seed(seed)
    ld = (H + 2 * K) * D + extra
    flat = torch.randn(rows * ld + skew, generator=g).to(TYPES[src]).cuda()
    pages = -(-(rows + 3) // page)
    ang = torch.rand(positions, D // 2, generator=g) * 6.28
    return {"qkv": flat[skew:].view(rows, ld), "slots": torch.randperm(pages * page, generator=g)[:rows].cuda(),
            "pos": torch.randint(0, positions, (rows,), generator=g, dtype=torch.int32).cuda(), "rope": torch.stack([ang.cos(), ang.sin()], -1).cuda(),
            "q_norm": (1 + 0.2 * torch.randn(D, generator=g)).cuda(), "k_norm": (1 + 0.2 * torch.randn(D, generator=g)).cuda(),
            "keys": torch.randn(pages, K, page, D, generator=g).to(TYPES[kind]).cuda(), "values": torch.randn(pages, K, page, D, generator=g).to(TYPES[kind]).cuda(),
            "q": torch.full((rows, H, D), 7.0, dtype=TYPES[kind], device="cuda"),
            "shape": nunchi_amd.PageShape(H, K, D, page, pages, dtype=kind), "dims": (rows, H, K, D, page), "kind": kind}


def put_reference(c, norms=True, rope=True):
    rows, H, K, D, page = c["dims"]
    x = c["qkv"].cpu().double()[:, :(H + 2 * K) * D].reshape(rows, -1, D)
    cs = c["rope"].cpu()[c["pos"].cpu().long().clamp(0, c["rope"].shape[0] - 1)] if rope else None
    q = heads_reference(x[:, :H], c["q_norm"].cpu() if norms else None, 1e-5, cs)
    k = heads_reference(x[:, H:H + K], c["k_norm"].cpu() if norms else None, 1e-5, cs)
    return q, k, x[:, H + K:]


def check_put(ctx, c, norms=True, rope=True, with_q=True):
    rows, H, K, D, page = c["dims"]
    q, k, v = put_reference(c, norms, rope)
    keys, values = c["keys"].cpu().double(), c["values"].cpu().double()
    ok = torch.ones(rows, dtype=torch.bool)
    if rope:
        ok = (c["pos"].cpu() >= 0) & (c["pos"].cpu() < c["rope"].shape[0])
        q = torch.where(ok[:, None, None], q, torch.zeros_like(q))
    for r, slot in enumerate(c["slots"].tolist()):
        if ok[r] and 0 <= slot < keys.shape[0] * page:
            keys[slot // page, :, slot % page], values[slot // page, :, slot % page] = k[r], v[r]
    nunchi_amd.page_put(ctx, c["shape"], c["qkv"], c["slots"], c["keys"], c["values"], q=c["q"] if with_q else None, pos=c["pos"],
                        q_norm=c["q_norm"] if norms else None, k_norm=c["k_norm"] if norms else None, rope=c["rope"] if rope else None)
    torch.cuda.synchronize()
    assert torch.equal(c["values"].cpu(), values.to(TYPES[c["kind"]])), "values are rounded once, exactly"
    for got, want in [(c["keys"], keys)] + ([(c["q"], q)] if with_q else []):
        got = got.cpu().double()
        tol = HALF[c["kind"]] * want.abs() + 2.0 ** -25 + 2.0 ** -19 * want.abs().amax(-1, keepdim=True) * math.sqrt(2)
        worst = ((got - want).abs() - tol).max().item()
        assert worst <= 0, worst


@pytest.mark.parametrize("rows,H,K,D,page,src,kind,extra", [
    (1, 8, 2, 64, 16, "f32", "f16", 8), (5, 32, 8, 64, 64, "f32", "f16", 32), (3, 16, 4, 128, 32, "bf16", "bf16", 0), (17, 7, 1, 128, 16, "f32", "bf16", 7),
    (33, 6, 6, 64, 256, "f16", "f16", 1), (2, 8, 2, 32, 128, "f16", "bf16", 0), (129, 1, 1, 32, 16, "bf16", "f16", 3), (1000, 12, 4, 64, 16, "f32", "f16", 12)])
def test_put(ctx, rows, H, K, D, page, src, kind, extra):
    check_put(ctx, put_case(rows + D, rows, H, K, D, page, src, kind, extra))


@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("skew", [1, 3])
def test_put_rows_that_start_anywhere(ctx, src, skew):
    check_put(ctx, put_case(5, 9, 4, 2, 64, 16, src, "f16", extra=skew, skew=skew))


@pytest.mark.parametrize("norms,rope,with_q", [(False, True, True), (True, False, True), (False, False, False)])
def test_put_without_norms_rotation_or_queries(ctx, norms, rope, with_q):
    check_put(ctx, put_case(6, 20, 8, 2, 64, 16, "f32", "bf16"), norms, rope, with_q)


def test_put_slots_and_positions_out_of_range(ctx):
    """Rows without a place, behind the cache, or at positions that the rotation table does not have."""
    c = put_case(7, 12, 4, 2, 64, 16, "f32", "f16")
    c["slots"][:4] = torch.tensor([-1, 16 * c["keys"].shape[0], 2 ** 40, -2 ** 40])
    c["pos"][5:8] = torch.tensor([-1, 50, 2 ** 31 - 1], dtype=torch.int32)
    check_put(ctx, c)


def test_put_values_that_overflow_and_nan(ctx):
    c = put_case(8, 4, 2, 1, 32, 16, "f32", "f16")
    v = c["qkv"].view(4, 4, 32)
    v[0, 3, 5], v[1, 3, 6], v[2, 3, 7] = 1e6, -math.inf, math.nan
    nunchi_amd.page_put(ctx, c["shape"], c["qkv"], c["slots"], c["keys"], c["values"], q=c["q"], pos=c["pos"], q_norm=c["q_norm"], k_norm=c["k_norm"], rope=c["rope"])
    got = [c["values"][s // 16, 0, s % 16].cpu() for s in c["slots"].tolist()]
    assert got[0][5] == math.inf and got[1][6] == -math.inf and math.isnan(got[2][7])
    for r in range(4):
        keep = torch.ones(32, dtype=torch.bool)
        keep[4 + r + 1 if r < 3 else 0] = r == 3
        assert torch.equal(got[r][keep], v[r, 3].cpu().half()[keep])


# ---------------------------------------------------------------- attention


def attn_case(seed, lens, H, K, D, page, kind, prefix=0, add=None, window=0, gate=True, scale=0.0, gain=1.0, max_len=None, cols=None, extra_rows=0):
    """Requests of these lengths in shuffled pages behind a shared prefix; everything that no request may see is NaN."""
    g = torch.Generator().manual_seed(seed)
    n = len(lens)
    pages = [-(-h // page) for h in lens]
    np_pages = -(-prefix // page)
    total = sum(pages) + np_pages + 2
    ids = torch.randperm(total, generator=g).tolist()
    dtype = TYPES[kind]
    keys, values = (torch.full((total, K, page, D), math.nan, dtype=dtype) for _ in range(2))

    def fill(where, count):
        for p, pid in enumerate(where):
            m = min(page, count - p * page)
            keys[pid, :, :m] = torch.randn(K, m, D, generator=g).to(dtype)
            values[pid, :, :m] = torch.randn(K, m, D, generator=g).to(dtype)

    shared, at = ids[:np_pages], np_pages
    fill(shared, prefix)
    width = max(max(pages), 1) if cols is None else cols
    table = torch.full((n, width), -1, dtype=torch.int32)
    for i in range(n):
        mine = ids[at:at + pages[i]]
        at += pages[i]
        fill(mine, lens[i])
        table[i, :pages[i]] = torch.tensor(mine, dtype=torch.int32)
    counts = [1] * n if add is None else add
    rows = sum(counts)
    q = (gain * torch.randn(rows + extra_rows, H, D, generator=g)).to(dtype)
    cu = None if add is None else torch.tensor([sum(counts[:k]) for k in range(n + 1)], dtype=torch.int32).cuda()
    return {"q": q.cuda(), "keys": keys.cuda(), "values": values.cuda(), "shared": torch.tensor(shared, dtype=torch.int32).cuda(), "prefix": prefix,
            "table": table.cuda(), "lens": list(lens), "length": i32(lens), "counts": counts, "cu": cu, "max_rows": max(max(counts), 1) if add else 1,
            "max_len": max(max(lens), 0) if max_len is None else max_len, "gate": torch.randn(rows + extra_rows, H, generator=g).cuda() if gate else None,
            "out": torch.full((rows + extra_rows, H, D), 7.0, dtype=dtype, device="cuda"), "lse": torch.full((rows + extra_rows, H), 7.0, device="cuda"),
            "shape": nunchi_amd.PageShape(H, K, D, page, total, dtype=kind, window=window, scale=scale), "dims": (H, K, D, page), "kind": kind,
            "window": window, "scale": scale or 1 / math.sqrt(D), "rows": rows}


def run_attn(ctx, c, work=None):
    rows = c["q"].shape[0]
    size = nunchi_amd.page_attn_work(c["shape"], len(c["lens"]), rows, c["max_len"], c["max_rows"], c["prefix"])
    work = torch.full((size,), 255, dtype=torch.uint8, device="cuda") if work is None else work    # (NaN in every part)
    nunchi_amd.page_attn(ctx, c["shape"], c["q"], c["keys"], c["values"], c["table"], c["length"], c["out"], work, c["max_len"], cu=c["cu"],
                         max_rows=c["max_rows"], prefix=c["shared"], prefix_len=c["prefix"], gate=c["gate"], lse=c["lse"])
    return c["out"], c["lse"]


def attn_reference(c):
    """(out, lse, tolerance of out, of lse) in 64 bits, request by request and key by key position."""
    H, K, D, page = c["dims"]
    keys, values, q = (c[k].cpu().double() for k in ("keys", "values", "q"))
    rows = c["rows"]
    out, lse = torch.zeros(rows, H, D, dtype=torch.float64), torch.full((rows, H), -math.inf, dtype=torch.float64)
    tol, tol_lse = torch.zeros(rows, H, 1, dtype=torch.float64), torch.zeros(rows, H, dtype=torch.float64)
    table, shared = c["table"].tolist(), c["shared"].tolist()
    r0 = 0
    for i, held in enumerate(c["lens"]):
        held = max(held, 0)
        places = [(shared[p // page], p % page, p) for p in range(c["prefix"])] + \
                 [(table[i][p // page], p % page, c["prefix"] + p) for p in range(held)]
        places = [x for x in places if 0 <= x[0] < keys.shape[0]]
        for r in range(r0, r0 + c["counts"][i]):
            own = held - c["counts"][i] + (r - r0)
            me = c["prefix"] + own
            seen = [(a, b) for a, b, p in places if (p < c["prefix"] or p <= me) and (not c["window"] or p > me - c["window"])]
            if not seen:
                continue
            a, b = torch.tensor([x[0] for x in seen]), torch.tensor([x[1] for x in seen])
            k, v = keys[a, :, b], values[a, :, b]                        # [keys][K][D]
            k, v = k.repeat_interleave(H // K, 1), v.repeat_interleave(H // K, 1)
            s = (q[r][None] * k).sum(-1) * c["scale"]                    # [keys][H]
            size = (q[r][None] * k).abs().sum(-1).amax(0) * c["scale"]
            top = s.amax(0)
            e = torch.exp(s - top)
            lse[r] = top + torch.log(e.sum(0))
            out[r] = (e / e.sum(0))[..., None].mul(v).sum(0)
            off = 2.0 ** -24 * (D * size + 3 * s.abs().amax(0) / math.log(2) + len(seen) / 128 + 16) + 2.0 ** -20
            tol_lse[r] = off + 2.0 ** -23 * lse[r].abs()
            h = HALF[c["kind"]]
            big = v.abs().amax(0).amax(-1)
            # (f16 weights are 2^11 of the running maximum's: below 2^-14 their places are 2^-24 apart)
            under = 2.0 ** -36 * len(seen) if c["kind"] == "f16" else 0.0
            tol[r, :, 0] = (h * 1.01 + under + 2 * off) * big
        r0 += c["counts"][i]
    if c["gate"] is not None:
        f = torch.sigmoid(c["gate"].cpu().double()[:rows])[..., None]
        out, tol = out * f, tol * f
    return out, lse, tol + HALF[c["kind"]] * out.abs() + 2.0 ** -25, tol_lse


def check_attn(ctx, c):
    out, lse = run_attn(ctx, c)
    want, want_lse, tol, tol_lse = attn_reference(c)
    rows = c["rows"]
    got, got_lse = out.cpu().double(), lse.cpu().double()
    assert torch.isfinite(got[:rows]).all()
    assert ((got[:rows] - want).abs() <= tol).all(), ((got[:rows] - want).abs() - tol).max().item()
    none = want_lse == -math.inf
    assert torch.equal(got_lse[:rows] == -math.inf, none)
    assert (got[:rows][none] == 0).all()
    assert ((got_lse[:rows] - want_lse).abs()[~none] <= tol_lse[~none]).all(), ((got_lse[:rows] - want_lse).abs() - tol_lse)[~none].max().item()
    assert (got[rows:] == 7).all() and (got_lse[rows:] == 7).all(), "rows behind the last request's"


EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 160]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("H,K,D,page", [(8, 2, 64, 16), (8, 2, 32, 32), (16, 4, 128, 16), (6, 6, 64, 64), (7, 1, 128, 256), (20, 1, 64, 16), (36, 2, 128, 32), (40, 1, 32, 128)])
def test_attn_lengths(ctx, H, K, D, page, kind):
    """One row per request, lengths on either side of every block, page and part edge, nothing shared."""
    check_attn(ctx, attn_case(H * D + page, EDGES, H, K, D, page, kind))


@pytest.mark.parametrize("H,K,D,page,kind", [(8, 2, 64, 16, "f16"), (16, 4, 128, 32, "bf16"), (8, 2, 32, 64, "f16"), (20, 1, 64, 128, "bf16")])
@pytest.mark.parametrize("prefix", [1, 16, 31, 100, 257, 700])
def test_attn_shared_prefix(ctx, H, K, D, page, kind, prefix):
    check_attn(ctx, attn_case(prefix, [1, 40, 17, 0, 130], H, K, D, page, kind, prefix=prefix))


@pytest.mark.parametrize("H,K,D,page,kind", [(8, 2, 64, 16, "f16"), (16, 4, 128, 32, "bf16"), (4, 1, 32, 16, "bf16"), (32, 8, 64, 64, "f16")])
@pytest.mark.parametrize("prefix,window", [(0, 0), (37, 0), (0, 9), (50, 40), (300, 1), (10, 33)])
def test_attn_prompts(ctx, H, K, D, page, kind, prefix, window):
    """Several rows per request (none, one, odd numbers), causal among themselves, some behind positions held before."""
    check_attn(ctx, attn_case(prefix + window, [5, 70, 0, 33, 90, 1], H, K, D, page, kind, prefix=prefix, add=[5, 33, 0, 1, 47, 1], window=window))


@pytest.mark.parametrize("window", [1, 2, 16, 31, 64, 100, 1000])
def test_attn_windows(ctx, window):
    check_attn(ctx, attn_case(window, [1, 60, 128, 200, 0], 8, 2, 64, 16, "f16", prefix=90, window=window))


@pytest.mark.parametrize("n,length,prefix", [(1, 3000, 0), (2, 1111, 2500), (40, 300, 1100)])
def test_attn_many_parts(ctx, n, length, prefix):
    check_attn(ctx, attn_case(n, [length - 7 * i for i in range(n)], 4, 2, 64, 64, "f16", prefix=prefix))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attn_finds_one_key_anywhere(ctx, kind):
    """One key that outweighs all others by e^30, at the edges of blocks, pages and parts: the output is its value."""
    H, K, D, page, n = 4, 1, 64, 32, 1500
    c = attn_case(3, [n], H, K, D, page, kind, prefix=700, gate=False)
    c["q"][:] = 0
    c["q"][:, :, 0] = 8.0
    c["keys"][..., 0] = torch.where(c["keys"][..., 0].isnan(), c["keys"][..., 0], torch.zeros_like(c["keys"][..., 0]))
    table, shared = c["table"][0].tolist(), c["shared"].tolist()
    for p in [0, 31, 32, 255, 256, 511, 699, 700, 701, 955, 956, 1000, 1211, 1212, 1700, 2198, 2199]:
        pid, o = (shared[p // page], p % page) if p < 700 else (table[(p - 700) // page], (p - 700) % page)
        c["keys"][pid, 0, o, 0] = 30.0
        out, lse = run_attn(ctx, c)
        want = c["values"][pid, 0, o].float()
        # the others' weights: 2199 e^-30 in all
        assert ((out[0].float() - want).abs() <= 2 * HALF[kind] * want.abs() + 2.0 ** -25 + 2200 * math.exp(-30) * 6).all(), p
        assert abs(lse[0, 0].item() - 30.0) < 1e-5
        c["keys"][pid, 0, o, 0] = 0.0


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attn_many_small_weights(ctx, kind):
    """20000 keys of weights 2^-25.5 of the largest, whose value is 0: the output is the small ones' sum. Each weight is
    rounded by half a step (h, or 2^-25 below 2^-14 in f16: here 2^-25.5 + 11), the result by h."""
    N, n, page = 20000, 512, 16
    pages = N // page
    keys, values = torch.zeros(pages, 2, page, 64, dtype=TYPES[kind], device="cuda"), torch.ones(pages, 2, page, 64, dtype=TYPES[kind], device="cuda")
    q = torch.zeros(n, 2, 64, dtype=TYPES[kind], device="cuda")
    q[..., 0] = 1
    keys[700, :, 5, 0] = 17.625
    values[700, :, 5] = 0
    shape = nunchi_amd.PageShape(2, 2, 64, page, pages, dtype=kind, scale=1.0)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(n, 1)       # (all requests read the same pages)
    out, work = torch.empty_like(q), torch.empty(nunchi_amd.page_attn_work(shape, n, n, N), dtype=torch.uint8, device="cuda")
    nunchi_amd.page_attn(ctx, shape, q, keys, values, table, i32([N] * n), out, work, N)
    e = math.exp(-keys[700, 0, 5, 0].item())
    want = (N - 1) * e / (1 + (N - 1) * e)
    assert ((out.double() / want - 1).abs() <= 2 * HALF[kind] + 2.0 ** -25 / 2.0 ** -14.5 + 2.0 ** -19).all(), out.double().mean().item() / want


def test_attn_windows_of_any_length(ctx):
    """A window that passes every position leaves nothing out, also for rows whose request holds less than them."""
    for window in (2 ** 31 - 1, 2 ** 31 - 200, 290, 291):
        check_attn(ctx, attn_case(21, [0, 200], 8, 2, 64, 16, "f16", prefix=90, add=[200, 30], window=window))


def test_attn_large_scores(ctx):
    """Scores of up to several hundred that grow along the keys: the running maximum moves in every block."""
    c = attn_case(11, [200, 131], 8, 2, 64, 16, "f16", prefix=150, gain=20.0)
    order = c["keys"].float()
    order *= (torch.arange(order.shape[0], device="cuda") + 1)[:, None, None, None] / order.shape[0]
    c["keys"][:] = order.half()
    check_attn(ctx, c)


def test_attn_scale_and_no_gate(ctx):
    check_attn(ctx, attn_case(12, [50, 9], 8, 2, 64, 16, "f16", prefix=20, scale=0.37, gate=False))
    check_attn(ctx, attn_case(12, [50, 9], 8, 2, 64, 16, "f16", prefix=20, scale=1e-45, gate=False))


def test_attn_rows_that_see_nothing(ctx):
    """No shared positions and a length of zero (or below): zeros and -inf, alone and among others."""
    c = attn_case(13, [0, 20, 0], 8, 2, 64, 16, "f16")
    check_attn(ctx, c)
    c = attn_case(14, [0], 8, 2, 64, 16, "bf16", cols=1)
    c["length"] = i32([-5])
    check_attn(ctx, c)


def test_attn_bad_pages_are_not_there(ctx):
    """Page ids below zero and past the cache, shared and own, at the start, between and at the end: their keys do not count."""
    for page in (16, 32):
        c = attn_case(15, [70, 100, 40], 8, 2, 64, page, "f16", prefix=80)
        c["table"][0, 0], c["table"][1, 1], c["table"][2, (40 - 1) // page], c["shared"][1] = -1, c["shape"].n_pages, 2 ** 31 - 1, -2 ** 31
        check_attn(ctx, c)
    c = attn_case(16, [10, 10], 8, 2, 64, 16, "f16")
    c["table"][0, 0] = -9
    check_attn(ctx, c)


def test_attn_lengths_past_the_table_and_max_len(ctx):
    """A length past max_len counts as max_len, one past the table's columns as the columns' positions."""
    c = attn_case(17, [64, 64], 8, 2, 64, 16, "f16")
    c["length"] = i32([2 ** 31 - 1, 64])
    check_attn(ctx, c)
    c["max_len"] = 48
    c["lens"] = [48, 48]
    check_attn(ctx, c)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("prefix,window", [(0, 0), (40, 0), (40, 24)])
def test_attn_bad_values_reach_only_rows_that_see_them(ctx, kind, bad, prefix, window):
    """An infinity or NaN among the values (and, for NaN, the keys) of one position: rows before it, and rows whose window
    has left it behind, are what they are without it; rows that see it get it."""
    add, at = 40, 21
    c = attn_case(18, [60], 8, 2, 64, 16, kind, prefix=prefix, add=[add], window=window, gate=False)
    out, _ = run_attn(ctx, c)
    clean = out.clone()
    pid, o = int(c["table"][0, at // 16]), at % 16
    c["values"][pid, :, o, 5] = bad
    spread = math.isnan(bad)
    if spread:
        c["keys"][pid, :, o, 3] = bad
    out, lse = run_attn(ctx, c)
    for r in range(add):
        me = 60 - add + r
        sees = me >= at and (not window or at > me - window)
        dims = torch.ones(64, dtype=torch.bool, device="cuda")
        dims[5] = False
        if sees:
            assert (out[r, :, 5].isnan() if spread else out[r, :, 5] == bad).all(), r
            assert spread or torch.equal(out[r][:, dims], clean[r][:, dims]), r
        else:
            assert torch.equal(out[r], clean[r]), r


def test_attn_bad_prefix_values_with_a_window(ctx):
    """The same in the shared positions, which rows of different requests leave behind at different places."""
    c = attn_case(19, [3, 30, 55, 80], 8, 2, 64, 16, "f16", prefix=70, window=64, gate=False)
    clean = run_attn(ctx, c)[0].clone()
    at = 66
    c["values"][int(c["shared"][at // 16]), :, at % 16, 9] = math.inf
    out, _ = run_attn(ctx, c)
    for r, held in enumerate(c["lens"]):
        if at > 70 + held - 1 - 64:
            assert (out[r, :, 9] == math.inf).all() and torch.equal(out[r, :, :9], clean[r, :, :9])
        else:
            assert torch.equal(out[r], clean[r])


def test_attn_leaves_rows_behind_and_past_max_rows(ctx):
    c = attn_case(20, [30, 12], 8, 2, 64, 16, "f16", prefix=20, add=[7, 3], extra_rows=5)
    check_attn(ctx, c)
    c = attn_case(20, [30, 12], 8, 2, 64, 16, "f16", prefix=20, add=[7, 3], extra_rows=5)
    want, _, tol, _ = attn_reference(c)
    c["max_rows"] = 4
    out, _ = run_attn(ctx, c)
    rows = [0, 1, 2, 3, 7, 8, 9]
    assert ((out.cpu().double()[rows] - want[rows]).abs() <= tol[rows]).all()
    assert (out[4:7] == 7).all() and (out[10:] == 7).all()


def test_attn_row_starts_that_contradict_each_other_stay_inside(ctx):
    """cu that is negative, falls, or passes the rows: rows without a sound place may hold anything, the others do not change."""
    c = attn_case(21, [30, 12, 9], 8, 2, 64, 16, "f16", prefix=20, add=[2, 2, 2])
    for cu in ([-5, 2, 4, 6], [0, 2, 1, 6], [0, 2, 4, 2 ** 31 - 1], [0, -2 ** 31, 2 ** 31 - 1, 3], [6, 6, 6, 6]):
        c["cu"] = i32(cu)
        run_attn(ctx, c)
        torch.cuda.synchronize()


def test_attn_past_32_bits(ctx):
    """Pages whose offsets pass 2^32 bytes and 2^31 values."""
    H, K, D, page = 4, 2, 128, 256
    pages = 36000                          # 4.7 G values: 9.4 GB of keys and of values
    c = attn_case(22, [300], H, K, D, page, "f16", prefix=260)
    small_k, small_v = c["keys"], c["values"]
    want = run_attn(ctx, c)[0].clone()
    big = {k: torch.empty(pages, K, page, D, dtype=torch.float16, device="cuda") for k in ("keys", "values")}
    far = torch.tensor([35999, 20000, 33000, 1, 30000, 34000], device="cuda")[:small_k.shape[0]]
    big["keys"][far], big["values"][far] = small_k, small_v
    c.update(big, shape=nunchi_amd.PageShape(H, K, D, page, pages, dtype="f16"))
    c["table"] = torch.where(c["table"] >= 0, far[c["table"].long().clamp(min=0)].int(), c["table"])
    c["shared"] = far[c["shared"].long()].int()
    assert torch.equal(run_attn(ctx, c)[0], want)
    # and the write to the far end
    p = put_case(23, 3, H, K, D, page, "f32", "f16")
    p.update(big)
    p["shape"] = c["shape"]
    p["slots"] = torch.tensor([35999 * 256 + 255, 30000 * 256, 17], device="cuda")
    nunchi_amd.page_put(ctx, p["shape"], p["qkv"], p["slots"], p["keys"], p["values"])
    v = p["qkv"].view(3, -1, D)[:, H + K:].half()
    for r, slot in enumerate(p["slots"].tolist()):
        assert torch.equal(big["values"][slot // 256, :, slot % 256], v[r])


def test_attn_same_bits_every_time(ctx):
    c = attn_case(24, [700, 300, 900], 8, 2, 64, 32, "f16", prefix=1300)
    first = [x.clone() for x in run_attn(ctx, c)]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run_attn(ctx, c)))


# ---------------------------------------------------------------- sampling


def sample_reference(x, u, temp=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(id, chance) of one row of scores in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64)) + 0.0
    if not (x > -np.inf).any() or not temp >= 0:
        return -1, 0.0
    if temp == 0:
        return int(np.argmax(x)), 1.0
    top_p = 1.0 if math.isnan(top_p) else top_p
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if x[order[0]] == np.inf:
        order = order[x[order] == np.inf]
        w = np.ones(len(order))
    else:
        w = np.exp((x[order] - x[order[0]]) / temp)
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    if top_p < 1:
        n = max(1, int(np.count_nonzero(np.cumsum(w) - w < top_p * w.sum())))
        order, w = order[:n], w[:n]
    if min_p > 0:
        keep = w >= min(min_p, 1.0)
        order, w = order[keep], w[keep]
    by_index = np.argsort(order)
    order, w = order[by_index], w[by_index]
    s = np.cumsum(w)
    u = 0.0 if not u > 0 else u
    at = min(int(np.searchsorted(s, u * s[-1], side="right")), len(order) - 1)
    return int(order[at]), w[at] / s[-1]


def run_sample(ctx, scores, u, **kw):
    rows, vocab = scores.shape
    ids, chance = i32(np.full(rows, -7)), torch.full((rows,), 7.0, device="cuda")
    work = torch.full((nunchi_amd.sample_work(rows, vocab),), 255, dtype=torch.uint8, device="cuda")
    types = {"temp": np.float32, "top_k": np.int32, "top_p": np.float32, "min_p": np.float32}
    kw = {k: dev(np.broadcast_to(np.asarray(v, types[k]), (rows,)).copy()) for k, v in kw.items()}
    nunchi_amd.sample(ctx, scores, dev(np.asarray(u, np.float64)), ids, work, chance=chance, **kw)
    torch.cuda.synchronize()
    return ids.cpu().numpy(), chance.cpu().numpy()


def check_sample(ctx, scores, u, **kw):
    ids, chance = run_sample(ctx, scores, u, **kw)
    x = scores.float().cpu().numpy()
    per_row = {k: np.broadcast_to(np.asarray(v, np.int32 if k == "top_k" else np.float32), (len(x),)) for k, v in kw.items()}
    for r in range(len(x)):
        want, c = sample_reference(x[r], u[r], **{k: v[r].item() for k, v in per_row.items()})
        assert ids[r] == want, (r, {k: v[r] for k, v in per_row.items()})
        assert abs(chance[r] - c) <= 2.0 ** -21 * c, (r, chance[r], c)


def random_scores(seed, rows, vocab, kind="f32", spread=3.0, banned=0.02):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=g)
    x[torch.rand(rows, vocab, generator=g) < banned] = -math.inf
    x[:, 0] = 0.5
    return x.to(TYPES[kind]).cuda(), torch.rand(rows, generator=g, dtype=torch.float64).numpy()


FILTERS = [dict(), dict(temp=0.7), dict(top_k=1), dict(top_k=40), dict(top_k=1000, temp=1.7), dict(top_p=0.9), dict(top_p=0.3, temp=0.6), dict(top_p=0.999, temp=2.5),
           dict(min_p=0.05), dict(min_p=0.9), dict(top_k=50, top_p=0.9, min_p=0.02, temp=0.8), dict(top_k=5000, top_p=0.97, temp=1.4), dict(temp=0.0)]


@pytest.mark.parametrize("kw", FILTERS, ids=str)
@pytest.mark.parametrize("vocab,kind", [(1, "f32"), (3, "f32"), (255, "bf16"), (1000, "f32"), (4097, "f16"), (32003, "f32"), (97496, "f32"), (50001, "bf16")])
def test_sample(ctx, vocab, kind, kw):
    x, u = random_scores(vocab, 7, vocab, kind)
    check_sample(ctx, x, u, **kw)


@pytest.mark.parametrize("vocab", [1000, 16384, 16385, 40000, 98304, 98305])
def test_sample_more_than_are_allowed(ctx, vocab):
    """top_k between the words that are allowed and all words, alone and with the other filters."""
    x, u = random_scores(vocab, 5, vocab, banned=0.5)
    for kw in (dict(top_k=int(0.7 * vocab)), dict(top_k=int(0.7 * vocab), top_p=0.8), dict(top_k=int(0.4 * vocab), top_p=0.95, min_p=0.001), dict(top_p=0.9)):
        check_sample(ctx, x, u, **kw)


@pytest.mark.parametrize("spread,temp", [(0.01, 1.0), (0.5, 3.0), (30.0, 1.0), (1000.0, 0.5), (1e30, 1e30), (1e-20, 1e-21)])
def test_sample_scales(ctx, spread, temp):
    """Weights that are nearly equal (cuts keep most words), and scores far apart."""
    g = torch.Generator().manual_seed(3)
    x = (spread * torch.randn(6, 30011, generator=g)).cuda()
    u = torch.rand(6, generator=g, dtype=torch.float64).numpy()
    for kw in (dict(), dict(top_k=900), dict(top_k=6000), dict(top_p=0.97), dict(top_k=20, top_p=0.7), dict(min_p=0.2)):
        check_sample(ctx, x, u, temp=temp, **kw)


def test_sample_largest_vocab(ctx):
    x, u = random_scores(1, 3, 524288)
    for kw in (dict(), dict(top_p=0.95), dict(top_k=100000), dict(top_k=70, top_p=0.9)):
        check_sample(ctx, x, u, **kw)


def test_sample_each_row_its_own_filters(ctx):
    rng = np.random.default_rng(4)
    x, u = random_scores(2, 64, 9001)
    check_sample(ctx, x, u, temp=rng.choice([0.0, 0.3, 1.0, 2.0], 64), top_k=rng.choice([-1, 0, 1, 7, 300, 9001, 20000], 64),
                 top_p=rng.choice([0.0, 0.2, 0.9, 1.0, 1.5, np.nan, -1.0], 64), min_p=rng.choice([0.0, 0.01, 0.5, 1.0, 2.0, np.nan, -1.0], 64))


@pytest.mark.parametrize("vocab", [40, 5000, 60000])
def test_sample_equal_scores(ctx, vocab):
    """All scores equal, or few different ones: cuts fall among equal words, which are kept by index."""
    rng = np.random.default_rng(vocab)
    u = rng.uniform(size=24)
    flat = torch.full((24, vocab), -2.5, device="cuda")
    for kw in (dict(), dict(top_k=13), dict(top_p=0.25), dict(top_k=30, top_p=0.5), dict(min_p=1.0), dict(top_k=vocab - 1), dict(temp=0.0)):
        check_sample(ctx, flat, u, **kw)
    steps = dev(rng.integers(0, 4, (24, vocab)).astype(np.float32))
    for kw in (dict(top_k=vocab // 3), dict(top_p=0.71), dict(top_k=vocab // 2, top_p=0.8), dict(min_p=0.3), dict(top_k=5, top_p=0.5)):
        check_sample(ctx, steps, u, **kw)


def test_sample_signed_zeros_are_equal(ctx):
    x = torch.zeros(2, 100, device="cuda")
    x[0, ::2] = -0.0
    x[1, 1::2] = -0.0
    for kw in (dict(top_k=3), dict(top_k=50), dict(temp=0.0), dict(top_p=0.105)):
        check_sample(ctx, x, [0.4, 0.99], **kw)


def test_sample_nothing_left_infinities_and_nan(ctx):
    x = torch.randn(9, 300, generator=torch.Generator().manual_seed(1))
    x[0] = -math.inf
    x[1] = math.nan
    x[2, :299] = -math.inf
    x[3, [7, 90]] = math.inf
    x[4, ::2] = math.nan
    x[5, 20] = 3e38
    x[5, 21] = -3e38
    x[6] = -3.4e38
    x[7, 0] = math.nan
    x = x.cuda()
    u = [0.5, 0.5, 0.999, 0.6, 0.3, 0.9, 0.77, 0.0, 0.1]
    for kw in (dict(), dict(top_k=2), dict(top_p=0.4), dict(min_p=0.2), dict(temp=0.0), dict(top_k=3, top_p=0.8, min_p=0.1), dict(temp=-1.0), dict(temp=float("nan")),
               dict(temp=float("inf")), dict(temp=1e-38), dict(temp=1e30)):
        check_sample(ctx, x, u, **kw)


def test_sample_random_numbers_at_and_past_the_ends(ctx):
    x, _ = random_scores(6, 8, 700)
    u = [0.0, -1.0, 1.0, 2.0, float("nan"), np.nextafter(1.0, 0.0), 1e-300, float("inf")]
    for kw in (dict(), dict(top_k=20), dict(top_p=0.8)):
        check_sample(ctx, x, u, **kw)


def test_sample_follows_the_chances(ctx):
    """Random numbers spread evenly over 4000 rows of the same scores: every word comes as often as its chance says, to one row."""
    x = torch.tensor([1.0, 0.0, -1.0, 2.0, 0.5]).repeat(4000, 1).cuda()
    ids, chance = run_sample(ctx, x, (np.arange(4000) + 0.5) / 4000, top_k=4)
    w = np.exp(np.array([1.0, 0.0, -np.inf, 2.0, 0.5]))
    assert (np.abs(np.bincount(ids, minlength=5) - 4000 * w / w.sum()) <= 1).all()


# ---------------------------------------------------------------- streams, graphs, and a run of them together


def test_streams_and_contexts(ctx):
    """The same calls from a context on another stream, and from one with a stream of its own."""
    c = attn_case(30, [200, 90], 8, 2, 64, 16, "f16", prefix=300)
    want = [t.clone() for t in run_attn(ctx, c)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    other = nunchi_amd.Context(0, stream=side.cuda_stream)
    with torch.cuda.stream(side):
        c["out"].fill_(3.0)
        got = [t.clone() for t in run_attn(other, c)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    own = nunchi_amd.Context(0)
    c["out"].fill_(3.0)
    work = torch.empty(nunchi_amd.page_attn_work(c["shape"], 2, 2, c["max_len"], 1, 300), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    run_attn(own, c, work)
    own.sync()
    assert all(torch.equal(a, b) for a, b in zip(want, (c["out"], c["lse"])))
    other.close()
    own.close()


def test_engine_on_the_default_stream(tiny_model):
    """A brain whose context is on the caller's stream steps as one with a stream of its own."""
    a = nunchi_amd.Brain(tiny_model, n_ctx=64)
    side = torch.cuda.Stream()
    for stream in (0, side.cuda_stream):
        b = nunchi_amd.Brain(tiny_model, n_ctx=64, ctx=nunchi_amd.Context(0, stream=stream))
        a.reset()
        for tok in (3, 141, 59):
            (ha, la, ia), (hb, lb, ib) = a.step(tok), b.step(tok)
            assert np.array_equal(ha, hb) and np.array_equal(la, lb) and ia == ib
        assert np.array_equal(a.generate(5, 6)[0], b.generate(5, 6)[0])
        u = np.random.default_rng(2).uniform(size=7)
        assert np.array_equal(a.generate_sampled(8, u, top_k=30)[0], b.generate_sampled(8, u, top_k=30)[0])
        # (a longer call after a shorter one, and a shorter one again)
        u = np.random.default_rng(3).uniform(size=20)
        x, y = (z.generate_sampled(9, u, a=z.new_state())[0] for z in (a, b))
        assert np.array_equal(x, y) and np.array_equal(x[:5], b.generate_sampled(9, u[:5], a=b.new_state())[0])


@pytest.mark.parametrize("kw", [dict(), dict(temp=0.7, top_k=20), dict(top_p=0.8, temp=1.3), dict(min_p=0.1), dict(temp=0.0)], ids=str)
def test_generate_sampled(mid_model, kw):
    """The device loop against single steps whose word scores go through the reference: one conversation and two."""
    rng = np.random.default_rng(8)
    brain = nunchi_amd.Brain(mid_model, n_ctx=64)
    u, ub = rng.uniform(size=9), rng.uniform(size=9)
    f32 = {k: (np.float32(v).item() if k != "top_k" else v) for k, v in kw.items()}

    def steps(first, u, st):
        tok, out = first, []
        for x in u:
            _, scores, _ = brain.step(tok, st=st)
            tok = sample_reference(scores, x, **f32)[0]
            out.append(tok)
        return out

    ids, secs = brain.generate_sampled(7, u, **kw)
    assert secs > 0 and brain.pos == 9
    assert ids.tolist() == steps(7, u, brain.new_state())
    if kw.get("temp") == 0.0:
        assert ids.tolist() == brain.generate(7, 9, a=brain.new_state())[0].tolist()
    a, b = brain.new_state(), brain.new_state()
    ia, ib, _ = brain.generate_sampled(11, u, b=b, first_b=12, u_b=ub, a=a, **kw)
    assert ia.tolist() == steps(11, u, brain.new_state()) and ib.tolist() == steps(12, ub, brain.new_state())
    assert a.pos == b.pos == 9


def test_generate_sampled_refuses(tiny_model):
    brain = nunchi_amd.Brain(tiny_model, n_ctx=16)
    for bad in (dict(temp=-1.0), dict(temp=float("nan")), dict(first=-1), dict(first=1000)):
        kw = {"first": 3, "u": [0.5] * 4, **bad}
        with pytest.raises(nunchi_amd.SeoulError):
            brain.generate_sampled(**kw)
    with pytest.raises(nunchi_amd.ContextFull):
        brain.generate_sampled(3, [0.5] * 17)
    with pytest.raises(nunchi_amd.SeoulError):
        brain.generate_sampled(3, [0.5], b=brain.state, u_b=[0.5])
    with pytest.raises(ValueError):
        brain.generate_sampled(3, [0.5], b=brain.new_state(), u_b=[0.5, 0.5])
    assert brain.pos == 0 and brain.generate_sampled(3, [])[0].size == 0


class Serving:
    """A small serving loop: conversations behind a shared prefix, step by step, in pages."""

    def __init__(self, ctx, kind="f16", window=0):
        self.H, self.K, self.D, self.page, self.n, self.prefix = 8, 2, 64, 16, 5, 40
        self.ctx, self.kind = ctx, kind
        g = self.g = torch.Generator().manual_seed(77)
        pages = 64
        self.shape = nunchi_amd.PageShape(self.H, self.K, self.D, self.page, pages, dtype=kind, window=window)
        self.window = window
        self.keys, self.values = (torch.full(self.shape.cache_shape, math.nan, dtype=TYPES[kind], device="cuda") for _ in range(2))
        order = torch.randperm(pages, generator=g).int()
        self.shared, self.free = order[:3].cuda(), order[3:].cuda()
        ang = torch.rand(400, self.D // 2, generator=g) * 6.28
        self.rope = torch.stack([ang.cos(), ang.sin()], -1).cuda()
        self.w = [(1 + 0.1 * torch.randn(self.D, generator=g)).cuda() for _ in range(2)]
        self.words = torch.randn(self.H * self.D, 500, generator=g).cuda() * 0.2
        self.table = torch.full((self.n, 8), -1, dtype=torch.int32, device="cuda")
        self.held, self.taken = torch.zeros(self.n, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        # the shared prefix: one "request" of its own
        ld = (self.H + 2 * self.K) * self.D
        x = torch.randn(self.prefix, ld, generator=g).cuda()
        slots = torch.tensor([int(self.shared[p // 16]) * 16 + p % 16 for p in range(self.prefix)]).cuda()
        nunchi_amd.page_put(ctx, self.shape, x, slots, self.keys, self.values, pos=torch.arange(self.prefix, dtype=torch.int32).cuda(), q_norm=self.w[0],
                            k_norm=self.w[1], rope=self.rope)
        self.history = [[x.cpu()] for _ in range(self.n)]

    def buffers(self, add):
        rows, f = int(add.sum()), dict(dtype=torch.int32, device="cuda")
        cap = 64   # the longest own context
        return {"add": add.cuda(), "len": torch.zeros(self.n, **f), "cu": torch.zeros(self.n + 1, **f), "slots": torch.zeros(rows, dtype=torch.int64, device="cuda"),
                "pos": torch.zeros(rows, **f), "taken": torch.zeros(1, **f), "q": torch.zeros(rows, self.H, self.D, dtype=TYPES[self.kind], device="cuda"),
                "out": torch.zeros(rows, self.H, self.D, dtype=TYPES[self.kind], device="cuda"), "cap": cap, "max_rows": int(add.max()),
                "x": torch.zeros(rows, (self.H + 2 * self.K) * self.D, device="cuda"), "u": torch.zeros(rows, dtype=torch.float64, device="cuda"),
                "ids": torch.zeros(rows, **f), "chance": torch.zeros(rows, device="cuda"), "scores": torch.zeros(rows, 500, device="cuda"),
                "work": torch.empty(nunchi_amd.page_attn_work(self.shape, self.n, rows, cap, int(add.max()), self.prefix), dtype=torch.uint8, device="cuda"),
                "swork": torch.empty(nunchi_amd.sample_work(rows, 500), dtype=torch.uint8, device="cuda")}

    def enqueue(self, b, ctx=None):
        ctx = ctx or self.ctx
        nunchi_amd.page_plan(ctx, self.held, b["add"], self.free, self.taken, self.table, self.page, b["len"], b["cu"], b["slots"], b["pos"], b["taken"], pos0=self.prefix)
        nunchi_amd.page_put(ctx, self.shape, b["x"], b["slots"], self.keys, self.values, q=b["q"], pos=b["pos"], q_norm=self.w[0], k_norm=self.w[1], rope=self.rope)
        nunchi_amd.page_attn(ctx, self.shape, b["q"], self.keys, self.values, self.table, b["len"], b["out"], b["work"], b["cap"], cu=b["cu"], max_rows=b["max_rows"],
                             prefix=self.shared, prefix_len=self.prefix)
        b["scores"].copy_(b["out"].view(-1, self.H * self.D).float() @ self.words)
        nunchi_amd.sample(ctx, b["scores"], b["u"], b["ids"], b["swork"], temp=None, top_k=None, top_p=torch.full_like(b["chance"], 0.9), chance=b["chance"])
        self.held.copy_(b["len"])
        self.taken.copy_(b["taken"])

    def fill(self, b):
        b["x"].copy_(torch.randn(b["x"].shape, generator=self.g))
        b["u"].copy_(torch.rand(b["u"].shape, generator=self.g, dtype=torch.float64))

    def check(self, b):
        """The step's outputs against contiguous keys and values in 64 bits."""
        at = 0
        h = HALF[self.kind]
        for i, a in enumerate(b["add"].tolist()):
            if not a:
                continue
            self.history[i].append(b["x"][at:at + a].cpu())
            x = torch.cat(self.history[i]).double().view(-1, self.H + 2 * self.K, self.D)
            cs = self.rope.cpu()[:len(x)]
            q = heads_reference(x[:, :self.H], self.w[0].cpu(), 1e-5, cs).to(TYPES[self.kind]).double()
            k = heads_reference(x[:, self.H:self.H + self.K], self.w[1].cpu(), 1e-5, cs).to(TYPES[self.kind]).double().repeat_interleave(self.H // self.K, 1)
            v = x[:, self.H + self.K:].to(TYPES[self.kind]).double().repeat_interleave(self.H // self.K, 1)
            for r in range(a):
                me = len(x) - a + r
                lo = max(0, me + 1 - self.window) if self.window else 0
                s = (q[me][None] * k[lo:me + 1]).sum(-1) / math.sqrt(self.D)
                want = torch.softmax(s, 0)[..., None].mul(v[lo:me + 1]).sum(0)
                # queries and keys may round the other way where single precision falls on a tie: one step of either moves
                # a score by 2 HALF of the sum of the products' sizes at most, the weights by twice that
                moved = 4 * h * (q[me][None].abs() * k[lo:me + 1].abs()).sum(-1).amax() / math.sqrt(self.D)
                tol = (2.01 * h + 2.0 ** -14 + moved) * v[lo:me + 1].abs().amax()
                assert ((b["out"][at + r].cpu().double() - want).abs() <= tol).all()
                # the next word, from the scores as they are
                want_id, c = sample_reference(b["scores"][at + r].cpu().numpy(), b["u"][at + r].item(), top_p=np.float32(0.9).item())
                assert b["ids"][at + r].item() == want_id and abs(b["chance"][at + r].item() - c) <= 2.0 ** -21 * c
            at += a


@pytest.mark.parametrize("kind,window", [("f16", 0), ("bf16", 24)])
def test_serving_run(ctx, kind, window):
    """Prompts, decode steps, a conversation that joins late and one that pauses: plan, put, attn and sample in turn."""
    s = Serving(ctx, kind, window)
    for add in ([7, 20, 0, 1, 33], [1, 1, 1, 1, 1], [1, 1, 0, 1, 1], [1, 1, 16, 1, 0], [1, 1, 1, 1, 1], [1, 1, 1, 1, 1]):
        b = s.buffers(torch.tensor(add, dtype=torch.int32))
        s.fill(b)
        s.enqueue(b)
        torch.cuda.synchronize()
        s.check(b)


def test_serving_step_in_a_graph():
    """A decode step captured once and replayed, its lengths and tables carried on the device, with eager work and waits
    between the replays; every replay is checked."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        side = nunchi_amd.Context(0, stream=stream.cuda_stream)
        s = Serving(side)
        b0 = s.buffers(torch.tensor([3, 17, 1, 16, 30], dtype=torch.int32))
        s.fill(b0)
        s.enqueue(b0)
        stream.synchronize()
        s.check(b0)
        b = s.buffers(torch.tensor([1, 1, 1, 1, 1], dtype=torch.int32))
        s.fill(b)
        s.enqueue(b)          # (once eagerly: the plain product's library sets itself up)
        stream.synchronize()
        s.check(b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s.enqueue(b)
        for k in range(6):
            s.fill(b)
            graph.replay()
            stream.synchronize()
            s.check(b)
            torch.randn(1000, device="cuda").sum().item()
    stream.synchronize()


def test_tensors_are_checked(ctx):
    """Types, shapes, strides and devices of tensors are refused before the call."""
    x, u = random_scores(1, 4, 100)
    ids, work = i32([0] * 4), torch.zeros(256, dtype=torch.uint8, device="cuda")
    ud = dev(u)
    with pytest.raises(TypeError):
        nunchi_amd.sample(ctx, x.double(), ud, ids, work)
    with pytest.raises(TypeError):
        nunchi_amd.sample(ctx, x, ud.float(), ids, work)
    with pytest.raises(ValueError):
        nunchi_amd.sample(ctx, x[:, ::2], ud, ids, work)
    with pytest.raises(ValueError):
        nunchi_amd.sample(ctx, x, ud, ids[:3], work)
    with pytest.raises(ValueError):
        nunchi_amd.sample(ctx, x.cpu(), ud, ids, work)
    with pytest.raises(nunchi_amd.SeoulError):
        nunchi_amd.sample(ctx, x, ud, ids, work[:8])
    c = attn_case(1, [20], 8, 2, 64, 16, "f16", prefix=20)
    with pytest.raises(ValueError):
        nunchi_amd.page_attn(ctx, c["shape"], c["q"], c["keys"], c["values"], c["table"], c["length"], c["out"], work, 20, prefix=c["shared"][:1], prefix_len=20)
    with pytest.raises(ValueError):
        run_attn(ctx, {**c, "keys": c["keys"][1:]})


LOW_LAYOUTS = [(700, "f32"), (40000, "f32"), (120000, "f32"), (1000, "bf16"), (70001, "f16"), (262144, "bf16")]


@pytest.mark.parametrize("kw", [dict(), dict(top_k=20), dict(top_k=300), dict(top_p=0.9), dict(top_k=12, top_p=0.8), dict(min_p=0.01), dict(temp=1.3)], ids=str)
@pytest.mark.parametrize("vocab,kind", LOW_LAYOUTS)
def test_sample_never_takes_words_without_weight(ctx, vocab, kind, kw):
    """Words 300 and more below the maximum (2^-432 of it: no weight in 2^-44ths) first and last in every block, u at the ends of
    its range: none of them is taken, whatever holds the row."""
    g = torch.Generator().manual_seed(vocab)
    u = [0.0, -1.0, math.nan, 1.0, 2.0, np.nextafter(1.0, 0.0), 1e-300, 0.5, 0.77]
    x = torch.full((len(u), vocab), -math.inf)
    for at in (0, 1, 255, 256, 511, 512):
        x[:, at::1024] = -300.0 - at
    x[:, 255::256], x[:, ::256], x[:, -1] = -1000.0, -60000.0, -60000.0
    good = torch.randperm(vocab, generator=g)[:60]
    x[:, good] = 5 + torch.randn(len(u), 60, generator=g)
    x = x.to(TYPES[kind])
    ids, chance = run_sample(ctx, x.cuda(), u, **kw)
    x = x.double().numpy()
    x[x < -100] = -np.inf
    kw = {k: v if k == "top_k" else np.float32(v).item() for k, v in kw.items()}
    for r in range(len(u)):
        want, c = sample_reference(x[r], u[r], **kw)
        assert ids[r] == want, (r, ids[r], want)
        assert chance[r] > 0 and abs(chance[r] - c) <= 2.0 ** -21 * c, (r, chance[r], c)


@pytest.mark.parametrize("vocab,kind", LOW_LAYOUTS)
def test_sample_small_weights_beside_a_large_one(ctx, vocab, kind):
    """255 words of e^-18 (one of e^-20) in the block of one of weight 1, and u inside the k-th one's share: sums in 2^-44ths tell
    them apart. A small weight is 2^-26 (2^-28.9), its last place 2^-18 (2^-15) of it and its exponential's 2^-22, so 255 of them
    are off by less than 1/500 of one; u is 1/4 of one from the next."""
    g = torch.Generator().manual_seed(1)
    k = torch.randint(0, 255, (24,), generator=g).numpy()
    e = math.exp(-18.0)
    x = torch.full((24, vocab), -math.inf)
    x[:, :256] = -18.0
    x[:, 128] = 0.0
    total = 1 + 255 * e
    u = np.where(k < 128, (k + 0.25) * e, 1 + (k + 0.25) * e) / total
    want = k + (k >= 128)
    x = x.to(TYPES[kind]).cuda()
    for kw in (dict(), dict(min_p=1e-9), dict(top_k=256)):
        ids, _ = run_sample(ctx, x, u, **kw)
        assert np.array_equal(ids, want), kw
    # one small word, last of the block and of the row
    for at in (255, vocab - 1):
        x = torch.full((6, vocab), -math.inf)
        x[:, 0], x[:, at] = 0.0, -20.0
        ids, chance = run_sample(ctx, x.to(TYPES[kind]).cuda(), [1.0, 1 - 1e-9, np.nextafter(1.0, 0.0), 1 - 3e-9, 0.0, 3.0])
        assert ids.tolist() == [at, at, at, 0, 0, at]
        assert abs(chance[0] / math.exp(-20.0) - 1) < 2.0 ** -21


def test_first_step_beside_work_on_the_same_stream(tiny_model):
    """A brain on the caller's stream makes its graph while another thread enqueues there: what that thread enqueues runs once,
    when it is its turn, and no replay of the graph repeats it."""
    side = torch.cuda.Stream()
    x = torch.zeros(64, device="cuda")
    torch.cuda.synchronize()
    stop, started, count, errors = threading.Event(), threading.Event(), [0], []

    def other():
        try:
            with torch.cuda.stream(side):
                while not stop.is_set():
                    x.add_(1)
                    count[0] += 1
                    started.set()
        except Exception as e:   # noqa: BLE001  (shown by the test's own thread)
            errors.append(e)
            started.set()

    brains = [nunchi_amd.Brain(tiny_model, n_ctx=64, ctx=nunchi_amd.Context(0, stream=side.cuda_stream)) for _ in range(6)]
    thread = threading.Thread(target=other)
    thread.start()
    try:
        assert started.wait(60)
        ids = [[b.step(t)[2] for t in (3, 141, 59)] for b in brains]
    finally:
        stop.set()
        thread.join()
    side.synchronize()
    assert not errors, errors
    assert (x == count[0]).all(), (x[0].item(), count[0])
    assert all(i == ids[0] for i in ids)
    for b in brains:
        b.step(7)
    side.synchronize()
    assert (x == count[0]).all(), "a replay repeats the other thread's work"


@pytest.mark.parametrize("rows", [509, 511, 512, 513, 1027])
def test_plan_row_counts_at_the_variants_border(ctx, rows):
    """Rows on either side of where a thread takes four neighbouring ones, shared by requests of none to nine."""
    rng = np.random.default_rng(rows)
    add = rng.integers(0, 10, 2 * rows)
    add = add[:int(np.searchsorted(np.cumsum(add), rows)) + 1]
    add[-1] -= add.sum() - rows
    n = len(add)
    held = rng.integers(0, 60, n)
    have, want = -(-held // 16), -(-(held + add) // 16)
    ids = rng.permutation(int(want.sum()))
    table, at = np.full((n, 5), -1), 0
    for i in range(n):
        table[i, :have[i]] = ids[at:at + have[i]]
        at += have[i]
    check_plan(ctx, held, add, 16, table, ids[at:], 0, rows, pos0=5)
