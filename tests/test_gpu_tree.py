"""The operators for drafted words (sh_tree_plan, sh_tree_attn, sh_word_probs, sh_tree_take, sh_page_keep) against plain
implementations in 64 bits on the CPU.

Tolerances count roundings (HALF: half a step of a 16-bit type relative to the value; single precision: 2^-24).
 attn:  as tests/test_gpu_batch.py derives them for sh_page_attn: the sums are the same, over other keys.
 probs: the largest score's weight is 1 exactly, so errors are the others' (the rest). A weight's exponent is a product of a
        difference (2^-24) and log2 e / temp (rounded three times); it is taken in up to four pieces (wave, part, lane, row)
        that add up to it, each through a hardware exponential (2^-22): 4 2^-24 |z| and 4 2^-22 of the weight, z its distance
        to the largest in temperatures. Sums of at most 2^19 words: 16 a lane's turn, 8 in a wave, 4 waves and 8 joins below 64
        roundings. With S1 = sum e^z |z|, S2 = sum e^z z^2 over L: log L is off by 2^-22 S1 + (2^-20 + 2^-18) rest, a log
        probability by that, 2^-22 of log L and 2^-22 |z|, the entropy by the same and 2^-22 S2 + 2^-17 S1.
"""
import math

import numpy as np
import pytest

import nunchi_amd
from conftest import ROOT  # noqa: F401  (the repository's root in sys.path)

torch = pytest.importorskip("torch")
import test_gpu_batch as tb  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES, HALF, dev, i32 = tb.TYPES, tb.HALF, tb.dev, tb.i32


@pytest.fixture(scope="module")
def ctx():
    return nunchi_amd.Context(0, stream=torch.cuda.current_stream().cuda_stream)


def trees(seed, sizes, bush=None):
    """Parents of the rows of requests of these sizes, the first of each without one."""
    rng = np.random.default_rng(seed)
    out = []
    for m in sizes:
        b = rng.choice([0.0, 0.3, 1.0]) if bush is None else bush
        out += [min(j - 1, int(rng.random() ** b * j)) if b and j else j - 1 for j in range(m)]
    return out


def follows(parent, sizes):
    """For each row the set of its request's words that it sees; None for a row that follows something that is not before it."""
    out, at = [], 0
    for m in sizes:
        sets = []
        for j in range(m):
            p = parent[at + j]
            ok = -1 <= p < j and (p < 0 or sets[p] is not None)
            sets.append((sets[p] if p >= 0 else frozenset()) | {j} if ok else None)
        out += sets
        at += m
    return out


def words_of(sets, words):
    out = np.zeros((len(sets), words), np.uint32)
    for r, s in enumerate(sets):
        for k in s or ():
            out[r, k >> 5] |= np.uint32(1 << (k & 31))
    return out.view(np.int32)


def starts(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)


# ---------------------------------------------------------------- masks and positions


def run_plan(ctx, cu, parent, held, length, max_rows, pos0=0, rows=None):
    rows = len(parent) if rows is None else rows
    mask, pos = torch.full((rows, (max_rows + 31) // 32), 77, dtype=torch.int32, device="cuda"), torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    nunchi_amd.tree_plan(ctx, i32(cu), i32(parent), i32(held), i32(length), mask, pos, max_rows, pos0=pos0)
    return mask.cpu().numpy(), pos.cpu().numpy()


@pytest.mark.parametrize("sizes,max_rows", [([1], 1), ([1, 0, 2], 2), ([8, 8], 8), ([31, 32, 33], 33), ([64, 63, 1, 0], 64), ([65, 2], 65), ([256, 129, 0, 255], 256),
                                            ([5] * 700, 31), ([0, 0, 3], 100), ([40], 256)])
@pytest.mark.parametrize("bush", [0.0, 0.3, 1.0, None])
def test_plan(ctx, sizes, max_rows, bush):
    parent = trees(sum(sizes), sizes, bush)
    held = np.random.default_rng(1).integers(0, 5000, len(sizes))
    mask, pos = run_plan(ctx, starts(sizes), parent, held, held + sizes, max_rows, pos0=13)
    sets = follows(parent, sizes)
    assert np.array_equal(mask, words_of(sets, mask.shape[1]))
    who = np.repeat(np.arange(len(sizes)), sizes)
    assert pos.tolist() == [13 + held[i] + len(s) - 1 for i, s in zip(who, sets)]


def test_plan_parents_that_are_not_before_their_words(ctx):
    """Such a word, and all that follow it, have no bits; the others do not notice."""
    sizes = [9, 4, 5]
    parent = [-1, 0, 1, 3, 3, 1, 8, 6, -2] + [0, -1, 1, 2] + [-1, -1, 2 ** 31 - 1, -2 ** 31, 1]
    sets = follows(parent, sizes)
    assert [s is None for s in sets] == [False, False, False, True, True, False, True, True, True] + [True, False, False, False] + [False, False, True, True, False]
    mask, pos = run_plan(ctx, starts(sizes), parent, [4, 0, 7], [13, 4, 12], 9)
    assert np.array_equal(mask, words_of(sets, 1))
    assert pos.tolist() == [{0: 4, 1: 0, 2: 7}[i] + len(s) - 1 if s else -1 for i, s in zip([0] * 9 + [1] * 4 + [2] * 5, sets)]


def test_plan_requests_that_were_refused(ctx):
    """No bits for a request whose length does not hold its rows, that has more rows than max_rows, or rows past the step's."""
    sizes = [3, 2, 5, 2]
    parent = trees(3, sizes, 0.0)
    mask, pos = run_plan(ctx, starts(sizes), parent, [5, 6, 7, 8], [5, 8, 12, 10], 4)
    assert pos.tolist() == [-1] * 3 + [6, 7] + [-1] * 5 + [8, 9]
    assert mask[:, 0].tolist() == [0] * 3 + [1, 3] + [0] * 5 + [1, 3]
    mask, pos = run_plan(ctx, starts(sizes), parent, [5, 6, 7, -1], [8, 8, 12, 1], 5, rows=12)
    assert pos.tolist() == [5, 6, 7, 6, 7, 7, 8, 9, 10, 11, -1, -1]
    mask, pos = run_plan(ctx, starts(sizes), parent[:11], [5, 6, 7, 8], [8, 8, 12, 10], 5)
    assert pos.tolist() == [5, 6, 7, 6, 7, 7, 8, 9, 10, 11, -1]


def test_plan_leaves_rows_behind_and_keeps_positions_inside(ctx):
    mask, pos = run_plan(ctx, [0, 2, 3], [-1, 0, -1, -1, -1], [2 ** 31 - 4, 3], [2 ** 31 - 2, 4], 2, pos0=2)
    assert pos.tolist() == [2 ** 31 - 2, 2 ** 31 - 1, 5, 77, 77] and mask[:, 0].tolist() == [1, 3, 1, 77, 77]
    _, pos = run_plan(ctx, [0, 2, 3], [-1, 0, -1], [2 ** 31 - 4, 3], [2 ** 31 - 2, 4], 2, pos0=9)
    assert pos.tolist() == [2 ** 31 - 1, 2 ** 31 - 1, 12]


def test_row_starts_that_contradict_each_other_stay_inside(ctx):
    for cu in ([-5, 2, 4, 6], [0, 2, 1, 6], [0, 2, 4, 2 ** 31 - 1], [0, -2 ** 31, 2 ** 31 - 1, 3], [6, 6, 6, 6]):
        run_plan(ctx, cu, [-1] * 6, [1, 2, 3], [3, 4, 5], 6)
        run_take(ctx, cu, [-1] * 6, [0] * 6, [0] * 6, [1, 2, 3], [3, 4, 5])
        c = keep_case(1, [20, 20, 20], [2, 2, 2], 2, 32, 16, "f16")
        c["cu"] = i32(cu)
        run_keep(ctx, c, [0, 1] * 3)
        torch.cuda.synchronize()


# ---------------------------------------------------------------- attention


def tree_case(seed, lens, sizes, H, K, D, page, kind, parent=None, sets=None, max_rows=None, **kw):
    c = tb.attn_case(seed, lens, H, K, D, page, kind, add=sizes, **kw)
    c["sets"] = sets if sets is not None else follows(trees(seed, sizes) if parent is None else parent, sizes)
    c["max_rows"] = max(max(sizes), 1) if max_rows is None else max_rows
    extra = c["q"].shape[0] - len(c["sets"])
    c["mask"] = torch.from_numpy(np.concatenate([words_of(c["sets"], (c["max_rows"] + 31) // 32), np.full((extra, (c["max_rows"] + 31) // 32), -1, np.int32)])).cuda()
    return c


def run_tree(ctx, c, work=None):
    rows = c["q"].shape[0]
    size = nunchi_amd.tree_attn_work(c["shape"], len(c["lens"]), rows, c["max_len"], c["max_rows"], c["prefix"])
    work = torch.full((size,), 255, dtype=torch.uint8, device="cuda") if work is None else work    # (NaN in every part)
    nunchi_amd.tree_attn(ctx, c["shape"], c["q"], c["keys"], c["values"], c["table"], c["length"], c["cu"], c["mask"], c["out"], work, c["max_len"],
                         c["max_rows"], prefix=c["shared"], prefix_len=c["prefix"], gate=c["gate"], lse=c["lse"])
    return c["out"], c["lse"]


def tree_reference(c):
    """(out, lse, tolerance of out, of lse) in 64 bits, row by row."""
    H, K, D, page = c["dims"]
    keys, values, q = (c[k].cpu().double() for k in ("keys", "values", "q"))
    rows, L0, window = c["rows"], c["prefix"], c["window"]
    out, lse = torch.zeros(rows, H, D, dtype=torch.float64), torch.full((rows, H), -math.inf, dtype=torch.float64)
    tol, tol_lse = torch.zeros(rows, H, 1, dtype=torch.float64), torch.zeros(rows, H, dtype=torch.float64)
    table, shared = c["table"].tolist(), c["shared"].tolist()
    r0 = 0
    for i, held in enumerate(c["lens"]):
        held, m = max(held, 0), c["counts"][i]
        base = held - m
        places = [(shared[p // page], p % page, p) for p in range(L0)] + [(table[i][p // page], p % page, L0 + p) for p in range(max(base, 0))]
        for r in range(r0, r0 + m):
            words = c["sets"][r] or frozenset()
            if r - r0 not in words or base < 0:
                continue
            order = sorted(words)
            me = L0 + base + len(order) - 1
            seen = [(a, b) for a, b, p in places if not window or p > me - window]
            for nth, k in enumerate(order):     # its words from the first to itself
                if 0 <= base + k < held and (not window or nth > len(order) - 1 - window):
                    seen.append((table[i][(base + k) // page], (base + k) % page))
            seen = [(a, b) for a, b in seen if 0 <= a < keys.shape[0]]
            if not seen:
                continue
            a, b = torch.tensor([x[0] for x in seen]), torch.tensor([x[1] for x in seen])
            k, v = keys[a, :, b].repeat_interleave(H // K, 1), values[a, :, b].repeat_interleave(H // K, 1)
            s = (q[r][None] * k).sum(-1) * c["scale"]
            size = (q[r][None] * k).abs().sum(-1).amax(0) * c["scale"]
            top = s.amax(0)
            e = torch.exp(s - top)
            lse[r] = top + torch.log(e.sum(0))
            out[r] = (e / e.sum(0))[..., None].mul(v).sum(0)
            off = 2.0 ** -24 * (D * size + 3 * s.abs().amax(0) / math.log(2) + len(seen) / 128 + 16) + 2.0 ** -20
            tol_lse[r] = off + 2.0 ** -23 * lse[r].abs()
            # (f16 weights are 2^8 of the running maximum's: below 2^-14 their places are 2^-24 apart)
            under = 2.0 ** -33 * len(seen) if c["kind"] == "f16" else 0.0
            tol[r, :, 0] = (HALF[c["kind"]] * 1.01 + under + 2 * off) * v.abs().amax(0).amax(-1)
        r0 += m
    if c["gate"] is not None:
        f = torch.sigmoid(c["gate"].cpu().double()[:rows])[..., None]
        out, tol = out * f, tol * f
    return out, lse, tol + HALF[c["kind"]] * out.abs() + 2.0 ** -25, tol_lse


def check_tree(ctx, c):
    out, lse = run_tree(ctx, c)
    want, want_lse, tol, tol_lse = tree_reference(c)
    rows = c["rows"]
    got, got_lse = out.cpu().double(), lse.cpu().double()
    assert torch.isfinite(got[:rows]).all()
    worst = ((got[:rows] - want).abs() - tol).max().item()
    assert worst <= 0, worst
    none = want_lse == -math.inf
    assert torch.equal(got_lse[:rows] == -math.inf, none)
    assert (got[:rows][none] == 0).all()
    assert ((got_lse[:rows] - want_lse).abs()[~none] <= tol_lse[~none]).all(), ((got_lse[:rows] - want_lse).abs() - tol_lse)[~none].max().item()
    assert (got[rows:] == 7).all() and (got_lse[rows:] == 7).all(), "rows behind the last request's"


LAYOUTS = [(8, 2, 64, 16, "f16"), (16, 4, 128, 32, "bf16"), (8, 2, 32, 64, "f16"), (7, 1, 128, 256, "f16"), (20, 1, 64, 16, "bf16"), (6, 6, 64, 128, "f16"), (4, 1, 32, 16, "bf16")]


@pytest.mark.parametrize("H,K,D,page,kind", LAYOUTS)
def test_attn_sizes(ctx, H, K, D, page, kind):
    """Trees of one word, of odd numbers and none, alone and behind lengths on either side of every block and page edge."""
    sizes = [1, 5, 0, 13, 1, 33, 2, 7, 3]
    base = [0, 0, 9, 31, 32, 17, 63, 127, 160]
    check_tree(ctx, tree_case(H * D, [b + m for b, m in zip(base, sizes)], sizes, H, K, D, page, kind))


@pytest.mark.parametrize("H,K,D,page,kind", LAYOUTS[:5])
@pytest.mark.parametrize("prefix", [1, 16, 31, 100, 257, 700])
def test_attn_shared_prefix(ctx, H, K, D, page, kind, prefix):
    check_tree(ctx, tree_case(prefix, [6, 40, 17, 0, 130], [6, 11, 17, 0, 1], H, K, D, page, kind, prefix=prefix))


@pytest.mark.parametrize("H,K,D,page,kind", LAYOUTS[:3])
@pytest.mark.parametrize("prefix,window", [(0, 1), (0, 9), (50, 40), (300, 3), (10, 33), (90, 100), (33, 2 ** 31 - 1)])
def test_attn_windows(ctx, H, K, D, page, kind, prefix, window):
    """Windows shorter than a branch, that end among the words, the own positions, the shared ones, and that leave nothing out."""
    sizes = [5, 40, 0, 12, 1, 20]
    check_tree(ctx, tree_case(prefix + window % 97, [5, 70, 0, 33, 90, 20], sizes, H, K, D, page, kind, prefix=prefix, window=window))
    check_tree(ctx, tree_case(prefix, [40, 60], [40, 37], H, K, D, page, kind, prefix=prefix, window=window, parent=trees(1, [40, 37], 0.0)))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D,H,K", [(64, 8, 2), (128, 4, 1), (32, 8, 1)])
def test_attn_largest_trees(ctx, kind, D, H, K):
    check_tree(ctx, tree_case(D, [256, 300, 129], [256, 255, 65], H, K, D, 64, kind, prefix=70))


@pytest.mark.parametrize("n,length,prefix,m", [(1, 3000, 0, 9), (2, 1111, 2500, 33), (30, 300, 1100, 5), (1, 9000, 100, 2)])
def test_attn_many_parts(ctx, n, length, prefix, m):
    check_tree(ctx, tree_case(n, [length - 7 * i for i in range(n)], [m] * n, 4, 2, 64, 64, "f16", prefix=prefix))


def test_attn_long_parts(ctx):
    """Requests that are one part each, of lengths on either side of a whole number of a wave's page lookups (63 blocks of 128
    keys): single words, against the attention of single rows."""
    K, D, page, lens = 8, 32, 128, [8063, 8064, 8065, 8066, 8191, 8192, 8193, 16127, 16128, 16129, 17000] * 7
    g = torch.Generator().manual_seed(8)
    pages, n = -(-max(lens) // page), len(lens)
    keys, values = (torch.randn(pages, K, page, D, generator=g).half().cuda() for _ in range(2))
    q = torch.randn(n, K, D, generator=g).half().cuda()
    shape = nunchi_amd.PageShape(K, K, D, page, pages)
    table, length = torch.randperm(pages, generator=g).int().repeat(n, 1).cuda(), i32(lens)
    out = [torch.zeros_like(q) for _ in range(2)]
    lse = [torch.zeros(n, K, device="cuda") for _ in range(2)]
    works = [torch.empty(f, dtype=torch.uint8, device="cuda") for f in (nunchi_amd.page_attn_work(shape, n, n, max(lens)), nunchi_amd.tree_attn_work(shape, n, n, max(lens), 1))]
    nunchi_amd.page_attn(ctx, shape, q, keys, values, table, length, out[0], works[0], max(lens), lse=lse[0])
    nunchi_amd.tree_attn(ctx, shape, q, keys, values, table, length, i32(range(n + 1)), i32([[1]] * n), out[1], works[1], max(lens), 1, lse=lse[1])
    # (both within half a step of the largest value and of the result; scores of 32 products below 32 in size)
    assert ((out[0].float() - out[1].float()).abs() <= 2 * HALF["f16"] * (5.5 + out[0].float().abs())).all()
    assert ((lse[0] - lse[1]).abs() <= 2 * (2.0 ** -24 * (32 * 32 + 140) + 2.0 ** -20 + 2.0 ** -23 * lse[0].abs())).all()


def test_attn_masks_that_are_no_trees(ctx):
    """Any bits count: words that see later ones, that see all, and rows without their own bit, which see nothing."""
    rng = np.random.default_rng(5)
    sizes, sets = [9, 40, 3], []
    for m in sizes:
        for j in range(m):
            s = {int(k) for k in np.flatnonzero(rng.random(m) < 0.4)} | {j}
            sets.append(frozenset(s if rng.random() < 0.8 else s - {j}))
    check_tree(ctx, tree_case(5, [9, 77, 50], sizes, 8, 2, 64, 16, "f16", sets=sets, prefix=20))
    check_tree(ctx, tree_case(5, [9, 77, 50], sizes, 16, 4, 128, 16, "bf16", sets=sets))
    check_tree(ctx, tree_case(5, [3], [3], 8, 2, 64, 16, "f16", sets=[frozenset()] * 3, prefix=40))


def test_attn_rows_of_requests_that_were_refused(ctx):
    """Without bits, whatever the length: zeros and -inf; also a length of zero or below among requests that are whole."""
    sizes = [4, 6, 2, 3]
    for kw in (dict(), dict(prefix=300), dict(prefix=30, window=7)):
        c = tree_case(6, [30, 26, 0, 3], sizes, 8, 2, 64, 16, "f16", parent=[-5] * 4 + [-1, 0, 0, 1, 1, 3] + [-5] * 2 + [-1, -1, 0], **kw)
        check_tree(ctx, c)
        c["length"] = i32([30, 26, -8, 3])
        check_tree(ctx, c)


def test_attn_lengths_below_the_rows(ctx):
    """Masks with bits over a length that holds fewer positions than the request has rows: it sees nothing."""
    check_tree(ctx, tree_case(7, [3, 9], [5, 9], 8, 2, 64, 16, "f16", parent=[-1, 0, 1, 2, 3] + trees(7, [9]), prefix=20))
    check_tree(ctx, tree_case(7, [3, 9], [5, 9], 8, 2, 64, 16, "f16", parent=[-1, 0, 1, 2, 3] + trees(7, [9]), prefix=20, window=2))


def test_attn_leaves_rows_behind_and_past_max_rows(ctx):
    check_tree(ctx, tree_case(20, [30, 12], [7, 3], 8, 2, 64, 16, "f16", prefix=20, extra_rows=5))
    c = tree_case(20, [30, 12], [7, 3], 8, 2, 64, 16, "f16", prefix=20, extra_rows=5)
    want, _, tol, _ = tree_reference(c)
    c["max_rows"] = 4
    out, _ = run_tree(ctx, c)
    rows = [0, 1, 2, 3, 7, 8, 9]
    assert ((out.cpu().double()[rows] - want[rows]).abs() <= tol[rows]).all()
    assert (out[4:7] == 7).all() and (out[10:] == 7).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("prefix,window", [(0, 0), (40, 0), (40, 5)])
def test_attn_bad_values_reach_only_rows_that_see_them(ctx, kind, bad, prefix, window):
    """An infinity or NaN among the values (and, for NaN, the keys) of one drafted word: only words that follow it get it."""
    sizes, at, base = [40], 11, 21
    c = tree_case(18, [base + 40], sizes, 8, 2, 64, 16, kind, prefix=prefix, window=window, gate=False)
    clean = run_tree(ctx, c)[0].clone()
    pid, o = int(c["table"][0, (base + at) // 16]), (base + at) % 16
    c["values"][pid, :, o, 5] = bad
    if math.isnan(bad):
        c["keys"][pid, :, o, 3] = bad
    out, _ = run_tree(ctx, c)
    hit = 0
    for r in range(40):
        order = sorted(c["sets"][r])
        dims = torch.ones(64, dtype=torch.bool, device="cuda")
        dims[5] = False
        if at in order and (not window or order.index(at) > len(order) - 1 - window):
            hit += 1
            assert (out[r, :, 5].isnan() if math.isnan(bad) else out[r, :, 5] == bad).all(), r
            assert math.isnan(bad) or torch.equal(out[r][:, dims], clean[r][:, dims]), r
        else:
            assert torch.equal(out[r], clean[r]), r
    assert 1 <= hit < 40


def test_attn_bad_pages_are_not_there(ctx):
    for page in (16, 32):
        c = tree_case(15, [70, 100, 40], [9, 30, 40], 8, 2, 64, page, "f16", prefix=80)
        c["table"][0, 0], c["table"][1, 1], c["table"][2, (40 - 1) // page], c["shared"][1] = -1, c["shape"].n_pages, 2 ** 31 - 1, -2 ** 31
        check_tree(ctx, c)


def test_attn_large_scores_scale_and_no_gate(ctx):
    check_tree(ctx, tree_case(11, [200, 131], [20, 3], 8, 2, 64, 16, "f16", prefix=150, gain=20.0))
    check_tree(ctx, tree_case(12, [50, 9], [8, 9], 8, 2, 64, 16, "f16", prefix=20, scale=0.37, gate=False))


def test_attn_row_starts_that_contradict_each_other_stay_inside(ctx):
    c = tree_case(21, [30, 12, 9], [2, 2, 2], 8, 2, 64, 16, "f16", prefix=20, window=6)
    for cu in ([-5, 2, 4, 6], [0, 2, 1, 6], [0, 2, 4, 2 ** 31 - 1], [0, -2 ** 31, 2 ** 31 - 1, 3], [6, 6, 6, 6]):
        c["cu"] = i32(cu)
        run_tree(ctx, c)
        torch.cuda.synchronize()


def test_attn_past_32_bits(ctx):
    """Pages whose offsets pass 2^32 bytes and 2^31 values."""
    H, K, D, page, pages = 4, 2, 128, 256, 36000
    c = tree_case(22, [300], [20], H, K, D, page, "f16", prefix=260)
    want = run_tree(ctx, c)[0].clone()
    far = torch.tensor([35999, 20000, 33000, 1, 30000, 34000], device="cuda")[:c["keys"].shape[0]]
    big = {k: torch.empty(pages, K, page, D, dtype=torch.float16, device="cuda") for k in ("keys", "values")}
    for k in big:
        big[k][far] = c[k]
    c.update(big, shape=nunchi_amd.PageShape(H, K, D, page, pages, dtype="f16"))
    c["table"] = torch.where(c["table"] >= 0, far[c["table"].long().clamp(min=0)].int(), c["table"])
    c["shared"] = far[c["shared"].long()].int()
    c["out"].fill_(7.0)
    assert torch.equal(run_tree(ctx, c)[0], want)


def test_attn_same_bits_every_time(ctx):
    c = tree_case(23, [2000, 1500, 300], [30, 64, 5], 8, 2, 64, 16, "f16", prefix=900)
    first = [t.clone() for t in run_tree(ctx, c)]
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, run_tree(ctx, c)))


def test_attn_of_a_chain_is_the_prompts(ctx):
    """Words in one chain are a prompt: the same keys, in an order of their own."""
    for window in (0, 12):
        c = tree_case(24, [70, 33, 5], [20, 33, 1], 8, 2, 64, 16, "f16", prefix=90, parent=trees(1, [20, 33, 1], 0.0), window=window)
        out, lse = (t.clone() for t in run_tree(ctx, c))
        want, want_lse = tb.run_attn(ctx, c)
        _, _, tol, tol_lse = tree_reference(c)
        assert ((out.double() - want.double()).abs().cpu() <= 2 * tol).all() and ((lse - want_lse).abs().cpu() <= 2 * tol_lse).all()


# ---------------------------------------------------------------- how likely words are


def run_probs(ctx, scores, temp=None, words=None, top=0, entropy=True, fill=77):
    rows, vocab = scores.shape
    t = {"logp": None if words is None else torch.full(words.shape, float(fill), device="cuda"), "entropy": torch.full((rows,), float(fill), device="cuda") if entropy else None,
         "top_words": torch.full((rows, top), fill, dtype=torch.int32, device="cuda") if top else None,
         "top_logp": torch.full((rows, top), float(fill), device="cuda") if top else None}
    work = torch.full((nunchi_amd.word_probs_work(rows, vocab, top),), 255, dtype=torch.uint8, device="cuda")
    nunchi_amd.word_probs(ctx, scores, work, temp=temp, words=words, **t)
    return {k: v.cpu().numpy() for k, v in t.items() if v is not None}


def probs_row(x, temp=1.0):
    """(log probability of every word, its tolerance, entropy, its tolerance, words in their order) of one row, in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    n = len(x)
    if not temp >= 0:
        return np.full(n, np.nan), np.zeros(n), np.nan, 0.0, order
    if not len(order):
        return np.full(n, -np.inf), np.zeros(n), 0.0, 0.0, order
    top = x[order[0]]
    lp, tol = np.full(n, -np.inf), np.zeros(n)
    if temp == 0:
        lp[order[0]] = 0.0
        return lp, tol, 0.0, 0.0, order
    ties = int((x == top).sum())
    if top == np.inf:
        lp[x == top] = -math.log(ties)
        return lp, tol + 2.0 ** -22 * math.log(ties), math.log(ties), 2.0 ** -22 * math.log(ties), order
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(x > -np.inf, (x - top) / temp, -np.inf)
    w = np.where(x == top, 0.0, np.exp(z))
    rest = w.sum()
    L = ties + rest
    log_sum = math.log(ties) + math.log1p(rest / ties)
    zz = np.where(w > 0, z, 0.0)
    s1, s2 = (w * np.abs(zz)).sum() / L, (w * zz * zz).sum() / L
    there = z > -np.inf
    lp[there] = z[there] - log_sum
    lp[lp < -3.4028235e38] = -np.inf            # (single precision ends there)
    off = 2.0 ** -22 * s1 + (2.0 ** -20 + 2.0 ** -18) * rest / L
    tol[there] = off + 2.0 ** -22 * (log_sum + np.abs(z[there])) + 2.0 ** -126
    return lp, tol, log_sum + s1, off + 2.0 ** -22 * (log_sum + s2) + 2.0 ** -17 * s1 + 2.0 ** -126, order


def check_probs(ctx, scores, temp=None, words=None, top=0):
    got = run_probs(ctx, scores, None if temp is None else dev(np.asarray(temp, np.float32)), None if words is None else i32(words), top)
    for r, x in enumerate(scores.float().cpu().numpy()):
        lp, tol, h, tol_h, order = probs_row(x, 1.0 if temp is None else float(np.float32(temp[r])))

        def close(a, b, t, what):
            assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.isinf(a), np.isinf(b)), (r, what, a, b)
            fine = np.isfinite(b)
            assert (np.abs(a[fine] - b[fine]) <= t[fine]).all(), (r, what, np.max(np.abs(a[fine] - b[fine]) - t[fine]))

        close(got["entropy"][r:r + 1].astype(np.float64), np.array([h]), np.array([tol_h]), "entropy")
        if words is not None:
            ok = (words[r] >= 0) & (words[r] < len(x))
            at = np.where(ok, words[r], 0)
            want = np.where(ok, lp[at], np.nan if temp is not None and not temp[r] >= 0 else -np.inf)
            close(got["logp"][r].astype(np.float64), want, tol[at], "logp")
        if top:
            k = min(top, len(order))
            assert np.array_equal(got["top_words"][r], np.concatenate([order[:k], np.full(top - k, -1)])), r
            want = np.concatenate([lp[order[:k]], np.full(top - k, np.nan if temp is not None and not temp[r] >= 0 else -np.inf)])
            close(got["top_logp"][r].astype(np.float64), want, np.concatenate([tol[order[:k]], np.zeros(top - k)]), "top_logp")


def random_rows(seed, rows, vocab, kind, spread=3.0, sure=12.0):
    rng = np.random.default_rng(seed)
    x = spread * rng.standard_normal((rows, vocab))
    x[np.arange(rows), rng.integers(0, vocab, rows)] += sure * rng.random(rows)
    x[::2, rng.random(vocab) < 0.02] = -np.inf
    words = rng.integers(0, vocab, (rows, 5))
    words[:, 0] = x.argmax(1)
    return dev(x.astype(np.float32)).to(TYPES[kind]), words


@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 9, 255, 2047, 2048, 2049, 8191, 8192, 8193, 16385, 32003, 97496])
@pytest.mark.parametrize("kind,top", [("f32", 5), ("f16", 20), ("bf16", 64), ("f32", 0)])
def test_probs(ctx, vocab, kind, top):
    scores, words = random_rows(vocab, 5, vocab, kind)
    check_probs(ctx, scores, [1.0, 0.7, 1.9, 0.0, 0.01], words, top)


@pytest.mark.parametrize("rows,vocab,kind", [(600, 300, "f32"), (3000, 9, "bf16"), (130, 40001, "f16"), (520, 9001, "f32")])
def test_probs_many_rows(ctx, rows, vocab, kind):
    scores, words = random_rows(rows, rows, vocab, kind)
    check_probs(ctx, scores, None, words, 3)


def test_probs_largest_vocab(ctx):
    for kind in ("f32", "bf16"):
        scores, words = random_rows(4, 2, 524288, kind)
        check_probs(ctx, scores, None, words, 64)


@pytest.mark.parametrize("top", [1, 20, 63, 64])
def test_probs_likeliest_words_of_many_parts(ctx, top):
    """The likeliest words spread evenly over the largest row, in every part's first places, and in steps from part to part."""
    i = np.arange(524288)
    x = np.stack([-(i % 8192.0), -(i % 8192) + (i // 8192) * 0.25, -(i % 8192) - (i // 8192) * 16.0, np.cos(i * 0.7)])
    check_probs(ctx, dev(x.astype(np.float32)), None, None, top)


@pytest.mark.parametrize("spread,temp", [(0.0, 1.0), (0.01, 1.0), (30.0, 1.0), (1000.0, 0.5), (1e30, 1e30), (1e-20, 1e-21), (3.0, 1e-38), (3.0, math.inf), (1e38, 1.0)])
def test_probs_scales(ctx, spread, temp):
    """From all words alike to one that has everything, and temperatures at the ends of the range."""
    for vocab in (1000, 20000):
        scores, words = random_rows(vocab, 3, vocab, "f32", spread=spread, sure=spread)
        check_probs(ctx, scores, [temp] * 3, words, 10)


@pytest.mark.parametrize("vocab", [40, 3000, 70000])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("top", [1, 30, 64])
def test_probs_equal_scores(ctx, vocab, kind, top):
    """All alike, two values, and a few values in long runs: the first indexes among equal ones."""
    rng = np.random.default_rng(vocab)
    x = np.zeros((5, vocab))
    x[1] = rng.integers(0, 2, vocab)
    x[2] = np.arange(vocab) // max(vocab // 7, 1)
    x[3] = -(np.arange(vocab) // max(vocab // 7, 1))
    x[4] = np.where(np.arange(vocab) % 2, 0.0, -0.0)
    check_probs(ctx, dev(x.astype(np.float32)).to(TYPES[kind]), None, rng.integers(0, vocab, (5, 3)), top)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_probs_likeliest_words_together(ctx, kind):
    """The likeliest words side by side, so that few threads hold them all, in order and turned round."""
    for vocab in (5000, 60000):
        for at in (0, 1234, vocab - 800):
            x = np.random.default_rng(at).standard_normal((2, vocab))
            x[0, at:at + 800] += 10 + np.arange(800) * 0.25
            x[1, at:at + 800] += 300 - np.arange(800) * 0.25
            check_probs(ctx, dev(x.astype(np.float32)).to(TYPES[kind]), None, None, 64)


def test_probs_one_word_has_nearly_everything(ctx):
    """Log probabilities and entropies far below 1 keep their digits."""
    x = np.random.default_rng(3).standard_normal((4, 50000)).astype(np.float32)
    for r, lead in enumerate((15.0, 25.0, 40.0, 60.0)):
        x[r, 777 * (r + 1)] = lead
    words = np.array([[777 * (r + 1), 5] for r in range(4)])
    check_probs(ctx, dev(x), None, words, 2)
    got = run_probs(ctx, dev(x), words=i32(words))
    assert (got["logp"][:3, 0] < 0).all() and (got["entropy"][:3] > 0).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [6, 700, 30000])
def test_probs_infinities_and_nan(ctx, vocab, kind):
    """Rows of nothing, of NaN, with some NaN, with one or several +inf, with one word left."""
    x = np.random.default_rng(8).standard_normal((8, vocab))
    x[0] = -np.inf
    x[1] = np.nan
    x[2, ::2] = np.nan
    x[3, 2] = np.inf
    x[4, [1, 3, 5]] = np.inf
    x[5] = -np.inf
    x[5, 4] = -3.0
    x[6, 1] = np.nan
    x[6, 2] = -np.inf
    x[7, [0, 5]] = [np.inf, np.nan]
    words = np.tile(np.array([1, 2, 4, 5, 0]), (8, 1))
    for temp in (None, [0.0] * 8, [0.5, -1.0, math.nan, 2.0, -0.0, -1e-30, 1.0, 1.0]):
        check_probs(ctx, dev(x.astype(np.float32)).to(TYPES[kind]), temp, words, 5)


def test_probs_words_out_of_range_and_wider_rows(ctx):
    """Words outside the table are never followed; rows of a wider table by their stride (through the C ABI)."""
    scores, _ = random_rows(9, 3, 100, "f32")
    check_probs(ctx, scores, None, np.array([[-1, 100, 2 ** 31 - 1, 5], [0, 99, -2 ** 31, 1], [101, -7, 3, 3]]), 2)
    for kind, code in (("f32", 0), ("bf16", 30)):
        for skew in (0, 1, 3):
            wide = torch.full((3 * 211 + skew,), math.nan, dtype=TYPES[kind], device="cuda")
            rows = torch.stack([wide[skew + 211 * r:skew + 211 * r + 205] for r in range(3)])
            part, _ = random_rows(10, 3, 205, kind)
            for r in range(3):
                wide[skew + 211 * r:skew + 211 * r + 205] = part[r]
            del rows
            out = {k: torch.zeros(3, 4, dtype=t, device="cuda") for k, t in (("words", torch.int32), ("logp", torch.float32))}
            work = torch.zeros(nunchi_amd.word_probs_work(3, 205, 4), dtype=torch.uint8, device="cuda")
            lib = nunchi_amd.load_library()
            assert lib.sh_word_probs(ctx.h, 3, 205, wide.data_ptr() + skew * wide.element_size(), 211, code, None, None, 0, None, None, out["words"].data_ptr(),
                                     out["logp"].data_ptr(), 4, work.data_ptr(), work.numel()) == 0
            want = run_probs(ctx, part, top=4, entropy=False)
            assert np.array_equal(out["words"].cpu().numpy(), want["top_words"]) and np.array_equal(out["logp"].cpu().numpy(), want["top_logp"])


def test_probs_outputs_one_by_one_and_repeated(ctx):
    """Each output alone is what it is among the others, the same every time."""
    scores, words = random_rows(11, 7, 33000, "f32")
    all_of = run_probs(ctx, scores, words=i32(words), top=9)
    for kw in (dict(words=i32(words), entropy=False), dict(), dict(top=9, entropy=False)):
        got = run_probs(ctx, scores, **kw)
        assert all(np.array_equal(v, all_of[k]) for k, v in got.items())
    for _ in range(5):
        again = run_probs(ctx, scores, words=i32(words), top=9)
        assert all(np.array_equal(again[k], all_of[k]) for k in again)


# ---------------------------------------------------------------- the branch that is kept


def run_take(ctx, cu, parent, words, picks, held, length, table=None, page=16, free=None, taken=None, rows=None):
    n, rows = len(cu) - 1, len(parent)
    t = {"path": i32(np.full(rows, 77)), "count": i32(np.full(n, 77)), "next": i32(np.full(n, 77)), "length": i32(np.full(n, 77))}
    kw = {}
    if table is not None:
        t["free"], t["taken"] = i32(free), i32([77])
        kw = dict(table=i32(table), page=page, free=t["free"], taken=i32([taken]), taken_out=t["taken"])
    nunchi_amd.tree_take(ctx, i32(cu), i32(parent), i32(words), i32(picks), i32(held), i32(length), t["path"], t["count"], t["next"], t["length"], **kw)
    return {k: v.cpu().numpy() for k, v in t.items()}


def take_reference(sizes, parent, words, picks, held, length, table=None, page=16, free=None, taken=None):
    out = {"path": [], "count": [], "next": [], "length": []}
    at = 0
    for i, m in enumerate(sizes):
        path, nxt = [], -1
        if m and m <= 256 and held[i] >= 0 and held[i] + m == length[i]:
            path, nxt = [0], picks[at]
            while nxt >= 0:
                child = [j for j in range(path[-1] + 1, m) if parent[at + j] == path[-1] and words[at + j] == nxt]
                if not child:
                    break
                path.append(child[0])
                nxt = picks[at + child[0]]
        out["path"] += path + [-1] * (m - len(path))
        out["count"].append(len(path))
        out["next"].append(nxt)
        out["length"].append(held[i] + len(path) if path else length[i])
        at += m
    if table is not None:
        back = [table[i][p] for i in range(len(sizes)) for p in range(min(-(-max(out["length"][i], 0) // page), len(table[i])), min(-(-max(length[i], 0) // page), len(table[i])))]
        taken = min(max(taken, 0), len(free))
        free, left = list(free), max(taken - len(back), 0)
        for k, p in enumerate(back):
            if left + k < taken:
                free[left + k] = p
        out["free"], out["taken"] = free, [left]
    return {k: np.asarray(v, np.int64) for k, v in out.items()}


def take_case(seed, sizes, vocab=50, good=0.75):
    rng = np.random.default_rng(seed)
    parent = np.array(trees(seed, sizes), np.int64).reshape(-1)
    rows = len(parent)
    words, picks = rng.integers(0, vocab, rows), rng.integers(0, vocab, rows)
    who = np.repeat(starts(sizes)[:-1], sizes)
    child = np.flatnonzero((parent >= 0) & (rng.random(rows) < good))
    picks[who[child] + parent[child]] = words[child]
    held = rng.integers(0, 500, len(sizes))
    return parent, words, picks, held


@pytest.mark.parametrize("sizes", [[1], [2, 0, 3], [8, 8], [63, 64, 65], [256, 255, 0, 1], [5] * 300, list(range(40))])
@pytest.mark.parametrize("vocab", [3, 50, 100000])
@pytest.mark.parametrize("page", [16, 64])
def test_take(ctx, sizes, vocab, page):
    parent, words, picks, held = take_case(len(sizes) + vocab, sizes, vocab)
    length = held + sizes
    cols = int((-(-length // page)).max()) + 2
    table = np.random.default_rng(2).permutation(len(sizes) * cols).reshape(-1, cols)
    free = 100000 + np.arange(len(sizes) * cols)
    for taken in (len(free), len(free) - 40):
        if taken < sum(sizes) // page + len(sizes):
            continue
        want = take_reference(sizes, parent, words, picks, held, length, table, page, free, taken)
        got = run_take(ctx, starts(sizes), parent, words, picks, held, length, table, page, free, taken)
        assert all(np.array_equal(got[k], want[k]) for k in want), [k for k in want if not np.array_equal(got[k], want[k])]
    got = run_take(ctx, starts(sizes), parent, words, picks, held, length)
    assert all(np.array_equal(got[k], want[k]) for k in got)


def test_take_first_of_equal_children_and_parents_out_of_range(ctx):
    parent = [-1, 0, 0, 0, 1, 2, 3, 9, 6, 7, -3]
    words = [5, 8, 8, 8, 9, 9, 9, 9, 4, 4, 4]
    picks = [8, 9, 9, 9, -1, 1, 4, 4, 2, 2, 2]
    want = take_reference([11], parent, words, picks, [3], [14])
    got = run_take(ctx, [0, 11], parent, words, picks, [3], [14])
    assert got["path"].tolist() == [0, 1, 4] + [-1] * 8 and got["next"].tolist() == [-1] and got["length"].tolist() == [6]
    assert all(np.array_equal(got[k], want[k]) for k in got)


def test_take_requests_that_were_refused(ctx):
    """They keep nothing and their length; more rows than 256 too. Words of -1 are never agreed with."""
    sizes = [3, 2, 257, 2]
    parent, words, picks, held = take_case(4, sizes, 3)
    length = held + sizes
    length[1] -= 2
    held[3] = -1
    table, free = np.arange(4 * 60).reshape(4, 60), np.arange(1000, 1300)
    want = take_reference(sizes, parent, words, picks, held, length, table, 16, free, 290)
    got = run_take(ctx, starts(sizes), parent, words, picks, held, length, table, 16, free, 290)
    assert all(np.array_equal(got[k], want[k]) for k in want)
    assert got["count"].tolist()[1:] == [0, 0, 0] and got["next"].tolist()[1:] == [-1, -1, -1]
    got = run_take(ctx, [0, 3], [-1, 0, 1], [5, -1, -1], [-1, -1, 3], [4], [7])
    assert got["count"].tolist() == [1] and got["next"].tolist() == [-1]


def test_take_more_pages_back_than_were_given(ctx):
    """What passes the pages that were given out is not written; nothing is taken below zero."""
    sizes = [40, 40]
    parent, words, picks, held = take_case(5, sizes, 100000, good=0.0)
    table, free = np.arange(2 * 60).reshape(2, 60) + 500, np.arange(1000, 1010)
    for taken in (0, 1, 3, 10, 2 ** 31 - 1, -4):
        want = take_reference(sizes, parent, words, picks, held, held + 40, table, 16, free, taken)
        got = run_take(ctx, [0, 40, 80], parent, words, picks, held, held + 40, table, 16, free, taken)
        assert all(np.array_equal(got[k], want[k]) for k in want), taken


def test_take_no_rows_and_most_requests(ctx):
    got = run_take(ctx, [0, 0, 0], [], [], [], [4, 9], [4, 9])
    assert got["count"].tolist() == [0, 0] and got["length"].tolist() == [4, 9] and got["next"].tolist() == [-1, -1]
    sizes = [3] * 4096
    parent, words, picks, held = take_case(6, sizes, 5)
    table = np.arange(4096 * 40).reshape(4096, 40)
    free = np.arange(9000) + 10 ** 6
    want = take_reference(sizes, parent, words, picks, held, held + 3, table, 16, free, 9000)
    got = run_take(ctx, starts(sizes), parent, words, picks, held, held + 3, table, 16, free, 9000)
    assert all(np.array_equal(got[k], want[k]) for k in want)


# ---------------------------------------------------------------- the branch's keys and values


def keep_case(seed, lens, sizes, K, D, page, kind, cols=None):
    g = torch.Generator().manual_seed(seed)
    counts = [-(-h // page) for h in lens]
    ids = torch.randperm(sum(counts) + 2, generator=g).tolist()
    table, at = torch.full((len(lens), max(counts) if cols is None else cols), -1, dtype=torch.int32), 0
    for i, k in enumerate(counts):
        table[i, :k] = torch.tensor(ids[at:at + k], dtype=torch.int32)[:table.shape[1]]
        at += k
    shape = nunchi_amd.PageShape(K, K, D, page, sum(counts) + 2, dtype=kind)
    return {"keys": torch.randn(shape.cache_shape, generator=g).to(TYPES[kind]).cuda(), "values": torch.randn(shape.cache_shape, generator=g).to(TYPES[kind]).cuda(),
            "table": table.cuda(), "lens": lens, "sizes": sizes, "length": i32(lens), "cu": i32(starts(sizes)), "shape": shape, "page": page}


def run_keep(ctx, c, path):
    nunchi_amd.page_keep(ctx, c["shape"], c["cu"], i32(path), c["length"], c["table"], c["keys"], c["values"])


def check_keep(ctx, c, path):
    want = [c["keys"].cpu(), c["values"].cpu()]
    table, page, at = c["table"].tolist(), c["page"], 0
    for i, (held, m) in enumerate(zip(c["lens"], c["sizes"])):
        base = held - m
        for j in range(m):
            k = path[at + j]
            if not j < k < m or base < 0 or m > 256 or (base + k) // page >= len(table[i]):
                continue
            a, b = (table[i][(base + p) // page] for p in (k, j))
            if 0 <= a < want[0].shape[0] and 0 <= b < want[0].shape[0]:
                for x in want:
                    x[b, :, (base + j) % page] = x[a, :, (base + k) % page]
        at += m
    run_keep(ctx, c, path)
    assert torch.equal(c["keys"].cpu(), want[0]) and torch.equal(c["values"].cpu(), want[1])


def branch(rng, m, most):
    """Places of a kept branch, 0 first, ascending."""
    if m == 0:
        return []
    n = int(rng.integers(1, min(m, most) + 1))
    p = [0] + sorted(rng.choice(np.arange(1, m), n - 1, replace=False).tolist()) if m > 1 else [0]
    return p + [-1] * (m - len(p))


@pytest.mark.parametrize("K,D,page,kind", [(2, 64, 16, "f16"), (4, 128, 32, "bf16"), (1, 32, 64, "f16"), (8, 64, 128, "bf16"), (40, 128, 16, "f16"), (3, 32, 256, "bf16")])
@pytest.mark.parametrize("most", [1, 5, 300])
def test_keep(ctx, K, D, page, kind, most):
    """Branches whose places overlap those they are moved to, across the ends of pages."""
    rng = np.random.default_rng(K + most)
    sizes = [5, 0, 64, 1, 33, 256, 2]
    lens = [m + b for m, b in zip(sizes, [0, 7, 15, 16, 17, 250, 63])]
    check_keep(ctx, keep_case(K, lens, sizes, K, D, page, kind), sum((branch(rng, m, most) for m in sizes), []))


def test_keep_every_place_one_to_the_front(ctx):
    """Each word is read from where the next is written: a chain of moves in order."""
    for m in (9, 200, 256):
        check_keep(ctx, keep_case(m, [m + 11], [m], 2, 64, 16, "f16"), list(range(1, m)) + [-1])
        check_keep(ctx, keep_case(m, [m + 11], [m], 2, 64, 16, "f16"), [min(2 * j, m - 1) for j in range(m)])


def test_keep_entries_that_move_nothing(ctx):
    """Entries at or before their own place, outside the rows, twice the same; pages that are not there; too many rows; lengths
    below the rows."""
    c = keep_case(3, [30, 40, 5, 300], [10, 12, 8, 257], 2, 64, 16, "f16")
    path = [0, 0, 5, 5, 2, -9, 10, 2 ** 31 - 1, 9, -2 ** 31] + [3, 3, 3, 3, 11, 11, 11, 11, 11, 11, 11, 11] + list(range(1, 9)) + list(range(1, 258))
    check_keep(ctx, c, path)
    c = keep_case(4, [30, 40], [20, 25], 2, 64, 16, "f16")
    c["table"][0, 1], c["table"][1, 2] = -1, c["shape"].n_pages
    check_keep(ctx, c, list(range(1, 20)) + [-1] + list(range(1, 25)) + [-1])
    check_keep(ctx, keep_case(5, [64], [40], 2, 64, 16, "f16", cols=3), list(range(3, 40)) + [-1] * 3)


def test_keep_past_32_bits(ctx):
    """Pages whose offsets pass 2^32 bytes and 2^31 values."""
    K, D, page, pages = 2, 128, 256, 36000
    shape = nunchi_amd.PageShape(K, K, D, page, pages, dtype="f16")
    keys, values = (torch.empty(shape.cache_shape, dtype=torch.float16, device="cuda") for _ in range(2))
    table = i32([[35999, 34000]])
    for x in (keys, values):
        x[35999].normal_()
        x[34000].normal_()
    want = [x[34000, :, 44].clone() for x in (keys, values)]
    nunchi_amd.page_keep(ctx, shape, i32([0, 60]), i32([0, 59] + [-1] * 58), i32([301]), table, keys, values)      # 241 + 59 -> 241 + 1
    assert all(torch.equal(x[35999, :, 242], w) for x, w in zip((keys, values), want))


# ---------------------------------------------------------------- all of them together


class Drafting:
    """A small model of one layer (a word's row, attention, scores over 400 words) whose conversations try drafted words: what it
    would say next by 64 bits, among wrong ones. `said` are each conversation's words, of which the last is not written yet."""

    def __init__(self, ctx, kind="f16", n=4):
        self.H, self.K, self.D, self.page, self.n, self.V, self.kind, self.ctx = 8, 2, 64, 16, n, 400, kind, ctx
        g = self.g = torch.Generator().manual_seed(5)
        self.rng = np.random.default_rng(5)
        pages, self.prefix = 80, 21
        self.shape = nunchi_amd.PageShape(self.H, self.K, self.D, self.page, pages, dtype=kind)
        self.keys, self.values = (torch.full(self.shape.cache_shape, math.nan, dtype=TYPES[kind], device="cuda") for _ in range(2))
        order = torch.randperm(pages, generator=g).int()
        self.shared, self.free = order[:2].cuda(), order[2:].cuda()
        ang = torch.rand(200, self.D // 2, generator=g) * 6.28
        self.rope = torch.stack([ang.cos(), ang.sin()], -1).cuda()
        self.rows_of = torch.randn(self.V, (self.H + 2 * self.K) * self.D, generator=g).cuda()
        self.out_of = torch.randn(self.H * self.D, self.V, generator=g).cuda()
        self.table = torch.full((n, 8), -1, dtype=torch.int32, device="cuda")
        self.held, self.taken = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        x = torch.randn(self.prefix, self.rows_of.shape[1], generator=g).cuda()
        slots = torch.tensor([int(self.shared[p // 16]) * 16 + p % 16 for p in range(self.prefix)]).cuda()
        nunchi_amd.page_put(ctx, self.shape, x, slots, self.keys, self.values, pos=torch.arange(self.prefix, dtype=torch.int32).cuda(), rope=self.rope)
        self.x0 = x.cpu()
        self.said, self.kept = [[7 + i] for i in range(n)], 0

    def attend(self, said):
        """(attention's output after these words [heads][D], its tolerance) in 64 bits from the rounded queries, keys and values."""
        x = torch.cat([self.x0, self.rows_of.cpu()[said]]).double().view(-1, self.H + 2 * self.K, self.D)
        cs, h = self.rope.cpu()[:len(x)], HALF[self.kind]
        as_held = lambda t: t.to(TYPES[self.kind]).double()     # noqa: E731
        q = as_held(tb.heads_reference(x[-1:, :self.H], None, 0, cs[-1:]))[0]
        k = as_held(tb.heads_reference(x[:, self.H:self.H + self.K], None, 0, cs)).repeat_interleave(self.H // self.K, 1)
        v = as_held(x[:, self.H + self.K:]).repeat_interleave(self.H // self.K, 1)
        p = torch.softmax((q[None] * k).sum(-1) / math.sqrt(self.D), 0)
        # queries and keys may round the other way where single precision falls on a tie (tests/test_gpu_batch.py, Serving.check)
        moved = 4 * h * (q[None].abs() * k.abs()).sum(-1).amax() / math.sqrt(self.D)
        return (p[..., None] * v).sum(0), ((2.01 * h + 2.0 ** -14 + moved) * v.abs().amax()).item()

    def say(self, said):
        return int((self.attend(said)[0].reshape(-1) @ self.out_of.cpu().double()).argmax())

    def buffers(self, sizes):
        rows, n, f = sum(sizes), self.n, dict(dtype=torch.int32, device="cuda")
        m = max(sizes)
        t16 = dict(dtype=TYPES[self.kind], device="cuda")
        return {"sizes": sizes, "add": i32(sizes), "len": torch.zeros(n, **f), "cu": torch.zeros(n + 1, **f), "slots": torch.zeros(rows, dtype=torch.int64, device="cuda"),
                "seq": torch.zeros(rows, **f), "taken": torch.zeros(1, **f), "parent": torch.zeros(rows, **f), "words": torch.zeros(rows, **f), "max_rows": m,
                "mask": torch.zeros(rows, (m + 31) // 32, **f), "pos": torch.zeros(rows, **f), "q": torch.zeros(rows, self.H, self.D, **t16),
                "out": torch.zeros(rows, self.H, self.D, **t16), "scores": torch.zeros(rows, self.V, device="cuda"), "picks": torch.zeros(rows, **f),
                "u": torch.zeros(rows, dtype=torch.float64, device="cuda"), "zero": torch.zeros(rows, device="cuda"), "path": torch.zeros(rows, **f), "count": torch.zeros(n, **f),
                "next": torch.zeros(n, **f), "len2": torch.zeros(n, **f), "taken2": torch.zeros(1, **f), "logp": torch.zeros(rows, 1, device="cuda"),
                "entropy": torch.zeros(rows, device="cuda"), "top": torch.zeros(rows, 3, **f), "top_logp": torch.zeros(rows, 3, device="cuda"),
                "work": torch.empty(nunchi_amd.tree_attn_work(self.shape, n, rows, 100, m, self.prefix), dtype=torch.uint8, device="cuda"),
                "swork": torch.empty(nunchi_amd.sample_work(rows, self.V), dtype=torch.uint8, device="cuda"),
                "pwork": torch.empty(nunchi_amd.word_probs_work(rows, self.V, 3), dtype=torch.uint8, device="cuda")}

    def enqueue(self, b, ctx=None):
        ctx = ctx or self.ctx
        nunchi_amd.page_plan(ctx, self.held, b["add"], self.free, self.taken, self.table, self.page, b["len"], b["cu"], b["slots"], b["seq"], b["taken"], pos0=self.prefix)
        nunchi_amd.tree_plan(ctx, b["cu"], b["parent"], self.held, b["len"], b["mask"], b["pos"], b["max_rows"], pos0=self.prefix)
        nunchi_amd.page_put(ctx, self.shape, self.rows_of[b["words"].long()], b["slots"], self.keys, self.values, q=b["q"], pos=b["pos"], rope=self.rope)
        nunchi_amd.tree_attn(ctx, self.shape, b["q"], self.keys, self.values, self.table, b["len"], b["cu"], b["mask"], b["out"], b["work"], 100, b["max_rows"],
                             prefix=self.shared, prefix_len=self.prefix)
        b["scores"].copy_(b["out"].view(-1, self.H * self.D).float() @ self.out_of)
        nunchi_amd.sample(ctx, b["scores"], b["u"], b["picks"], b["swork"], temp=b["zero"])
        nunchi_amd.word_probs(ctx, b["scores"], b["pwork"], words=b["picks"][:, None], logp=b["logp"], entropy=b["entropy"], top_words=b["top"], top_logp=b["top_logp"])
        nunchi_amd.tree_take(ctx, b["cu"], b["parent"], b["words"], b["picks"], self.held, b["len"], b["path"], b["count"], b["next"], b["len2"], table=self.table,
                             page=self.page, free=self.free, taken=b["taken"], taken_out=b["taken2"])
        nunchi_amd.page_keep(ctx, self.shape, b["cu"], b["path"], b["len"], self.table, self.keys, self.values)
        self.held.copy_(b["len2"])
        self.taken.copy_(b["taken2"])

    def draft(self, b):
        """Trees that hold the words the model would say, to a depth of the seed's, among wrong ones."""
        parent, words = [], []
        for i, m in enumerate(b["sizes"]):
            if not m:
                continue
            good, p, w, line = int(self.rng.integers(0, m)), [-1], [self.said[i][-1]], [0]
            while len(p) < m:
                if len(line) <= good and self.rng.random() < 0.5:
                    p.append(line[-1])
                    w.append(self.say(self.said[i] + [w[k] for k in line[1:]]))
                    line.append(len(p) - 1)
                else:
                    p.append(int(self.rng.integers(0, len(p))))
                    w.append(int(self.rng.integers(0, self.V)))
            parent += p
            words += w
        self.parent, self.words = parent, words
        b["parent"].copy_(i32(parent))
        b["words"].copy_(i32(words))

    def check(self, b):
        """The step's outputs against 64 bits; then what it kept is what was said."""
        sizes, picks = b["sizes"], b["picks"].tolist()
        held = [len(s) - 1 for s in self.said]
        sets = follows(self.parent, sizes)
        at = 0
        for i, m in enumerate(sizes):
            for r in range(at, at + m):
                out, tol = self.attend(self.said[i][:-1] + [self.words[at + k] for k in sorted(sets[r])])
                assert ((b["out"][r].cpu().double() - out).abs() <= tol).all()
                lp, tol, h, tol_h, order = probs_row(b["scores"][r].cpu().numpy())
                assert b["top"][r].tolist() == order[:3].tolist() and picks[r] == order[0]
                assert abs(b["logp"][r, 0].item() - lp[order[0]]) <= tol[order[0]] and abs(b["entropy"][r].item() - h) <= tol_h
            at += m
        want = take_reference(sizes, self.parent, self.words, picks, held, [h + m for h, m in zip(held, sizes)])
        for k, name in (("path", "path"), ("count", "count"), ("next", "next"), ("length", "len2")):
            assert b[name].tolist() == want[k].tolist(), k
        at = 0
        for i, m in enumerate(sizes):
            if m:
                self.said[i] += [self.words[at + k] for k in want["path"][at + 1:at + want["count"][i]]] + [int(want["next"][i])]
                self.kept += int(want["count"][i])
            at += m
        # pages: each is free, shared or some conversation's, once
        mine = [self.table[i, :-(-(len(s) - 1) // self.page)].tolist() for i, s in enumerate(self.said)]
        assert sorted(sum(mine, []) + self.shared.tolist() + self.free[self.taken.item():].tolist()) == list(range(self.shape.n_pages))

    def check_cache(self):
        """Keys and values are those of the words said, written one after the other."""
        for i, said in enumerate(self.said):
            n = len(said) - 1
            if not n:
                continue
            shape = nunchi_amd.PageShape(self.H, self.K, self.D, 256, 1, dtype=self.kind)
            k, v = (torch.zeros(shape.cache_shape, dtype=TYPES[self.kind], device="cuda") for _ in range(2))
            nunchi_amd.page_put(self.ctx, shape, self.rows_of[said[:-1]], torch.arange(n).cuda(), k, v, pos=(self.prefix + torch.arange(n, dtype=torch.int32)).cuda(),
                                rope=self.rope)
            ids = self.table[i, :-(-n // self.page)].long()
            for cache, want in ((self.keys, k), (self.values, v)):
                assert torch.equal(cache[ids].transpose(1, 2).reshape(-1, self.K, self.D)[:n], want[0].transpose(0, 1)[:n])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_drafting_run(ctx, kind):
    """Steps with trees of many sizes, some conversations pausing: plan, masks, writes, attention, picks, the kept branch, its
    moves and its pages in turn."""
    s = Drafting(ctx, kind)
    rows = 0
    for sizes in ([1, 5, 0, 9], [8, 8, 8, 8], [3, 0, 20, 1], [33, 2, 7, 12], [4, 4, 4, 4], [1, 30, 1, 2]):
        b = s.buffers(sizes)
        s.draft(b)
        s.enqueue(b)
        torch.cuda.synchronize()
        s.check(b)
        s.check_cache()
        rows += sum(sizes)
    assert 22 < s.kept < rows      # (more than each step's first words, fewer than all)


def test_drafting_step_in_a_graph():
    """One step captured and replayed, lengths, tables and free pages carried on the device, with eager work and waits between
    the replays; every replay is checked."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        s = Drafting(nunchi_amd.Context(0, stream=stream.cuda_stream))
        b = s.buffers([6, 5, 1, 4])
        s.draft(b)
        s.enqueue(b)          # (once eagerly: the plain product's library sets itself up)
        stream.synchronize()
        s.check(b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s.enqueue(b)
        for _ in range(6):
            s.draft(b)
            graph.replay()
            stream.synchronize()
            s.check(b)
            torch.randn(1000, device="cuda").sum().item()
        s.check_cache()
    stream.synchronize()


def test_streams_and_contexts(ctx):
    """The same calls from a context on another stream, two at once with work memory of their own."""
    c = tree_case(30, [700, 90], [20, 9], 8, 2, 64, 16, "f16", prefix=300)
    scores, words = random_rows(31, 9, 40000, "f32")
    want = [t.clone() for t in run_tree(ctx, c)]
    want_p = run_probs(ctx, scores, words=i32(words), top=5)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [nunchi_amd.Context(0, stream=x.cuda_stream) for x in sides]
    got, got_p = [], []
    for x, k in zip(sides, ctxs):
        with torch.cuda.stream(x):
            mine = {**c, "out": torch.full_like(c["out"], 3.0), "lse": torch.full_like(c["lse"], 3.0)}
            got.append(run_tree(k, mine))
            t = {"logp": torch.zeros(words.shape, device="cuda"), "top_words": torch.zeros(9, 5, dtype=torch.int32, device="cuda")}
            nunchi_amd.word_probs(k, scores, torch.empty(nunchi_amd.word_probs_work(9, 40000, 5), dtype=torch.uint8, device="cuda"), words=i32(words), **t)
            got_p.append(t)
    torch.cuda.synchronize()
    for g, p in zip(got, got_p):
        assert all(torch.equal(a, b) for a, b in zip(want, g))
        assert all(np.array_equal(p[k].cpu().numpy(), want_p[k]) for k in p)
    for k in ctxs:
        k.close()
