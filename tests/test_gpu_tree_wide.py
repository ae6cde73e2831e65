"""Every kernel of tree_attn (tests/tree_cases.py: workgroups of their own for the shared positions, one, two and four column groups, parts) against a
reference in 64 bits, request by request on the GPU: plain trees, windows, rows without bits, masks that are no trees, pages that are not there,
lengths below the rows, rows behind the last request's, infinities and NaN.

Tolerances as tests/test_gpu_tree.py derives them: scores of D products in 32 bits, their exponentials and sums (`off`), half a step for each weight's
rounding to 16 bits for its product with the values and for the result's. f16 weights are 2^11 of the running maximum's, so those below 2^-14 are off by
2^-36 of it each."""
import math

import numpy as np
import pytest

import nunchi_amd
import tree_cases

torch = pytest.importorskip("torch")
import test_gpu_tree as tt  # noqa: E402

pytestmark = pytest.mark.gpu

CASES = tree_cases.cases()
HALF = tt.HALF


@pytest.fixture(scope="module")
def ctx():
    return nunchi_amd.Context(0, stream=torch.cuda.current_stream().cuda_stream)


def make(c, kind, seed, **kw):
    return tt.tree_case(seed, c["lens"], c["sizes"], c["H"], c["K"], c["D"], c["page"], kind, prefix=c["prefix"], window=c["window"], **kw)


def reference(c):
    """(out, lse, tolerance of out, of lse) in 64 bits."""
    H, K, D, page = c["dims"]
    rows, L0, window, G = c["rows"], c["prefix"], c["window"], H // K
    f64 = dict(dtype=torch.float64, device="cuda")
    out, lse = torch.zeros(rows, H, D, **f64), torch.full((rows, H), -math.inf, **f64)
    tol, tol_lse = torch.zeros(rows, H, 1, **f64), torch.zeros(rows, H, **f64)
    shared = c["shared"].long().repeat_interleave(page)[:L0] if L0 else torch.zeros(0, dtype=torch.int64, device="cuda")
    r0 = 0
    for i, held in enumerate(c["lens"]):
        held, m = max(held, 0), c["counts"][i]
        base, r0 = held - m, r0 + m
        if m == 0 or base < 0:
            continue
        ids = torch.cat([shared, c["table"][i].long().repeat_interleave(page)[:held]])
        at = torch.cat([torch.arange(L0, device="cuda"), torch.arange(held, device="cuda")]) % page
        known = (ids >= 0) & (ids < c["keys"].shape[0])
        ids = torch.where(known, ids, 0)
        seen = torch.zeros(m, L0 + held, dtype=torch.bool)
        for j in range(m):
            words = sorted(c["sets"][r0 - m + j] or ())
            if j not in words:
                continue
            seen[j, :L0 + base] = True
            if window:
                seen[j, :max(L0 + base + len(words) - window, 0)] = False
                words = words[-window:]
            seen[j, L0 + base + torch.tensor(words)] = True
        seen = seen.cuda() & known
        live = seen.any(1)
        if not live.any():
            continue
        for g in range(K):
            k, v = (torch.where(known[:, None], c[x][ids, g, at].double(), 0.0) for x in ("keys", "values"))
            q = c["q"][r0 - m:r0, g * G:(g + 1) * G].double()
            kt = k.t().contiguous()
            for h in range(G):
                s = (q[:, h] @ kt * c["scale"]).masked_fill(~seen, -math.inf)[live]
                size = (q[:, h].abs() @ kt.abs() * c["scale"]).masked_fill(~seen, 0.0)[live].amax(1)
                most = s.masked_fill(s == -math.inf, 0.0).abs().amax(1)
                top = s.amax(1)
                e = torch.exp(s - top[:, None])
                n, at_h = seen[live].sum(1), g * G + h
                who = torch.arange(r0 - m, r0, device="cuda")[live]
                lse[who, at_h] = top + torch.log(e.sum(1))
                out[who, at_h] = (e / e.sum(1, keepdim=True)) @ v
                off = 2.0 ** -24 * (D * size + 3 * most / math.log(2) + n / 128 + 16) + 2.0 ** -20
                tol_lse[who, at_h] = off + 2.0 ** -23 * lse[who, at_h].abs()
                under = 2.0 ** -36 * n if c["kind"] == "f16" else 0.0
                largest = v.abs().amax(1).expand(m, -1).masked_fill(~seen, 0.0)[live].amax(1)
                tol[who, at_h, 0] = (HALF[c["kind"]] * 1.01 + under + 2 * off) * largest
    if c["gate"] is not None:
        f = torch.sigmoid(c["gate"].double()[:rows])[..., None]
        out, tol = out * f, tol * f
    return out, lse, tol + HALF[c["kind"]] * out.abs() + 2.0 ** -25, tol_lse


def check(ctx, c):
    out, lse = tt.run_tree(ctx, c)
    rows = c["rows"]
    got, got_lse = out[:rows].double(), lse[:rows].double()
    want, want_lse, tol, tol_lse = reference(c)
    assert torch.isfinite(got).all()
    assert ((got - want).abs() - tol).max().item() <= 0
    none = want_lse == -math.inf
    assert torch.equal(got_lse == -math.inf, none) and (got[none] == 0).all()
    assert ((got_lse - want_lse).abs() <= tol_lse)[~none].all()
    assert (out[rows:] == 7).all() and (lse[rows:] == 7).all(), "rows behind the last request's"


def odd_masks(c, seed):
    """Some rows without bits, some that see later words, some words whose parent is not before them."""
    rng = np.random.default_rng(seed)
    parent = tt.trees(seed, c["sizes"])
    for r in np.flatnonzero(rng.random(len(parent)) < 0.1):
        parent[r] = 10 ** 6
    sets, at = tt.follows(parent, c["sizes"]), 0
    for m in c["sizes"]:
        for j in range(m):
            if rng.random() < 0.15:
                s = {int(k) for k in np.flatnonzero(rng.random(m) < 0.4)}
                sets[at + j] = frozenset(s | {j} if rng.random() < 0.7 else s - {j})
        at += m
    return sets


def test_reference_is_the_row_by_row_one(ctx):
    """The reference here against tests/test_gpu_tree.py's, which goes row by row on the CPU."""
    for window in (0, 5, 30):
        c = tt.tree_case(3, [40, 30, 5, 0, 20], [9, 30, 5, 0, 1], 8, 2, 64, 16, "f16", prefix=40, window=window)
        c["table"][1, 0], c["shared"][1] = -1, 2 ** 30
        # (the tolerances differ by what f16 weights are off by: 2^-33 and 2^-36 of the largest value, below 6, for each of 110 keys at most)
        for a, b, most in zip(reference(c), tt.tree_reference(c), (1e-12, 1e-12, 110 * 6 * 2.0 ** -33, 1e-12)):
            off = torch.where(a.cpu() == b, torch.zeros_like(b), (a.cpu() - b).abs()).max().item()
            assert off <= most


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("c", CASES, ids=tree_cases.name)
def test_trees(ctx, c, kind):
    """Trees of every shape; the same call gives the same bits."""
    x = make(c, kind, c["prefix"] + c["window"] + c["D"], extra_rows=3)
    check(ctx, x)
    first = [t.clone() for t in (x["out"], x["lse"])]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, tt.run_tree(ctx, x)))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("c", CASES, ids=tree_cases.name)
def test_masks_pages_and_lengths(ctx, c, kind):
    """Rows without bits, masks that are no trees, missing pages, and a length below its request's rows, all at once."""
    seed = c["prefix"] + c["window"] + c["D"] + 1
    x = make(c, kind, seed, sets=odd_masks(c, seed))
    rng = np.random.default_rng(seed)
    n = len(c["sizes"])
    for i in rng.choice(n, max(n // 4, 1), replace=False):
        x["table"][i, int(rng.integers(0, x["table"].shape[1]))] = int(rng.choice([-1, x["shape"].n_pages, 2 ** 31 - 1, -2 ** 31]))
    if c["prefix"]:
        x["shared"][rng.integers(0, x["shared"].shape[0], 2)] = -3
        x["shared"][-1] = x["shape"].n_pages
    short = int(np.argmax(np.array(c["sizes"]) * (np.array(c["lens"]) < 400)))       # (its length holds fewer positions than its rows)
    x["lens"][short] = c["sizes"][short] - 1
    x["length"] = tt.i32(x["lens"])
    check(ctx, x)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("c", [c for c in CASES if not c["window"] or c["kernel"][0]], ids=tree_cases.name)
def test_bad_values_reach_only_rows_that_see_them(ctx, c, bad):
    """An infinity or NaN among the values (and, for NaN, the keys) of a drafted word of every other request, and, where windows begin among the shared
    positions, of one of these that some rows see: only rows that see one get it; the others' bits do not change."""
    kind = "f16" if math.isinf(bad) else "bf16"
    x = make(c, kind, 5, gate=False)
    clean = tt.run_tree(ctx, x)[0].clone()
    H, K, D, page = x["dims"]
    hit, at, L0 = torch.zeros(x["rows"], dtype=torch.bool), 0, c["prefix"]
    shared_bad = L0 - c["window"] + 30 if 30 < c["window"] <= L0 + 30 else None       # (rows at positions from L0 + 30 on do not see it)
    if shared_bad is not None:
        pid, o = int(x["shared"][shared_bad // page]), shared_bad % page
        x["values"][pid, :, o, 5] = bad
    for i, m in enumerate(c["sizes"]):
        base, nth = c["lens"][i] - m, m // 2
        if m and i % 2 == 0:
            pid, o = int(x["table"][i, (base + nth) // page]), (base + nth) % page
            x["values"][pid, :, o, 5] = bad
            if math.isnan(bad):
                x["keys"][pid, :, o, 3] = bad
        for j in range(m):
            words = sorted(x["sets"][at + j])
            me = L0 + base + len(words) - 1
            hit[at + j] = i % 2 == 0 and nth in (words[-c["window"]:] if c["window"] else words)
            if shared_bad is not None and shared_bad > me - c["window"]:
                hit[at + j] = True
        at += m
    out, hit = tt.run_tree(ctx, x)[0], hit.cuda()
    assert torch.equal(out[~hit], clean[~hit]) and hit.any() and not hit.all()
    assert (out[hit][..., 5].isnan() if math.isnan(bad) else out[hit][..., 5] == bad).all()
    if not math.isnan(bad):
        dims = [d for d in range(D) if d != 5]
        assert torch.equal(out[hit][..., dims], clean[hit][..., dims])
