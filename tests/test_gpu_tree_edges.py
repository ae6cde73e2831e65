"""The operators for drafted words where plans, masks, pages and lengths are not the ordinary ones: what one of them refuses, the others do not
take for whole. References and tolerances are tests/test_gpu_tree.py's."""
import math

import numpy as np
import pytest

import nunchi_amd

torch = pytest.importorskip("torch")
import test_gpu_tree as tt  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return nunchi_amd.Context(0, stream=torch.cuda.current_stream().cuda_stream)


def test_take_first_rows_with_a_parent(ctx):
    """A first row whose parent is not before it has no bits in the plan, nor has what follows it: nothing of the request is kept, the
    positions of its rows and their pages go back. The requests beside it do not notice."""
    sizes, held = [3, 20, 4, 2, 3], [40, 30, 15, 16, 9]
    for first in (0, 2, -2, 2 ** 31 - 1, -2 ** 31):
        parent, words, picks, _ = tt.take_case(8, sizes, 2)
        for at in (3, 23):
            parent[at] = first
        length = [h + m for h, m in zip(held, sizes)]
        table, free = np.arange(5 * 6).reshape(5, 6) + 400, np.arange(900, 960)
        want = tt.take_reference(sizes, parent, words, picks, held, length, table, 16, free, 40)
        _, pos = tt.run_plan(ctx, tt.starts(sizes), parent, held, length, 32)
        assert (pos[3:27] == -1).all() and (pos[:3] >= 0).all() and (pos[27:] >= 0).all()
        got = tt.run_take(ctx, tt.starts(sizes), parent, words, picks, held, length, table, 16, free, 40)
        assert got["count"][1] == got["count"][2] == 0 and got["next"][1] == got["next"][2] == -1 and (got["path"][3:27] == -1).all()
        assert got["length"][1:3].tolist() == held[1:3]
        other = [0, 3, 4]
        assert got["count"][other].tolist() == want["count"][other].tolist() and got["length"][other].tolist() == want["length"][other].tolist()
        # pages of positions 30 .. 49 (16 a page: two behind the first two) and 15 .. 18 (one behind the first)
        back = sum((table[i, -(-int(got["length"][i]) // 16):-(-length[i] // 16)].tolist() for i in range(5)), [])
        assert [int(x) for x in table[1, 2:4]] == [x for x in back if x in table[1]] and [int(table[2, 1])] == [x for x in back if x in table[2]]
        assert got["taken"].tolist() == [40 - len(back)] and got["free"][40 - len(back):40].tolist() == back


class Planned(tt.Drafting):
    """Conversations whose steps tell tree_take what tree_plan refused: those of more rows than the step's max_rows."""

    def buffers(self, sizes, max_rows):
        b = super().buffers(sizes)
        b.update(max_rows=max_rows, mask=torch.zeros(sum(sizes), (max_rows + 31) // 32, dtype=torch.int32, device="cuda"))
        return b

    def enqueue(self, b, ctx=None):
        take = nunchi_amd.tree_take
        try:
            nunchi_amd.tree_take = lambda *args, **kw: take(*args, **kw, pos=b["pos"])
            super().enqueue(b, ctx)
        finally:
            nunchi_amd.tree_take = take

    def check(self, b):
        sizes = [m if m <= b["max_rows"] else 0 for m in b["sizes"]]
        kept = np.repeat([m > 0 for m in sizes], b["sizes"])
        rows = torch.from_numpy(np.flatnonzero(kept)).cuda()
        self.parent, self.words = ([x for x, k in zip(y, kept) if k] for y in (self.parent, self.words))
        super().check({**b, "sizes": sizes, **{k: b[k][rows] for k in ("out", "scores", "picks", "logp", "entropy", "top", "path")}})
        assert (b["path"].cpu()[torch.from_numpy(~kept)] == -1).all() and (b["pos"].cpu()[torch.from_numpy(~kept)] == -1).all()


@pytest.mark.parametrize("many", [33, 70, 100])
def test_step_with_a_request_that_the_plan_refused(many):
    """One conversation drafts more words than the step's max_rows: page_plan gives it pages, tree_plan no bits. It keeps its length, its
    pages go back, and its next step reads what it held."""
    s = Planned(nunchi_amd.Context(0, stream=torch.cuda.current_stream().cuda_stream))
    for sizes, max_rows in [([4, 5, 3, 9], 9), ([9, many, 3, 5], 32), ([5, 8, 1, 3], 8), ([many, many, many, many], many - 1), ([2, 6, 7, 8], 64)]:
        b = s.buffers(sizes, max_rows)
        s.draft(b)
        before = [len(x) for x in s.said]
        s.enqueue(b)
        torch.cuda.synchronize()
        s.check(b)
        assert [len(x) == k for x, k in zip(s.said, before)] == [m > max_rows for m in sizes]
        s.check_cache()


@pytest.mark.parametrize("page", [16, 64])
def test_take_requests_that_the_plan_refused(ctx, page):
    """Those of more rows than max_rows (and than 256) keep nothing and the length before the step; their pages go back."""
    sizes, max_rows = [5, 40, 257, 0, 40, 39, 300, 2] * 9, 39
    parent, words, picks, held = tt.take_case(11, sizes, 2)
    length = held + sizes
    length[3], held[7] = length[3] - 1, -1       # (refused by the page plan: the length stays)
    _, pos = tt.run_plan(ctx, tt.starts(sizes), parent, held, length, max_rows)
    table = np.random.default_rng(3).permutation(len(sizes) * 60).reshape(-1, 60)
    free, t = np.arange(3000) + 10 ** 6, {k: tt.i32(np.full(v, 77)) for k, v in dict(path=len(parent), count=len(sizes), next=len(sizes), length=len(sizes)).items()}
    refused = np.array([m > max_rows for m in sizes])
    want = tt.take_reference(sizes, parent, words, picks, held, np.where(refused, held, length))
    back = [table[i, p] for i in range(len(sizes)) for p in range(-(-max(want["length"][i], 0) // page), -(-max(length[i], 0) // page))]
    for at in (None, 3000):
        got, kw = tt.i32(free), {}
        if at:
            kw = dict(table=tt.i32(table), page=page, free=got, taken=tt.i32([at]), taken_out=tt.i32([77]))
        nunchi_amd.tree_take(ctx, *(tt.i32(x) for x in (tt.starts(sizes), parent, words, picks, held, length)), t["path"], t["count"], t["next"], t["length"],
                             pos=tt.i32(pos), **kw)
        assert all(np.array_equal(t[k].cpu().numpy(), want[k]) for k in t), [k for k in t if not np.array_equal(t[k].cpu().numpy(), want[k])]
        if at:
            assert kw["taken_out"].item() == at - len(back) and got[at - len(back):].tolist() == back


@pytest.mark.parametrize("prefix,window", [(0, 0), (0, 3), (0, 40), (50, 7), (50, 64), (130, 100)])
@pytest.mark.parametrize("D,kind", [(64, "f16"), (128, "bf16")])
def test_attn_bits_behind_the_rows(ctx, D, kind, prefix, window):
    """Bits of places that the request does not have move neither its rows' positions nor their windows."""
    sizes, max_rows = [5, 40, 1, 32, 33, 64], 64
    c = tt.tree_case(9, [30, 90, 8, 32, 70, 64], sizes, 8, 2, D, 16, kind, prefix=prefix, window=window, max_rows=max_rows)
    mask, rng = c["mask"].cpu().numpy().view(np.uint64).reshape(-1).copy(), np.random.default_rng(2)
    for r, m in enumerate(np.repeat(sizes, sizes)):
        if m < 64:
            mask[r] |= np.uint64(int(rng.integers(0, 2 ** 63)) >> m << m) | np.uint64(1 << 63)
    c["mask"].copy_(torch.from_numpy(mask.view(np.int32).reshape(-1, 2)))
    tt.check_tree(ctx, c)


@pytest.mark.parametrize("n", [2, 40])
def test_take_of_a_table_without_columns(ctx, n):
    """Nothing goes back, and what was taken is written all the same."""
    sizes = [0] * n
    for free, taken, left in (([], 0, 0), ([5, 6, 7], 2, 2), ([5, 6, 7], 9, 3), ([], 4, 0)):
        got = tt.run_take(ctx, tt.starts(sizes), [], [], [], [3] * n, [3] * n, np.zeros((n, 0)), 16, np.array(free), taken)
        assert got["taken"].tolist() == [left] and got["free"].tolist() == free and got["length"].tolist() == [3] * n


@pytest.mark.parametrize("prefix", [0, 20, 7000])
def test_rows_of_a_request_past_max_rows(ctx, prefix):
    """Without bits: zeros and -inf for the first max_rows of them, whatever the keys, and the rows past these stay as they were. Writes
    without a rotation table go by the slots; with one they pass such rows over."""
    sizes, lens, max_rows = [3, 40, 2] + [1] * 16, [30, 90, 9] + [5] * 16, 32
    parent = tt.trees(3, sizes)
    sets = [None if 3 <= r < 43 else s for r, s in enumerate(tt.follows(parent, sizes))]
    c = tt.tree_case(3, lens, sizes, 8, 2, 64, 16, "f16", prefix=prefix, gate=False, max_rows=max_rows, sets=sets)
    mask, pos = tt.run_plan(ctx, tt.starts(sizes), parent, [a - b for a, b in zip(lens, sizes)], lens, max_rows)
    assert (mask[3:43] == 0).all() and (pos[3:43] == -1).all()
    assert np.array_equal(mask, c["mask"].cpu().numpy())
    out, lse = tt.run_tree(ctx, c)
    want, want_lse, tol, tol_lse = tt.tree_reference(c)
    rows = [r for r in range(sum(sizes)) if not 35 <= r < 43]
    assert ((out.cpu().double()[rows] - want[rows]).abs() <= tol[rows]).all() and (out[3:35] == 0).all() and (lse[3:35] == -float("inf")).all()
    assert (out[35:43] == 7).all() and (lse[35:43] == 7).all()

    shape = nunchi_amd.PageShape(1, 1, 32, 16, 4, dtype="f16")
    qkv, slots, at = torch.ones(8, 96, device="cuda"), torch.arange(8).cuda() * 5, tt.i32([0, -1, 1, -1, -1, 2, 3, -1])
    for rope in (None, torch.ones(5, 16, 2, device="cuda")):
        keys, values = (torch.zeros(shape.cache_shape, dtype=torch.float16, device="cuda") for _ in range(2))
        nunchi_amd.page_put(ctx, shape, qkv, slots, keys, values, pos=at, rope=rope)
        there = (values.view(-1, 32)[slots] == 1).all(1)
        assert there.tolist() == [rope is None or p >= 0 for p in at.tolist()]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_attn_many_small_weights(ctx, kind, D):
    """20000 keys of weights 2^-25.5 of the largest, whose value is 0 and which the first block has: the output is the small ones' sum, as
    close as page_attn's. Each weight is rounded by half a step (h, or 2^-25 below 2^-14 in f16: here 2^-25.52 + 11, the word's own 17.6875),
    the result by h."""
    N, n, page, h = 20000, 512, 16, tt.HALF[kind]
    pages = N // page
    keys, values = torch.zeros(pages, 2, page, D, dtype=tt.TYPES[kind], device="cuda"), torch.ones(pages, 2, page, D, dtype=tt.TYPES[kind], device="cuda")
    q = torch.zeros(n, 2, D, dtype=tt.TYPES[kind], device="cuda")
    q[..., 0] = 1
    keys[0, :, 5, 0] = 17.6875
    values[0, :, 5] = 0
    shape = nunchi_amd.PageShape(2, 2, D, page, pages, dtype=kind, scale=1.0)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(n, 1)       # (all requests read the same pages)
    out, work = torch.empty_like(q), torch.empty(nunchi_amd.tree_attn_work(shape, n, n, N, 1), dtype=torch.uint8, device="cuda")
    nunchi_amd.tree_attn(ctx, shape, q, keys, values, table, tt.i32([N] * n), tt.i32(range(n + 1)), tt.i32([[1]] * n), out, work, N, 1)
    e = math.exp(-keys[0, 0, 5, 0].item())
    want = (N - 1) * e / (1 + (N - 1) * e)
    assert ((out.double() / want - 1).abs() <= 2 * h + 2.0 ** -25 / 2.0 ** -14.52 + 2.0 ** -19).all(), out.double().mean().item() / want
