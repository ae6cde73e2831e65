"""Refusals of the operators for drafted words (sh_tree_plan, sh_tree_attn, sh_word_probs, sh_tree_take, sh_page_keep) that need
no GPU: every check below comes before the context or any buffer is touched, so the context and the buffers are addresses only."""
import ctypes as C
from types import SimpleNamespace

import pytest

import nunchi_amd
from test_batch_args import ARG, BAD_SHAPES, BASE, _lib, at, shape


PLAN = dict(ctx=BASE, n=4, rows=9, cu=at(0), parent=at(1), held=at(2), len=at(3), max_rows=40, mask=at(4), pos=at(5), pos0=0)


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(n=0), dict(n=1 << 24), dict(rows=-1), dict(cu=None), dict(parent=None), dict(held=None), dict(len=None),
                                 dict(max_rows=0), dict(max_rows=257), dict(mask=None), dict(pos=None), dict(pos0=-1),
                                 # an output over an input, or over the other output
                                 dict(mask=at(1)), dict(mask=at(0) + 16), dict(pos=at(2) + 12), dict(pos=at(3)), dict(pos=at(4) + 68), dict(mask=at(5) + 32)], ids=str)
def test_plan_refused(bad):
    assert _lib().sh_tree_plan(*{**PLAN, **bad}.values()) == ARG
    assert b"sh_tree_plan" in _lib().sh_last_error()


@pytest.mark.parametrize("bad", BAD_SHAPES, ids=str)
def test_shapes_refused(bad):
    L, size, s = _lib(), C.c_size_t(7), shape(**bad)
    assert L.sh_tree_attn_work(C.byref(s), 1, 1, 1, 0, 10, C.byref(size)) == ARG
    assert L.sh_tree_attn(BASE, C.byref(s), 1, 1, at(9), 1, at(8), at(0), at(1), at(2), None, 0, at(3), 4, at(4), 10, None, at(5), None, at(6), 1 << 20) == ARG
    assert L.sh_page_keep(BASE, C.byref(s), 1, 1, at(0), at(1), at(2), at(3), 4, at(4), at(5)) == ARG
    assert b"sh_page_keep" in L.sh_last_error()


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(n=0), dict(rows=-1), dict(cu=None), dict(max_rows=0), dict(max_rows=257), dict(mask=None), dict(q=None),
                                 dict(q=at(0) + 8), dict(keys=None), dict(keys=at(1) + 2), dict(values=None), dict(values=at(2) + 8), dict(prefix=None),
                                 dict(prefix_len=-1), dict(prefix_len=(1 << 31) - 1), dict(table=None), dict(cols=-1), dict(len=None), dict(max_len=-1),
                                 dict(out=None), dict(out=at(6) + 2), dict(work=None), dict(work=at(7) + 64), dict(bytes=100),
                                 # an output over an input, or over another output
                                 dict(out=at(0)), dict(out=at(1) + 64), dict(out=at(2)), dict(work=at(5)), dict(lse=at(6)), dict(lse=at(0) + 32), dict(lse=at(7) + 256),
                                 dict(gate=at(6) + 16), dict(out=at(3)), dict(out=at(4) + 112), dict(cu=at(7)), dict(mask=at(6) + 32), dict(mask=at(7) - 4)], ids=str)
def test_attn_refused(bad):
    s, size = shape(), C.c_size_t()
    assert _lib().sh_tree_attn_work(C.byref(s), 4, 9, 5, 4096, 90, C.byref(size)) == 0 and size.value > 256
    v = {**dict(ctx=BASE, shape=C.byref(s), n=4, rows=9, cu=at(8), max_rows=5, mask=at(9), q=at(0), keys=at(1), values=at(2), prefix=at(3), prefix_len=4096,
                table=at(4), cols=8, len=at(5), max_len=90, gate=None, out=at(6), lse=None, work=at(7), bytes=size.value), **bad}
    assert _lib().sh_tree_attn(*v.values()) == ARG


def test_attn_launches_that_are_too_large_are_refused():
    s, size = shape(n_head=65536, n_kv=65536, n_pages=1000), C.c_size_t()
    assert _lib().sh_tree_attn_work(C.byref(s), 40000, 40000, 1, 0, 100, C.byref(size)) == ARG
    assert b"fewer rows" in _lib().sh_last_error()


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(rows=-1), dict(rows=1 << 24), dict(vocab=0), dict(vocab=524289), dict(scores=None), dict(scores=at(0) + 2), dict(ld=99),
                                 dict(type=3), dict(words=None), dict(n_words=-1), dict(logp=None), dict(top_words=None, top_logp=None), dict(n_top=-1),
                                 dict(n_top=65), dict(work=None), dict(work=at(7) + 128), dict(bytes=16),
                                 # an output over an input, or over another output
                                 dict(logp=at(0) + 64), dict(entropy=at(1)), dict(top_words=at(2) + 8), dict(top_logp=at(3) + 12), dict(entropy=at(3) + 20),
                                 dict(top_words=at(6)), dict(work=at(0)), dict(work=at(4))], ids=str)
def test_probs_refused(bad):
    size = C.c_size_t()
    assert _lib().sh_word_probs_work(2, 100, 5, C.byref(size)) == 0
    v = {**dict(ctx=BASE, rows=2, vocab=100, scores=at(0), ld=100, type=0, temp=at(1), words=at(2), n_words=3, logp=at(3), entropy=at(4), top_words=at(5),
                top_logp=at(6), n_top=5, work=at(7), bytes=size.value), **bad}
    assert _lib().sh_word_probs(*v.values()) == ARG


@pytest.mark.parametrize("rows,vocab,top", [(0, 1, 0), (1, 1, 64), (1, 524288, 64), (300, 97496, 5), (5000, 8192, 1)])
def test_probs_work_holds_every_part(rows, vocab, top):
    """16 bytes of sums and 8 a word of each part: parts of 2048 or 8192 words."""
    size = C.c_size_t()
    assert _lib().sh_word_probs_work(rows, vocab, top, C.byref(size)) == 0
    each = 16 + 8 * max(top, 1)
    assert size.value % 256 == 0 and size.value >= max(256, rows * -(-vocab // 8192) * each)
    assert size.value <= 1024 + rows * -(-vocab // 2048) * each


TAKE = dict(ctx=BASE, n=4, rows=9, cu=at(0), parent=at(1), words=at(2), picks=at(3), held=at(4), len=at(5), path=at(6), count=at(7), next=at(8), len_out=at(9),
            page=16, table=at(10), cols=8, free=at(11), n_free=20, taken=at(12), taken_out=at(13))


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(n=0), dict(n=4097), dict(rows=-1), *[{k: None} for k in ("cu", "parent", "words", "picks", "held", "len",
                                 "path", "count", "next", "len_out", "free", "taken", "taken_out")], dict(page=24), dict(cols=-1), dict(n_free=-1),
                                 # an output over an input, or over another output
                                 dict(path=at(1)), dict(count=at(0) + 16), dict(next=at(3) + 32), dict(len_out=at(5)), dict(free=at(10) + 124), dict(taken_out=at(12)),
                                 dict(free=at(5) - 76), dict(count=at(7), next=at(7) + 12), dict(taken_out=at(11) + 76), dict(len_out=at(4) + 12)], ids=str)
def test_take_refused(bad):
    assert _lib().sh_tree_take(*{**TAKE, **bad}.values()) == ARG
    assert b"sh_tree_take" in _lib().sh_last_error()


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(n=0), dict(n=1 << 24), dict(rows=-1), dict(cu=None), dict(path=None), dict(len=None), dict(table=None), dict(cols=-1),
                                 dict(keys=None), dict(keys=at(4) + 2), dict(values=None), dict(values=at(5) + 8),
                                 dict(keys=at(0)), dict(keys=at(1) - 16), dict(values=at(2)), dict(values=at(3) + 112), dict(keys=at(5) + 64)], ids=str)
def test_keep_refused(bad):
    s = shape()
    v = {**dict(ctx=BASE, shape=C.byref(s), n=4, rows=9, cu=at(0), path=at(1), len=at(2), table=at(3), cols=8, keys=at(4), values=at(5)), **bad}
    assert _lib().sh_page_keep(*v.values()) == ARG


def test_no_rows_is_no_work():
    L, s = _lib(), shape()
    assert L.sh_tree_plan(BASE, 2, 0, at(0), None, None, None, 8, None, None, 0) == 0
    assert L.sh_tree_attn(BASE, C.byref(s), 2, 0, at(1), 1, None, None, None, None, None, 0, None, 0, None, 0, None, None, None, None, 0) == 0
    assert L.sh_word_probs(BASE, 0, 100, None, 100, 0, None, None, 0, None, None, None, None, 0, None, 0) == 0
    assert L.sh_page_keep(BASE, C.byref(s), 2, 0, None, None, None, None, 0, None, None) == 0


def test_tensors_are_checked():
    """Types, shapes and places of tensors, before the call: host tensors and a context that says that is where it is."""
    torch = pytest.importorskip("torch")
    ctx = SimpleNamespace(h=SimpleNamespace(value=BASE), device=-1)

    def i(*size):
        return torch.zeros(size, dtype=torch.int32)

    def f(*size):
        return torch.zeros(size)

    plan = dict(cu=i(5), parent=i(0), held=i(4), length=i(4), mask=i(0, 2), pos=i(0), max_rows=40)
    nunchi_amd.tree_plan(ctx, **plan)          # (no rows: nothing is enqueued)
    for bad, error in [(dict(cu=i(1)), ValueError), (dict(cu=f(5)), TypeError), (dict(mask=i(0, 1)), ValueError), (dict(mask=i(0)), ValueError), (dict(held=i(5)), ValueError),
                       (dict(pos=i(1)), ValueError), (dict(max_rows=257), ValueError), (dict(max_rows=0), ValueError), (dict(parent=None), ValueError)]:
        with pytest.raises(error):
            nunchi_amd.tree_plan(ctx, **{**plan, **bad})
    s = shape()
    cache = torch.zeros(s.cache_shape, dtype=torch.float16)
    keep = dict(cu=i(5), path=i(0), length=i(4), table=i(4, 3), keys=cache, values=cache.clone())
    nunchi_amd.page_keep(ctx, s, **keep)
    for bad, error in [(dict(keys=cache[1:]), ValueError), (dict(values=cache.bfloat16()), TypeError), (dict(table=i(5, 3)), ValueError), (dict(length=i(3)), ValueError),
                       (dict(path=f(0)), TypeError), (dict(keys=cache.transpose(1, 2).contiguous().transpose(1, 2)), ValueError)]:
        with pytest.raises(error):
            nunchi_amd.page_keep(ctx, s, **{**keep, **bad})
    probs = dict(scores=f(0, 50), work=torch.zeros(256, dtype=torch.uint8), words=i(0, 3), logp=f(0, 3), entropy=f(0), top_words=i(0, 4), top_logp=f(0, 4))
    nunchi_amd.word_probs(ctx, **probs)
    for bad, error in [(dict(words=None), ValueError), (dict(logp=f(0, 2)), ValueError), (dict(top_logp=f(0, 5)), ValueError), (dict(entropy=f(1)), ValueError),
                       (dict(scores=f(0, 50).double()), TypeError), (dict(words=f(0, 3)), TypeError), (dict(temp=f(1)), ValueError)]:
        with pytest.raises(error):
            nunchi_amd.word_probs(ctx, **{**probs, **bad})
    q = torch.zeros(0, 8, 64, dtype=torch.float16)
    attn = dict(q=q, keys=cache, values=cache.clone(), table=i(4, 3), length=i(4), cu=i(5), mask=i(0, 2), out=q.clone(), work=torch.zeros(256, dtype=torch.uint8),
                max_len=30, max_rows=40)
    nunchi_amd.tree_attn(ctx, s, **attn)
    for bad, error in [(dict(mask=i(0, 1)), ValueError), (dict(mask=i(1, 2)), ValueError), (dict(cu=None), ValueError), (dict(cu=i(4)), ValueError), (dict(q=q.float()), TypeError),
                       (dict(prefix=i(1), prefix_len=17), ValueError), (dict(max_rows=300), ValueError), (dict(gate=f(0, 7)), ValueError)]:
        with pytest.raises(error):
            nunchi_amd.tree_attn(ctx, s, **{**attn, **bad})
    take = dict(cu=i(5), parent=i(2), words=i(2), picks=i(2), held=i(4), length=i(4), path=i(2), count=i(4), next=i(4), length_out=i(4), table=i(4, 3), page=16, free=i(9),
                taken=i(1), taken_out=i(1))
    for bad, error in [(dict(words=i(3)), ValueError), (dict(picks=f(2)), TypeError), (dict(free=None), ValueError), (dict(taken=i(2)), ValueError), (dict(table=i(3, 3)), ValueError),
                       (dict(next=i(5)), ValueError), (dict(taken_out=None), ValueError)]:
        with pytest.raises(error):
            nunchi_amd.tree_take(ctx, **{**take, **bad})
