"""Refusals of the batch operators (sh_page_plan, sh_page_put, sh_page_attn, sh_sample) that need no GPU: every check below
comes before the context or any buffer is touched, so the context and the buffers here are addresses only."""
import copy
import ctypes as C
import gc
import pickle
from types import SimpleNamespace

import pytest

import nunchi_amd
from nunchi_amd.batch import PageShape

ARG = nunchi_amd.SH_E_ARG
FAKE = C.create_string_buffer(1 << 16)             # stands for a context
BASE = (C.addressof(FAKE) + 4095) & ~4095


def _lib():
    return nunchi_amd.load_library()


def at(k):
    """An address of its own for buffer k (never read)."""
    return BASE + (k + 1) * (1 << 32)


def shape(**kw):
    s = dict(n_head=8, n_kv=2, head_dim=64, page=16, n_pages=10)
    fix = {k: kw.pop(k) for k in ("type",) if k in kw}
    s.update(kw)
    out = PageShape(**s)
    for k, v in fix.items():
        setattr(out, k, v)
    return out


BAD_SHAPES = [dict(n_head=7), dict(n_kv=0), dict(n_head=0), dict(head_dim=48), dict(head_dim=256), dict(page=8), dict(page=48), dict(page=512),
              dict(n_pages=0), dict(n_pages=1 << 31), dict(window=-1), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
              dict(eps=-1.0), dict(eps=float("nan")), dict(type=0), dict(type=7), dict(n_head=1 << 17, n_kv=1)]


@pytest.mark.parametrize("bad", BAD_SHAPES, ids=str)
def test_shapes_refused(bad):
    L, size, s = _lib(), C.c_size_t(7), shape(**bad)
    assert L.sh_page_attn_work(C.byref(s), 1, 1, 1, 0, 10, C.byref(size)) == ARG
    assert L.sh_page_put(BASE, C.byref(s), 1, at(0), 4096, 0, None, None, None, 0, None, at(1), None, at(2), at(3)) == ARG
    assert L.sh_page_attn(BASE, C.byref(s), 1, 1, None, 1, at(0), at(1), at(2), None, 0, at(3), 4, at(4), 10, None, at(5), None, at(6), 1 << 20) == ARG
    assert b"sh_page_attn" in L.sh_last_error()


def test_null_shape_refused():
    size = C.c_size_t()
    assert _lib().sh_page_attn_work(None, 1, 1, 1, 0, 10, C.byref(size)) == ARG
    s = shape()
    assert _lib().sh_page_attn_work(C.byref(s), 1, 1, 1, 0, 10, None) == ARG


def test_page_shape_takes_16_bit_types_only():
    with pytest.raises(ValueError):
        PageShape(8, 2, 64, 16, 10, dtype="f32")


PLAN = dict(ctx=BASE, n=4, held=at(0), add=at(1), page=16, table=at(2), cols=8, free=at(3), n_free=10, taken=at(4), taken_out=at(5), len=at(6),
            cu=at(7), slots=at(8), pos=at(9), rows=4, pos0=0)


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(n=0), dict(n=4097), dict(held=None), dict(add=None), dict(page=24), dict(page=0), dict(table=None),
                                 dict(cols=-1), dict(free=None), dict(n_free=-1), dict(taken=None), dict(taken_out=None), dict(len=None), dict(cu=None),
                                 dict(slots=None), dict(pos=None), dict(rows=-1), dict(pos0=-1),
                                 # an output over an input, or over another output
                                 dict(len=at(0)), dict(len=at(0) + 12), dict(cu=at(1)), dict(taken_out=at(4)), dict(table=at(3) + 36), dict(pos=at(8) + 28),
                                 dict(len=at(7) + 16), dict(slots=at(2) + 124)], ids=str)
def test_plan_refused(bad):
    v = {**PLAN, **bad}
    assert _lib().sh_page_plan(*v.values()) == ARG
    assert b"sh_page_plan" in _lib().sh_last_error()


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(rows=-1), dict(qkv=None), dict(qkv=at(0) + 2), dict(ld=767), dict(src=2), dict(src=8), dict(rope=at(4)),
                                 dict(rope=at(4), pos=at(5), n_rope=0), dict(slots=None), dict(q=at(6) + 8), dict(keys=None), dict(keys=at(1) + 2),
                                 dict(values=None), dict(values=at(2) + 4), dict(rows=(1 << 31) - 1, ld=1 << 40),
                                 # an output over an input, or over another output
                                 dict(q=at(0)), dict(q=at(0) + (2 * 768 + 767) * 4 // 16 * 16), dict(keys=at(0) + 16), dict(values=at(3)), dict(keys=at(2) + 16),
                                 dict(q=at(1) + 10 * 2 * 16 * 64 * 2 - 16), dict(q=at(2))], ids=str)
def test_put_refused(bad):
    s = shape(n_head=8, n_kv=2) if "ld" not in bad or bad["ld"] < 1 << 20 else shape(n_head=65536, n_kv=1)
    v = {**dict(ctx=BASE, shape=C.byref(s), rows=3, qkv=at(0), ld=768, src=0, q_norm=None, k_norm=None, rope=None, n_rope=5, pos=None, slots=at(3),
                q=None, keys=at(1), values=at(2)), **bad}
    assert _lib().sh_page_put(*v.values()) == ARG


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(n=0), dict(rows=-1), dict(rows=3), dict(max_rows=2), dict(max_rows=0, cu=at(9)), dict(q=None), dict(q=at(0) + 8),
                                 dict(keys=None), dict(keys=at(1) + 2), dict(values=None), dict(values=at(2) + 8), dict(prefix=None), dict(prefix_len=-1),
                                 dict(prefix_len=(1 << 31) - 1), dict(table=None), dict(cols=-1), dict(len=None), dict(max_len=-1), dict(out=None),
                                 dict(out=at(6) + 2), dict(work=None), dict(work=at(7) + 64), dict(bytes=100),
                                 # an output over an input, or over another output
                                 dict(out=at(0)), dict(out=at(1) + 64), dict(out=at(2)), dict(work=at(5)), dict(lse=at(6)), dict(lse=at(0) + 32), dict(lse=at(7) + 256),
                                 dict(gate=at(6) + 16), dict(out=at(3)), dict(out=at(4) + 112), dict(cu=at(7))], ids=str)
def test_attn_refused(bad):
    s = shape()
    size = C.c_size_t()
    assert _lib().sh_page_attn_work(C.byref(s), 4, 4, 1, 4096, 90, C.byref(size)) == 0 and size.value > 256
    v = {**dict(ctx=BASE, shape=C.byref(s), n=4, rows=4, cu=None, max_rows=1, q=at(0), keys=at(1), values=at(2), prefix=at(3), prefix_len=4096, table=at(4),
                cols=8, len=at(5), max_len=90, gate=None, out=at(6), lse=None, work=at(7), bytes=size.value), **bad}
    assert _lib().sh_page_attn(*v.values()) == ARG


def test_attn_launches_that_are_too_large_are_refused():
    s, size = shape(n_head=65536, n_kv=65536, n_pages=1000), C.c_size_t()
    assert _lib().sh_page_attn_work(C.byref(s), 40000, 40000, 1, 0, 100, C.byref(size)) == ARG
    assert b"fewer rows" in _lib().sh_last_error()


@pytest.mark.parametrize("n,rows,max_rows,prefix,own", [(1, 1, 1, 0, 1), (3, 3, 1, 500, 70), (2, 600, 400, 0, 1000), (256, 256, 1, 8192, 2048)])
def test_attn_work_fits_every_split(n, rows, max_rows, prefix, own):
    """Work memory is a multiple of 256 bytes and grows by whole parts: [parts][rows][heads] of 64 sums, a maximum and a
    sum of weights."""
    s, size = shape(), C.c_size_t()
    assert _lib().sh_page_attn_work(C.byref(s), n, rows, max_rows, prefix, own, C.byref(size)) == 0
    part = rows * 8 * (64 + 2) * 4
    assert size.value % 256 == 0 and (size.value == 256 or (size.value // part >= 2 and size.value % part < 512))


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(rows=-1), dict(vocab=0), dict(vocab=524289), dict(scores=None), dict(ld=99), dict(type=3), dict(u=None),
                                 dict(ids=None), dict(scores=at(0) + 2), dict(work=None), dict(work=at(3) + 128), dict(bytes=16),
                                 dict(ids=at(0) + 64), dict(chance=at(0)), dict(chance=at(2) + 4), dict(ids=at(1) + 8)], ids=str)
def test_sample_refused(bad):
    size = C.c_size_t()
    assert _lib().sh_sample_work(2, 100, C.byref(size)) == 0
    v = {**dict(ctx=BASE, rows=2, vocab=100, scores=at(0), ld=100, type=0, temp=None, top_k=None, top_p=None, min_p=None, u=at(1), ids=at(2), chance=None,
                work=at(3), bytes=size.value), **bad}
    assert _lib().sh_sample(*v.values()) == ARG


def test_no_rows_is_no_work():
    L, s = _lib(), shape()
    assert L.sh_page_put(BASE, C.byref(s), 0, None, 0, 0, None, None, None, 0, None, None, None, None, None) == 0
    assert L.sh_page_attn(BASE, C.byref(s), 2, 0, at(1), 1, None, None, None, None, 0, None, 0, None, 0, None, None, None, None, 0) == 0
    assert L.sh_sample(BASE, 0, 100, None, 100, 0, None, None, None, None, None, None, None, None, 0) == 0


def test_create_on_refuses_like_create():
    h = C.c_void_p()
    assert _lib().sh_create_on(0, None, None) == ARG
    assert _lib().sh_create_on(-1, None, C.byref(h)) != 0
    with pytest.raises(nunchi_amd.SeoulError):
        nunchi_amd.Context(4096, stream=0)


@pytest.mark.parametrize("way", [copy.copy, copy.deepcopy, lambda s: pickle.loads(pickle.dumps(s))], ids=["copy", "deepcopy", "pickle"])
def test_a_copied_shape_is_the_one_a_call_reads(way):
    """What a call reads is the copy's own: its page count (11, the original's is 10) and window, also once the original is gone.
    The tensors are host memory and have no rows, so the call ends before it touches the context."""
    torch = pytest.importorskip("torch")
    first = shape()
    second = way(first)
    second.n_pages, second.window = 11, 256
    assert second.address == C.addressof(second) and first.address == C.addressof(first) != second.address
    assert PageShape.from_address(second.address).window == 256 and PageShape.from_address(first.address).window == 0
    del first
    gc.collect()
    ctx = SimpleNamespace(h=SimpleNamespace(value=BASE), device=-1)
    keys, values = (torch.zeros(second.cache_shape, dtype=torch.float16) for _ in range(2))
    nunchi_amd.page_put(ctx, second, torch.zeros(0, 768), torch.zeros(0, dtype=torch.int64), keys, values)
    with pytest.raises(ValueError, match="11"):
        nunchi_amd.page_put(ctx, second, torch.zeros(0, 768), torch.zeros(0, dtype=torch.int64), keys[1:], values[1:])
    out = torch.zeros(0, 8, 64, dtype=torch.float16)
    nunchi_amd.page_attn(ctx, second, out, keys, values, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), out.clone(),
                         torch.zeros(256, dtype=torch.uint8), 4, cu=torch.zeros(3, dtype=torch.int32))


def test_generate_sampled_wants_the_second_conversations_random_numbers():
    """Refused before anything is called, also for one step (where a missing array would pass for one number, NaN)."""
    brain = nunchi_amd.Brain.__new__(nunchi_amd.Brain)      # (a model needs a GPU)
    brain.state, other = SimpleNamespace(), SimpleNamespace()
    for u in ([0.5], [0.5, 0.25], []):
        with pytest.raises(ValueError, match="u_b"):
            brain.generate_sampled(3, u, b=other, first_b=4)


def test_launches_of_2_to_the_32_threads_are_refused():
    """A launch holds less than 2^32 threads: 2^24 - 1 workgroups of 256 for attention and writes, 2^22 - 1 rows of 1024 for
    sampling. What passes that is an argument error of the size functions and the calls, before anything runs."""
    L, size = _lib(), C.c_size_t()
    s = shape(n_head=65536, n_kv=65536, n_pages=1000)      # (a workgroup for each row and head)
    assert L.sh_page_attn_work(C.byref(s), 255, 255, 1, 0, 100, C.byref(size)) == 0
    assert L.sh_page_attn_work(C.byref(s), 256, 256, 1, 0, 100, C.byref(size)) == ARG
    assert b"fewer rows" in L.sh_last_error()
    s = shape(n_head=16, n_kv=16)
    assert L.sh_page_attn_work(C.byref(s), 1 << 22, 1 << 22, 1, 4096, 100, C.byref(size)) == ARG
    assert b"fewer rows" in L.sh_last_error()
    s = shape(n_head=14, n_kv=1)                           # (a workgroup for each row of 16 heads)
    assert L.sh_page_put(BASE, C.byref(s), 1 << 24, at(0), 1024, 0, None, None, None, 0, None, at(1), None, at(2), at(3)) == ARG
    assert b"more rows" in L.sh_last_error()
    assert L.sh_sample_work((1 << 22) - 1, 10, C.byref(size)) == 0
    assert L.sh_sample_work(1 << 22, 10, C.byref(size)) == ARG
    assert L.sh_sample(BASE, 1 << 22, 10, at(0), 10, 0, None, None, None, None, at(1), at(2), None, at(3), 256) == ARG
    assert b"rows" in L.sh_last_error()
