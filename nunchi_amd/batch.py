"""Operators that serve a batch of conversations, on device tensors: pages of keys and values with their block tables and
slot maps (page_plan), the write of a step's positions (page_put), attention over a shared prefix and each conversation's
own pages (page_attn), and the next words (sample). For steps that try drafted words: their masks and positions (tree_plan),
attention over trees of them (tree_attn), how likely words are (word_probs), the branch that is kept (tree_take) and its moves
(page_keep). include/seoul_hip.h says what each computes.

Tensors are torch's, or anything with its data_ptr, dtype, shape, is_contiguous and get_device; they are contiguous and on
the context's device. Calls are enqueued on the context's stream and do not wait, so a context made on the stream that the
tensors are used on (Context(device, stream=...)) keeps everything in order. The checks of tensors are in csrc/py_batch.cpp.
"""
from __future__ import annotations

import ctypes as C

import nunchi_amd as _n

_TYPES = {"f16": 1, "bf16": 30}
_ENTRIES = ("sh_page_plan", "sh_page_put", "sh_page_attn", "sh_sample", "sh_tree_plan", "sh_tree_attn", "sh_word_probs", "sh_tree_take_planned", "sh_page_keep")
_native = None      # (the module, addresses of _ENTRIES): made by the first call


def _load():
    global _native
    try:
        from . import _batch
    except ImportError as e:
        raise ImportError("nunchi_amd._batch is not built for this Python: run `python -m nunchi_amd.build` (it needs a C++ compiler and Python.h)") from e
    lib = _n.load_library()
    _native = (_batch, *(C.cast(getattr(lib, f), C.c_void_p).value for f in _ENTRIES))
    return _native


class PageShape(C.Structure):
    """sh_page_shape: the layout of one layer's pages and what attention over them needs to know. keys and values are
    [n_pages][n_kv][page][head_dim] tensors of dtype ("f16" or "bf16")."""
    _fields_ = [("n_head", C.c_int), ("n_kv", C.c_int), ("head_dim", C.c_int), ("page", C.c_int), ("type", C.c_int), ("window", C.c_int),
                ("n_pages", C.c_longlong), ("scale", C.c_float), ("eps", C.c_float)]

    def __init__(self, n_head: int, n_kv: int, head_dim: int, page: int, n_pages: int, dtype: str = "f16", window: int = 0,
                 scale: float = 0.0, eps: float = 1e-5):
        if dtype not in _TYPES:
            raise ValueError("pages hold f16 or bf16")
        super().__init__(int(n_head), int(n_kv), int(head_dim), int(page), _TYPES[dtype], int(window), int(n_pages), float(scale), float(eps))

    @property
    def address(self) -> int:
        """Where this object's fields are (a copy's are its own: the address is not kept)."""
        return C.addressof(self)

    @property
    def cache_shape(self) -> tuple:
        return (self.n_pages, self.n_kv, self.page, self.head_dim)


def page_plan(ctx, held, add, free, taken, table, page: int, length, cu, slots, pos, taken_out, pos0: int = 0):
    """Block tables and slot maps of a step (sh_page_plan): held, add [n] i32, free [n_free] i32, taken [1] i32 in;
    table [n][cols] i32 completed in place; length [n], cu [n + 1], pos [rows], taken_out [1] i32 and slots [rows] i64 out."""
    native = _native or _load()
    rc = native[0].page_plan(native[1], ctx.h.value, ctx.device, held, add, free, taken, table, page, length, cu, slots, pos, taken_out, pos0)
    if rc:
        _n._check(rc)


def page_put(ctx, shape: PageShape, qkv, slots, keys, values, q=None, pos=None, q_norm=None, k_norm=None, rope=None):
    """Norm, rotation and write of a step's positions (sh_page_put): qkv [rows][ld] in f32, f16 or bf16 (q heads, k heads,
    v heads, anything else), slots [rows] i64, rope [positions][head_dim / 2][2] and the norms [head_dim] in f32."""
    native = _native or _load()
    rc = native[0].page_put(native[2], ctx.h.value, ctx.device, shape.address, qkv, slots, keys, values, q, pos, q_norm, k_norm, rope)
    if rc:
        _n._check(rc)


def page_attn_work(shape: PageShape, n: int, rows: int, max_len: int, max_rows: int = 1, prefix_len: int = 0) -> int:
    """Bytes of work memory of a page_attn call of these sizes."""
    size = C.c_size_t()
    _n._check(_n.load_library().sh_page_attn_work(C.byref(shape), int(n), int(rows), int(max_rows), int(prefix_len), int(max_len), C.byref(size)))
    return size.value


def page_attn(ctx, shape: PageShape, q, keys, values, table, length, out, work, max_len: int, cu=None, max_rows: int = 1, prefix=None,
              prefix_len: int = 0, gate=None, lse=None):
    """Attention over the shared prefix and each request's own pages (sh_page_attn): q, out [rows][n_head][head_dim],
    table [n][cols] and length [n] i32, cu [n + 1] i32 (None: one row for each request), prefix [pages] i32,
    gate and lse [rows][n_head] f32, work u8 of page_attn_work's bytes."""
    native = _native or _load()
    rc = native[0].page_attn(native[3], ctx.h.value, ctx.device, shape.address, q, keys, values, table, length, out, work, max_len, cu, max_rows,
                             prefix, prefix_len, gate, lse)
    if rc:
        _n._check(rc)


def sample_work(rows: int, vocab: int) -> int:
    """Bytes of work memory of a sample call of these sizes."""
    size = C.c_size_t()
    _n._check(_n.load_library().sh_sample_work(int(rows), int(vocab), C.byref(size)))
    return size.value


def sample(ctx, scores, u, ids, work, temp=None, top_k=None, top_p=None, min_p=None, chance=None):
    """One word for each row of scores [rows][vocab] in f32, f16 or bf16 (sh_sample): u [rows] f64 in [0, 1); temp, top_p,
    min_p f32 and top_k i32, [rows] or None; ids [rows] i32 and chance [rows] f32 out; work u8 of sample_work's bytes."""
    native = _native or _load()
    rc = native[0].sample(native[4], ctx.h.value, ctx.device, scores, u, ids, work, temp, top_k, top_p, min_p, chance)
    if rc:
        _n._check(rc)


def tree_plan(ctx, cu, parent, held, length, mask, pos, max_rows: int, pos0: int = 0):
    """Masks and positions of drafted words (sh_tree_plan): cu [n + 1], parent [rows], held and length [n] i32 in;
    mask [rows][ceil(max_rows / 32)] i32 (its bits) and pos [rows] i32 out."""
    native = _native or _load()
    rc = native[0].tree_plan(native[5], ctx.h.value, ctx.device, cu, parent, held, length, mask, pos, max_rows, pos0)
    if rc:
        _n._check(rc)


def tree_attn_work(shape: PageShape, n: int, rows: int, max_len: int, max_rows: int, prefix_len: int = 0) -> int:
    """Bytes of work memory of a tree_attn call of these sizes."""
    size = C.c_size_t()
    _n._check(_n.load_library().sh_tree_attn_work(C.byref(shape), int(n), int(rows), int(max_rows), int(prefix_len), int(max_len), C.byref(size)))
    return size.value


def tree_attn(ctx, shape: PageShape, q, keys, values, table, length, cu, mask, out, work, max_len: int, max_rows: int, prefix=None,
              prefix_len: int = 0, gate=None, lse=None):
    """Attention of trees of drafted words over the shared prefix, each request's own pages and the words before them
    (sh_tree_attn): cu [n + 1] i32 and tree_plan's mask, the others as page_attn's, work u8 of tree_attn_work's bytes."""
    native = _native or _load()
    rc = native[0].tree_attn(native[6], ctx.h.value, ctx.device, shape.address, q, keys, values, table, length, cu, mask, out, work, max_len, max_rows,
                             prefix, prefix_len, gate, lse)
    if rc:
        _n._check(rc)


def word_probs_work(rows: int, vocab: int, n_top: int = 0) -> int:
    """Bytes of work memory of a word_probs call of these sizes."""
    size = C.c_size_t()
    _n._check(_n.load_library().sh_word_probs_work(int(rows), int(vocab), int(n_top), C.byref(size)))
    return size.value


def word_probs(ctx, scores, work, temp=None, words=None, logp=None, entropy=None, top_words=None, top_logp=None):
    """How likely words are (sh_word_probs): scores [rows][vocab] in f32, f16 or bf16, temp [rows] f32 or None (1), words
    [rows][m] i32 in; logp [rows][m], entropy [rows], top_logp [rows][k] f32 and top_words [rows][k] i32 (k up to 64) out,
    each or None; work u8 of word_probs_work's bytes."""
    native = _native or _load()
    rc = native[0].word_probs(native[7], ctx.h.value, ctx.device, scores, work, temp, words, logp, entropy, top_words, top_logp)
    if rc:
        _n._check(rc)


def tree_take(ctx, cu, parent, words, picks, held, length, path, count, next, length_out, table=None, page: int = 16, free=None, taken=None,
              taken_out=None, pos=None):
    """The branch of drafted words that the picks agree with (sh_tree_take): cu [n + 1], parent, words and picks [rows], held
    and length [n] i32 in; path [rows], count, next and length_out [n] i32 out. With table [n][cols] i32 the pages behind the
    new lengths go back to free [n_free] i32, taken [1] i32 in and taken_out [1] out. With pos [rows] i32, tree_plan's, requests
    that it refused keep nothing and the length they had (sh_tree_take_planned); without it a request of more rows than the
    plan's max_rows counts as planned."""
    native = _native or _load()
    rc = native[0].tree_take(native[8], ctx.h.value, ctx.device, cu, parent, words, picks, held, length, path, count, next, length_out, table, page, free,
                             taken, taken_out, pos)
    if rc:
        _n._check(rc)


def page_keep(ctx, shape: PageShape, cu, path, length, table, keys, values):
    """Keys and values of the kept branch moved to where the next step expects them, in one layer (sh_page_keep): cu [n + 1],
    tree_take's path [rows], length [n] (with the step's rows) and table [n][cols] i32."""
    native = _native or _load()
    rc = native[0].page_keep(native[9], ctx.h.value, ctx.device, shape.address, cu, path, length, table, keys, values)
    if rc:
        _n._check(rc)
