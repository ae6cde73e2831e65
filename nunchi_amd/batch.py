"""Operators that serve a batch of conversations, on device tensors: pages of keys and values with their block tables and
slot maps (page_plan), the write of a step's positions (page_put), attention over a shared prefix and each conversation's
own pages (page_attn), and the next words (sample). include/seoul_hip.h says what each computes.

Tensors are torch's, or anything with its data_ptr, dtype, shape, is_contiguous and get_device; they are contiguous and on
the context's device. Calls are enqueued on the context's stream and do not wait, so a context made on the stream that the
tensors are used on (Context(device, stream=...)) keeps everything in order. The checks of tensors are in csrc/py_batch.cpp.
"""
from __future__ import annotations

import ctypes as C

import nunchi_amd as _n

_TYPES = {"f16": 1, "bf16": 30}
_native = None      # (the module, addresses of the four entry points): made by the first call


def _load():
    global _native
    try:
        from . import _batch
    except ImportError as e:
        raise ImportError("nunchi_amd._batch is not built for this Python: run `python -m nunchi_amd.build` (it needs a C++ compiler and Python.h)") from e
    lib = _n.load_library()
    _native = (_batch, *(C.cast(getattr(lib, f), C.c_void_p).value for f in ("sh_page_plan", "sh_page_put", "sh_page_attn", "sh_sample")))
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
