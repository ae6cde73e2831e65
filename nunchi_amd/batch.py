"""Operators that serve a batch of conversations, on device tensors: pages of keys and values with their block tables and
slot maps (page_plan), the write of a step's positions (page_put), attention over a shared prefix and each conversation's
own pages (page_attn), and the next words (sample). include/seoul_hip.h says what each computes.

Tensors are torch's, or anything with its data_ptr, dtype, shape, is_contiguous and device; they are contiguous and on the
context's device. Calls are enqueued on the context's stream and do not wait, so a context made on the stream that the
tensors are used on (Context(device, stream=...)) keeps everything in order.
"""
from __future__ import annotations

import ctypes as C

import nunchi_amd as _n

F32, F16, BF16 = 0, 1, 30
_TYPES = {"f32": F32, "f16": F16, "bf16": BF16}
_NAMES = {"torch.float32": F32, "torch.float16": F16, "torch.bfloat16": BF16, "torch.float64": "f64", "torch.int32": "i32",
          "torch.int64": "i64", "torch.uint8": "u8"}
_kinds: dict = {}   # a dtype's kind, by the dtype


def _kind(dtype):
    k = _kinds.get(dtype)
    if k is None:
        k = _kinds[dtype] = _NAMES.get(str(dtype), str(dtype))
    return k


def _at(ctx, name, x, kinds, shape=None):
    """The address of a device tensor after its checks; None stays None."""
    if x is None:
        return None
    if _kind(x.dtype) not in kinds:
        raise TypeError(f"{name} has type {x.dtype}")
    if shape is not None and tuple(x.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(x.shape)}, not {shape}")
    if not x.is_contiguous():
        raise ValueError(f"{name} is not contiguous")
    d = x.device
    if d.type != "cuda" or (d.index or 0) != ctx.device:
        raise ValueError(f"{name} is on {d}, the context on device {ctx.device}")
    return x.data_ptr()


class PageShape(C.Structure):
    """sh_page_shape: the layout of one layer's pages and what attention over them needs to know. keys and values are
    [n_pages][n_kv][page][head_dim] tensors of dtype ("f16" or "bf16")."""
    _fields_ = [("n_head", C.c_int), ("n_kv", C.c_int), ("head_dim", C.c_int), ("page", C.c_int), ("type", C.c_int), ("window", C.c_int),
                ("n_pages", C.c_longlong), ("scale", C.c_float), ("eps", C.c_float)]

    def __init__(self, n_head: int, n_kv: int, head_dim: int, page: int, n_pages: int, dtype: str = "f16", window: int = 0,
                 scale: float = 0.0, eps: float = 1e-5):
        if dtype not in ("f16", "bf16"):
            raise ValueError("pages hold f16 or bf16")
        super().__init__(int(n_head), int(n_kv), int(head_dim), int(page), _TYPES[dtype], int(window), int(n_pages), float(scale), float(eps))

    @property
    def cache_shape(self) -> tuple:
        return (self.n_pages, self.n_kv, self.page, self.head_dim)


_I32, _I64, _F32, _F64, _U8 = ("i32",), ("i64",), (F32,), ("f64",), ("u8",)


def page_plan(ctx, held, add, free, taken, table, page: int, length, cu, slots, pos, taken_out, pos0: int = 0):
    """Block tables and slot maps of a step (sh_page_plan): held, add [n] i32, free [n_free] i32, taken [1] i32 in;
    table [n][cols] i32 completed in place; length [n], cu [n + 1], pos [rows], taken_out [1] i32 and slots [rows] i64 out."""
    n, rows = held.shape[0], slots.shape[0]
    cols = table.shape[1]
    _n._check(_n._lib.sh_page_plan(
        ctx.h, n, _at(ctx, "held", held, _I32, (n,)), _at(ctx, "add", add, _I32, (n,)), int(page), _at(ctx, "table", table, _I32, (n, cols)),
        cols, _at(ctx, "free", free, _I32, (free.shape[0],)), free.shape[0], _at(ctx, "taken", taken, _I32, (1,)),
        _at(ctx, "taken_out", taken_out, _I32, (1,)), _at(ctx, "length", length, _I32, (n,)), _at(ctx, "cu", cu, _I32, (n + 1,)),
        _at(ctx, "slots", slots, _I64, (rows,)), _at(ctx, "pos", pos, _I32, (rows,)), rows, int(pos0)))


def page_put(ctx, shape: PageShape, qkv, slots, keys, values, q=None, pos=None, q_norm=None, k_norm=None, rope=None):
    """Norm, rotation and write of a step's positions (sh_page_put): qkv [rows][ld] in f32, f16 or bf16 (q heads, k heads,
    v heads, anything else), slots [rows] i64, rope [positions][head_dim / 2][2] and the norms [head_dim] in f32."""
    rows, ld = qkv.shape
    D, kind = shape.head_dim, (shape.type,)
    n_rope = 0 if rope is None else rope.shape[0]
    _n._check(_n._lib.sh_page_put(
        ctx.h, C.byref(shape), rows, _at(ctx, "qkv", qkv, (F32, F16, BF16)), ld, _kind(qkv.dtype), _at(ctx, "q_norm", q_norm, _F32, (D,)),
        _at(ctx, "k_norm", k_norm, _F32, (D,)), _at(ctx, "rope", rope, _F32, (n_rope, D // 2, 2)), n_rope, _at(ctx, "pos", pos, _I32, (rows,)),
        _at(ctx, "slots", slots, _I64, (rows,)), _at(ctx, "q", q, kind, (rows, shape.n_head, D)),
        _at(ctx, "keys", keys, kind, shape.cache_shape), _at(ctx, "values", values, kind, shape.cache_shape)))


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
    rows, H, n, cols = q.shape[0], shape.n_head, length.shape[0], table.shape[1]
    kind, heads = (shape.type,), (rows, H, shape.head_dim)
    if prefix_len and (prefix is None or prefix.shape[0] * shape.page < prefix_len):
        raise ValueError("prefix has fewer pages than prefix_len needs")
    _n._check(_n._lib.sh_page_attn(
        ctx.h, C.byref(shape), n, rows, _at(ctx, "cu", cu, _I32, (n + 1,)), int(max_rows), _at(ctx, "q", q, kind, heads),
        _at(ctx, "keys", keys, kind, shape.cache_shape), _at(ctx, "values", values, kind, shape.cache_shape),
        _at(ctx, "prefix", prefix, _I32) if prefix_len else None, int(prefix_len), _at(ctx, "table", table, _I32, (n, cols)), cols,
        _at(ctx, "length", length, _I32, (n,)), int(max_len), _at(ctx, "gate", gate, _F32, (rows, H)), _at(ctx, "out", out, kind, heads),
        _at(ctx, "lse", lse, _F32, (rows, H)), _at(ctx, "work", work, _U8), work.numel()))


def sample_work(rows: int, vocab: int) -> int:
    """Bytes of work memory of a sample call of these sizes."""
    size = C.c_size_t()
    _n._check(_n.load_library().sh_sample_work(int(rows), int(vocab), C.byref(size)))
    return size.value


def sample(ctx, scores, u, ids, work, temp=None, top_k=None, top_p=None, min_p=None, chance=None):
    """One word for each row of scores [rows][vocab] in f32, f16 or bf16 (sh_sample): u [rows] f64 in [0, 1); temp, top_p,
    min_p f32 and top_k i32, [rows] or None; ids [rows] i32 and chance [rows] f32 out; work u8 of sample_work's bytes."""
    rows, vocab = scores.shape
    one = (rows,)
    _n._check(_n._lib.sh_sample(
        ctx.h, rows, vocab, _at(ctx, "scores", scores, (F32, F16, BF16)), vocab, _kind(scores.dtype), _at(ctx, "temp", temp, _F32, one),
        _at(ctx, "top_k", top_k, _I32, one), _at(ctx, "top_p", top_p, _F32, one), _at(ctx, "min_p", min_p, _F32, one),
        _at(ctx, "u", u, _F64, one), _at(ctx, "ids", ids, _I32, one), _at(ctx, "chance", chance, _F32, one), _at(ctx, "work", work, _U8),
        work.numel()))
