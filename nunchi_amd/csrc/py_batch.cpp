// CPython module nunchi_amd._batch: the device tensors of a batch operator's call checked (type, shape, contiguous, device)
// and handed to the C ABI. A decode step makes such calls every few microseconds and a tensor's checks from Python cost
// 0.6 us each, more together than the kernel behind them; here they cost 0.2 us. Tensors are torch's, or anything with
// its dtype, shape, is_contiguous(), get_device() and data_ptr(). Nothing here includes or links torch.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <cstring>

#include "../../include/seoul_hip.h"

namespace {

enum { K_F32 = 1, K_F16 = 2, K_BF16 = 4, K_F64 = 8, K_I32 = 16, K_I64 = 32, K_U8 = 64 };

PyObject *s_dtype, *s_shape, *s_is_contiguous, *s_get_device, *s_data_ptr;

// a dtype's kind, by the dtype (a program has a handful, each one object for its life; they are kept alive here)
struct { PyObject* dtype; int kind; } seen[32];
int n_seen = 0;

int kind_of(PyObject* dtype) {
    for (int i = 0; i < n_seen; i++)
        if (seen[i].dtype == dtype) return seen[i].kind;
    PyObject* text = PyObject_Str(dtype);
    if (!text) return -1;
    const char* t = PyUnicode_AsUTF8(text);
    if (!t) {
        Py_DECREF(text);
        return -1;
    }
    static const struct { const char* name; int kind; } known[] = {{"torch.float32", K_F32}, {"torch.float16", K_F16}, {"torch.bfloat16", K_BF16},
        {"torch.float64", K_F64}, {"torch.int32", K_I32}, {"torch.int64", K_I64}, {"torch.uint8", K_U8}};
    int kind = 0;
    for (auto& k : known)
        if (!strcmp(t, k.name)) kind = k.kind;
    Py_DECREF(text);
    if (n_seen < 32) {
        Py_INCREF(dtype);
        seen[n_seen++] = {dtype, kind};
    }
    return kind;
}

struct tensor {
    void* p = nullptr;         // null: None
    int kind = 0, nd = 0;
    long long d[4] = {0, 0, 0, 0};
    bool none() const { return nd == 0 && kind == 0; }
};

// x's address, kind and shape; false with an exception set. kinds: those it may have
bool read(PyObject* x, const char* name, long device, int kinds, tensor& t) {
    if (x == Py_None) return true;
    PyObject* v = PyObject_GetAttr(x, s_dtype);
    if (!v) return false;
    t.kind = kind_of(v);
    if (t.kind < 0) {
        Py_DECREF(v);
        return false;
    }
    if (!(t.kind & kinds)) {
        PyErr_Format(PyExc_TypeError, "%s has type %S", name, v);
        Py_DECREF(v);
        return false;
    }
    Py_DECREF(v);
    if (!(v = PyObject_GetAttr(x, s_shape))) return false;
    const Py_ssize_t nd = PyTuple_Check(v) ? PyTuple_GET_SIZE(v) : -1;
    if (nd < 1 || nd > 4) {
        PyErr_Format(PyExc_ValueError, "%s has shape %S", name, v);
        Py_DECREF(v);
        return false;
    }
    t.nd = (int)nd;
    for (Py_ssize_t i = 0; i < nd; i++) t.d[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(v, i));
    Py_DECREF(v);
    if (PyErr_Occurred()) return false;
    if (!(v = PyObject_CallMethodNoArgs(x, s_is_contiguous))) return false;
    const int contiguous = PyObject_IsTrue(v);
    Py_DECREF(v);
    if (contiguous != 1) {
        if (!PyErr_Occurred()) PyErr_Format(PyExc_ValueError, "%s is not contiguous", name);
        return false;
    }
    if (!(v = PyObject_CallMethodNoArgs(x, s_get_device))) return false;
    const long at = PyLong_AsLong(v);
    Py_DECREF(v);
    if (at != device) {
        if (!PyErr_Occurred()) PyErr_Format(PyExc_ValueError, "%s is on device %ld (-1: host memory), the context on device %ld", name, at, device);
        return false;
    }
    if (!(v = PyObject_CallMethodNoArgs(x, s_data_ptr))) return false;
    t.p = PyLong_AsVoidPtr(v);
    Py_DECREF(v);
    return !PyErr_Occurred();
}

// whether t (None too, where it may be) has the shape
bool has(const tensor& t, const char* name, int nd, long long a, long long b = 0, long long c = 0, long long d = 0, bool maybe = false) {
    if (t.none() && maybe) return true;
    const long long want[4] = {a, b, c, d};
    bool ok = t.nd == nd;
    for (int i = 0; ok && i < nd; i++) ok = t.d[i] == want[i];
    if (ok) return true;
    if (t.none()) PyErr_Format(PyExc_ValueError, "%s is None", name);
    else if (nd == 1) PyErr_Format(PyExc_ValueError, "%s does not have the shape (%lld,)", name, a);
    else if (nd == 2) PyErr_Format(PyExc_ValueError, "%s does not have the shape (%lld, %lld)", name, a, b);
    else if (nd == 3) PyErr_Format(PyExc_ValueError, "%s does not have the shape (%lld, %lld, %lld)", name, a, b, c);
    else PyErr_Format(PyExc_ValueError, "%s does not have the shape (%lld, %lld, %lld, %lld)", name, a, b, c, d);
    return false;
}
bool dims(const tensor& t, const char* name, int nd) {
    if (t.nd == nd) return true;
    PyErr_Format(PyExc_ValueError, "%s does not have %d dimensions", name, nd);
    return false;
}

int type_of(int kind) { return kind == K_F32 ? SH_F32 : kind == K_F16 ? SH_F16 : SH_BF16; }
int kind_for(int type) { return type == SH_F16 ? K_F16 : type == SH_BF16 ? K_BF16 : 0; }

bool number(PyObject* x, long long lo, long long hi, const char* name, long long& out) {
    out = PyLong_AsLongLong(x);
    if (out == -1 && PyErr_Occurred()) return false;
    if (out >= lo && out <= hi) return true;
    PyErr_Format(PyExc_ValueError, "%s is out of range", name);
    return false;
}
constexpr long long I32_MIN = INT32_MIN, I32_MAX = INT32_MAX;

// the entry point's address, the context's and its device: the first three arguments of every call
template <class F> bool head(PyObject* const* a, Py_ssize_t n, Py_ssize_t want, F& fn, sh_ctx*& ctx, long& device) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", n, want);
        return false;
    }
    fn = reinterpret_cast<F>(PyLong_AsVoidPtr(a[0]));
    ctx = a[1] == Py_None ? nullptr : static_cast<sh_ctx*>(PyLong_AsVoidPtr(a[1]));
    device = PyLong_AsLong(a[2]);
    return !PyErr_Occurred();
}
bool fits(const tensor& t, const char* name) {
    for (int i = 0; i < t.nd; i++)
        if (t.d[i] > I32_MAX) {
            PyErr_Format(PyExc_ValueError, "%s has more than 2^31 - 1 entries in a dimension", name);
            return false;
        }
    return true;
}

PyObject* page_plan(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    decltype(&sh_page_plan) fn;
    sh_ctx* ctx;
    long dev;
    if (!head(a, n_args, 15, fn, ctx, dev)) return nullptr;
    tensor held, add, free_pages, taken, table, length, cu, slots, pos, taken_out;
    long long page, pos0;
    if (!read(a[3], "held", dev, K_I32, held) || !read(a[4], "add", dev, K_I32, add) || !read(a[5], "free", dev, K_I32, free_pages) ||
        !read(a[6], "taken", dev, K_I32, taken) || !read(a[7], "table", dev, K_I32, table) || !number(a[8], I32_MIN, I32_MAX, "page", page) ||
        !read(a[9], "length", dev, K_I32, length) || !read(a[10], "cu", dev, K_I32, cu) || !read(a[11], "slots", dev, K_I64, slots) ||
        !read(a[12], "pos", dev, K_I32, pos) || !read(a[13], "taken_out", dev, K_I32, taken_out) || !number(a[14], I32_MIN, I32_MAX, "pos0", pos0))
        return nullptr;
    const long long n = held.d[0], rows = slots.d[0];
    if (!dims(held, "held", 1) || !dims(slots, "slots", 1) || !dims(table, "table", 2) || !dims(free_pages, "free", 1) || !fits(held, "held") ||
        !fits(slots, "slots") || !fits(table, "table") || !fits(free_pages, "free"))
        return nullptr;
    if (!has(add, "add", 1, n) || !has(taken, "taken", 1, 1) || !has(table, "table", 2, n, table.d[1]) || !has(length, "length", 1, n) ||
        !has(cu, "cu", 1, n + 1) || !has(pos, "pos", 1, rows) || !has(taken_out, "taken_out", 1, 1))
        return nullptr;
    return PyLong_FromLong(fn(ctx, (int)n, (const int32_t*)held.p, (const int32_t*)add.p, (int)page, (int32_t*)table.p, (int)table.d[1],
                              (const int32_t*)free_pages.p, (int)free_pages.d[0], (const int32_t*)taken.p, (int32_t*)taken_out.p,
                              (int32_t*)length.p, (int32_t*)cu.p, (int64_t*)slots.p, (int32_t*)pos.p, (int)rows, (int)pos0));
}

const sh_page_shape* shape_of(PyObject* x) { return static_cast<const sh_page_shape*>(PyLong_AsVoidPtr(x)); }

PyObject* page_put(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    decltype(&sh_page_put) fn;
    sh_ctx* ctx;
    long dev;
    if (!head(a, n_args, 13, fn, ctx, dev)) return nullptr;
    const sh_page_shape* s = shape_of(a[3]);
    if (!s) return nullptr;
    const int kind = kind_for(s->type);
    tensor qkv, slots, keys, values, q, pos, q_norm, k_norm, rope;
    if (!read(a[4], "qkv", dev, K_F32 | K_F16 | K_BF16, qkv) || !read(a[5], "slots", dev, K_I64, slots) || !read(a[6], "keys", dev, kind, keys) ||
        !read(a[7], "values", dev, kind, values) || !read(a[8], "q", dev, kind, q) || !read(a[9], "pos", dev, K_I32, pos) ||
        !read(a[10], "q_norm", dev, K_F32, q_norm) || !read(a[11], "k_norm", dev, K_F32, k_norm) || !read(a[12], "rope", dev, K_F32, rope))
        return nullptr;
    if (!dims(qkv, "qkv", 2) || !fits(qkv, "qkv") || (!rope.none() && (!dims(rope, "rope", 3) || !fits(rope, "rope")))) return nullptr;
    const long long rows = qkv.d[0], D = s->head_dim;
    if (!has(slots, "slots", 1, rows) || !has(keys, "keys", 4, s->n_pages, s->n_kv, s->page, D) || !has(values, "values", 4, s->n_pages, s->n_kv, s->page, D) ||
        !has(q, "q", 3, rows, s->n_head, D, 0, true) || !has(pos, "pos", 1, rows, 0, 0, 0, true) || !has(q_norm, "q_norm", 1, D, 0, 0, 0, true) ||
        !has(k_norm, "k_norm", 1, D, 0, 0, 0, true) || !has(rope, "rope", 3, rope.d[0], D / 2, 2, 0, true))
        return nullptr;
    return PyLong_FromLong(fn(ctx, s, (int)rows, qkv.p, qkv.d[1], type_of(qkv.kind), (const float*)q_norm.p, (const float*)k_norm.p,
                              (const float*)rope.p, (int)rope.d[0], (const int32_t*)pos.p, (const int64_t*)slots.p, q.p, keys.p, values.p));
}

PyObject* page_attn(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    decltype(&sh_page_attn) fn;
    sh_ctx* ctx;
    long dev;
    if (!head(a, n_args, 18, fn, ctx, dev)) return nullptr;
    const sh_page_shape* s = shape_of(a[3]);
    if (!s) return nullptr;
    const int kind = kind_for(s->type);
    tensor q, keys, values, table, length, out, work, cu, prefix, gate, lse;
    long long max_len, max_rows, prefix_len;
    if (!read(a[4], "q", dev, kind, q) || !read(a[5], "keys", dev, kind, keys) || !read(a[6], "values", dev, kind, values) ||
        !read(a[7], "table", dev, K_I32, table) || !read(a[8], "length", dev, K_I32, length) || !read(a[9], "out", dev, kind, out) ||
        !read(a[10], "work", dev, K_U8, work) || !number(a[11], I32_MIN, I32_MAX, "max_len", max_len) || !read(a[12], "cu", dev, K_I32, cu) ||
        !number(a[13], I32_MIN, I32_MAX, "max_rows", max_rows) || !number(a[15], I32_MIN, I32_MAX, "prefix_len", prefix_len) ||
        (prefix_len && !read(a[14], "prefix", dev, K_I32, prefix)) || !read(a[16], "gate", dev, K_F32, gate) || !read(a[17], "lse", dev, K_F32, lse))
        return nullptr;
    if (!dims(q, "q", 3) || !dims(length, "length", 1) || !dims(table, "table", 2) || !dims(work, "work", 1) || !fits(q, "q") || !fits(length, "length") ||
        !fits(table, "table"))
        return nullptr;
    const long long rows = q.d[0], n = length.d[0], H = s->n_head, D = s->head_dim;
    if (!has(q, "q", 3, rows, H, D) || !has(keys, "keys", 4, s->n_pages, s->n_kv, s->page, D) || !has(values, "values", 4, s->n_pages, s->n_kv, s->page, D) ||
        !has(table, "table", 2, n, table.d[1]) || !has(out, "out", 3, rows, H, D) || !has(cu, "cu", 1, n + 1, 0, 0, 0, true) ||
        !has(gate, "gate", 2, rows, H, 0, 0, true) || !has(lse, "lse", 2, rows, H, 0, 0, true))
        return nullptr;
    if (prefix_len > 0 && (!dims(prefix, "prefix", 1) || prefix.d[0] * s->page < prefix_len)) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "prefix has fewer pages than prefix_len needs");
        return nullptr;
    }
    return PyLong_FromLong(fn(ctx, s, (int)n, (int)rows, (const int32_t*)cu.p, (int)max_rows, q.p, keys.p, values.p, (const int32_t*)prefix.p, (int)prefix_len,
                              (const int32_t*)table.p, (int)table.d[1], (const int32_t*)length.p, (int)max_len, (const float*)gate.p, out.p, (float*)lse.p,
                              work.p, (size_t)work.d[0]));
}

PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    decltype(&sh_sample) fn;
    sh_ctx* ctx;
    long dev;
    if (!head(a, n_args, 12, fn, ctx, dev)) return nullptr;
    tensor scores, u, ids, work, temp, top_k, top_p, min_p, chance;
    if (!read(a[3], "scores", dev, K_F32 | K_F16 | K_BF16, scores) || !read(a[4], "u", dev, K_F64, u) || !read(a[5], "ids", dev, K_I32, ids) ||
        !read(a[6], "work", dev, K_U8, work) || !read(a[7], "temp", dev, K_F32, temp) || !read(a[8], "top_k", dev, K_I32, top_k) ||
        !read(a[9], "top_p", dev, K_F32, top_p) || !read(a[10], "min_p", dev, K_F32, min_p) || !read(a[11], "chance", dev, K_F32, chance))
        return nullptr;
    if (!dims(scores, "scores", 2) || !dims(work, "work", 1) || !fits(scores, "scores")) return nullptr;
    const long long rows = scores.d[0], vocab = scores.d[1];
    if (!has(u, "u", 1, rows) || !has(ids, "ids", 1, rows) || !has(temp, "temp", 1, rows, 0, 0, 0, true) || !has(top_k, "top_k", 1, rows, 0, 0, 0, true) ||
        !has(top_p, "top_p", 1, rows, 0, 0, 0, true) || !has(min_p, "min_p", 1, rows, 0, 0, 0, true) || !has(chance, "chance", 1, rows, 0, 0, 0, true))
        return nullptr;
    return PyLong_FromLong(fn(ctx, (int)rows, (int)vocab, scores.p, vocab, type_of(scores.kind), (const float*)temp.p, (const int32_t*)top_k.p,
                              (const float*)top_p.p, (const float*)min_p.p, (const double*)u.p, (int32_t*)ids.p, (float*)chance.p, work.p, (size_t)work.d[0]));
}

// rows of a step in packed order: cu [n + 1] and so many rows
bool packed(const tensor& cu, const tensor& rows, const char* name) {
    if (!dims(cu, "cu", 1) || !dims(rows, name, 1) || !fits(cu, "cu") || !fits(rows, name)) return false;
    if (cu.d[0] >= 2) return true;
    PyErr_SetString(PyExc_ValueError, "cu has fewer than 2 entries");
    return false;
}

PyObject* tree_plan(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    decltype(&sh_tree_plan) fn;
    sh_ctx* ctx;
    long dev;
    if (!head(a, n_args, 11, fn, ctx, dev)) return nullptr;
    tensor cu, parent, held, length, mask, pos;
    long long max_rows, pos0;
    if (!read(a[3], "cu", dev, K_I32, cu) || !read(a[4], "parent", dev, K_I32, parent) || !read(a[5], "held", dev, K_I32, held) ||
        !read(a[6], "length", dev, K_I32, length) || !read(a[7], "mask", dev, K_I32, mask) || !read(a[8], "pos", dev, K_I32, pos) ||
        !number(a[9], 1, 256, "max_rows", max_rows) || !number(a[10], I32_MIN, I32_MAX, "pos0", pos0))
        return nullptr;
    if (!packed(cu, parent, "parent")) return nullptr;
    const long long n = cu.d[0] - 1, rows = parent.d[0];
    if (!has(held, "held", 1, n) || !has(length, "length", 1, n) || !has(mask, "mask", 2, rows, (max_rows + 31) / 32) || !has(pos, "pos", 1, rows)) return nullptr;
    return PyLong_FromLong(fn(ctx, (int)n, (int)rows, (const int32_t*)cu.p, (const int32_t*)parent.p, (const int32_t*)held.p, (const int32_t*)length.p,
                              (int)max_rows, (uint32_t*)mask.p, (int32_t*)pos.p, (int)pos0));
}

PyObject* tree_attn(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    decltype(&sh_tree_attn) fn;
    sh_ctx* ctx;
    long dev;
    if (!head(a, n_args, 19, fn, ctx, dev)) return nullptr;
    const sh_page_shape* s = shape_of(a[3]);
    if (!s) return nullptr;
    const int kind = kind_for(s->type);
    tensor q, keys, values, table, length, cu, mask, out, work, prefix, gate, lse;
    long long max_len, max_rows, prefix_len;
    if (!read(a[4], "q", dev, kind, q) || !read(a[5], "keys", dev, kind, keys) || !read(a[6], "values", dev, kind, values) ||
        !read(a[7], "table", dev, K_I32, table) || !read(a[8], "length", dev, K_I32, length) || !read(a[9], "cu", dev, K_I32, cu) ||
        !read(a[10], "mask", dev, K_I32, mask) || !read(a[11], "out", dev, kind, out) || !read(a[12], "work", dev, K_U8, work) ||
        !number(a[13], I32_MIN, I32_MAX, "max_len", max_len) || !number(a[14], 1, 256, "max_rows", max_rows) ||
        !number(a[16], I32_MIN, I32_MAX, "prefix_len", prefix_len) || (prefix_len && !read(a[15], "prefix", dev, K_I32, prefix)) ||
        !read(a[17], "gate", dev, K_F32, gate) || !read(a[18], "lse", dev, K_F32, lse))
        return nullptr;
    if (!dims(q, "q", 3) || !dims(length, "length", 1) || !dims(table, "table", 2) || !dims(work, "work", 1) || !fits(q, "q") || !fits(length, "length") ||
        !fits(table, "table"))
        return nullptr;
    const long long rows = q.d[0], n = length.d[0], H = s->n_head, D = s->head_dim;
    if (!has(q, "q", 3, rows, H, D) || !has(keys, "keys", 4, s->n_pages, s->n_kv, s->page, D) || !has(values, "values", 4, s->n_pages, s->n_kv, s->page, D) ||
        !has(table, "table", 2, n, table.d[1]) || !has(out, "out", 3, rows, H, D) || !has(cu, "cu", 1, n + 1) ||
        !has(mask, "mask", 2, rows, (max_rows + 31) / 32) || !has(gate, "gate", 2, rows, H, 0, 0, true) || !has(lse, "lse", 2, rows, H, 0, 0, true))
        return nullptr;
    if (prefix_len > 0 && (!dims(prefix, "prefix", 1) || prefix.d[0] * s->page < prefix_len)) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "prefix has fewer pages than prefix_len needs");
        return nullptr;
    }
    return PyLong_FromLong(fn(ctx, s, (int)n, (int)rows, (const int32_t*)cu.p, (int)max_rows, (const uint32_t*)mask.p, q.p, keys.p, values.p,
                              (const int32_t*)prefix.p, (int)prefix_len, (const int32_t*)table.p, (int)table.d[1], (const int32_t*)length.p, (int)max_len,
                              (const float*)gate.p, out.p, (float*)lse.p, work.p, (size_t)work.d[0]));
}

PyObject* word_probs(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    decltype(&sh_word_probs) fn;
    sh_ctx* ctx;
    long dev;
    if (!head(a, n_args, 11, fn, ctx, dev)) return nullptr;
    tensor scores, work, temp, words, logp, entropy, top_words, top_logp;
    if (!read(a[3], "scores", dev, K_F32 | K_F16 | K_BF16, scores) || !read(a[4], "work", dev, K_U8, work) || !read(a[5], "temp", dev, K_F32, temp) ||
        !read(a[6], "words", dev, K_I32, words) || !read(a[7], "logp", dev, K_F32, logp) || !read(a[8], "entropy", dev, K_F32, entropy) ||
        !read(a[9], "top_words", dev, K_I32, top_words) || !read(a[10], "top_logp", dev, K_F32, top_logp))
        return nullptr;
    if (!dims(scores, "scores", 2) || !dims(work, "work", 1) || !fits(scores, "scores")) return nullptr;
    if ((!words.none() && (!dims(words, "words", 2) || !fits(words, "words"))) || (!top_words.none() && (!dims(top_words, "top_words", 2) || !fits(top_words, "top_words"))) ||
        (!top_logp.none() && (!dims(top_logp, "top_logp", 2) || !fits(top_logp, "top_logp"))))
        return nullptr;
    const long long rows = scores.d[0], vocab = scores.d[1], n_words = words.none() ? 0 : words.d[1];
    const long long n_top = !top_words.none() ? top_words.d[1] : !top_logp.none() ? top_logp.d[1] : 0;
    if (words.none() != logp.none()) {
        PyErr_SetString(PyExc_ValueError, "words and logp go together");
        return nullptr;
    }
    if (!has(temp, "temp", 1, rows, 0, 0, 0, true) || !has(words, "words", 2, rows, n_words, 0, 0, true) || !has(logp, "logp", 2, rows, n_words, 0, 0, true) ||
        !has(entropy, "entropy", 1, rows, 0, 0, 0, true) || !has(top_words, "top_words", 2, rows, n_top, 0, 0, true) ||
        !has(top_logp, "top_logp", 2, rows, n_top, 0, 0, true))
        return nullptr;
    return PyLong_FromLong(fn(ctx, (int)rows, (int)vocab, scores.p, vocab, type_of(scores.kind), (const float*)temp.p, (const int32_t*)words.p, (int)n_words,
                              (float*)logp.p, (float*)entropy.p, (int32_t*)top_words.p, (float*)top_logp.p, (int)n_top, work.p, (size_t)work.d[0]));
}

PyObject* tree_take(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    decltype(&sh_tree_take_planned) fn;
    sh_ctx* ctx;
    long dev;
    if (!head(a, n_args, 19, fn, ctx, dev)) return nullptr;
    tensor cu, parent, pos, words, picks, held, length, path, count, next, length_out, table, free_pages, taken, taken_out;
    long long page;
    if (!read(a[3], "cu", dev, K_I32, cu) || !read(a[4], "parent", dev, K_I32, parent) || !read(a[5], "words", dev, K_I32, words) ||
        !read(a[6], "picks", dev, K_I32, picks) || !read(a[7], "held", dev, K_I32, held) || !read(a[8], "length", dev, K_I32, length) ||
        !read(a[9], "path", dev, K_I32, path) || !read(a[10], "count", dev, K_I32, count) || !read(a[11], "next", dev, K_I32, next) ||
        !read(a[12], "length_out", dev, K_I32, length_out) || !read(a[13], "table", dev, K_I32, table) || !number(a[14], I32_MIN, I32_MAX, "page", page) ||
        !read(a[15], "free", dev, K_I32, free_pages) || !read(a[16], "taken", dev, K_I32, taken) || !read(a[17], "taken_out", dev, K_I32, taken_out) ||
        !read(a[18], "pos", dev, K_I32, pos))
        return nullptr;
    if (!packed(cu, parent, "parent")) return nullptr;
    const long long n = cu.d[0] - 1, rows = parent.d[0];
    if (!has(words, "words", 1, rows) || !has(picks, "picks", 1, rows) || !has(held, "held", 1, n) || !has(length, "length", 1, n) || !has(path, "path", 1, rows) ||
        !has(count, "count", 1, n) || !has(next, "next", 1, n) || !has(length_out, "length_out", 1, n) || !has(pos, "pos", 1, rows, 0, 0, 0, true))
        return nullptr;
    if (!table.none() && (!dims(table, "table", 2) || !fits(table, "table") || !has(table, "table", 2, n, table.d[1]) || !dims(free_pages, "free", 1) ||
                          !fits(free_pages, "free") || !has(taken, "taken", 1, 1) || !has(taken_out, "taken_out", 1, 1)))
        return nullptr;
    // (a table of no columns has no address, but it is a table: what was taken is written)
    if (!table.none() && !table.p) table.p = cu.p;
    return PyLong_FromLong(fn(ctx, (int)n, (int)rows, (const int32_t*)cu.p, (const int32_t*)parent.p, (const int32_t*)pos.p, (const int32_t*)words.p, (const int32_t*)picks.p,
                              (const int32_t*)held.p, (const int32_t*)length.p, (int32_t*)path.p, (int32_t*)count.p, (int32_t*)next.p, (int32_t*)length_out.p,
                              (int)page, (const int32_t*)table.p, (int)table.d[1], (int32_t*)free_pages.p, (int)free_pages.d[0], (const int32_t*)taken.p,
                              (int32_t*)taken_out.p));
}

PyObject* page_keep(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    decltype(&sh_page_keep) fn;
    sh_ctx* ctx;
    long dev;
    if (!head(a, n_args, 10, fn, ctx, dev)) return nullptr;
    const sh_page_shape* s = shape_of(a[3]);
    if (!s) return nullptr;
    const int kind = kind_for(s->type);
    tensor cu, path, length, table, keys, values;
    if (!read(a[4], "cu", dev, K_I32, cu) || !read(a[5], "path", dev, K_I32, path) || !read(a[6], "length", dev, K_I32, length) ||
        !read(a[7], "table", dev, K_I32, table) || !read(a[8], "keys", dev, kind, keys) || !read(a[9], "values", dev, kind, values))
        return nullptr;
    if (!packed(cu, path, "path") || !dims(table, "table", 2) || !fits(table, "table")) return nullptr;
    const long long n = cu.d[0] - 1, rows = path.d[0], D = s->head_dim;
    if (!has(length, "length", 1, n) || !has(table, "table", 2, n, table.d[1]) || !has(keys, "keys", 4, s->n_pages, s->n_kv, s->page, D) ||
        !has(values, "values", 4, s->n_pages, s->n_kv, s->page, D))
        return nullptr;
    return PyLong_FromLong(fn(ctx, s, (int)n, (int)rows, (const int32_t*)cu.p, (const int32_t*)path.p, (const int32_t*)length.p, (const int32_t*)table.p,
                              (int)table.d[1], keys.p, values.p));
}

PyMethodDef methods[] = {
    {"page_plan", (PyCFunction)(void (*)())page_plan, METH_FASTCALL, nullptr},
    {"page_put", (PyCFunction)(void (*)())page_put, METH_FASTCALL, nullptr},
    {"page_attn", (PyCFunction)(void (*)())page_attn, METH_FASTCALL, nullptr},
    {"sample", (PyCFunction)(void (*)())sample, METH_FASTCALL, nullptr},
    {"tree_plan", (PyCFunction)(void (*)())tree_plan, METH_FASTCALL, nullptr},
    {"tree_attn", (PyCFunction)(void (*)())tree_attn, METH_FASTCALL, nullptr},
    {"word_probs", (PyCFunction)(void (*)())word_probs, METH_FASTCALL, nullptr},
    {"tree_take", (PyCFunction)(void (*)())tree_take, METH_FASTCALL, nullptr},
    {"page_keep", (PyCFunction)(void (*)())page_keep, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_batch", "Calls of the batch operators on device tensors.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__batch() {
    s_dtype = PyUnicode_InternFromString("dtype");
    s_shape = PyUnicode_InternFromString("shape");
    s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
    s_get_device = PyUnicode_InternFromString("get_device");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    if (!s_dtype || !s_shape || !s_is_contiguous || !s_get_device || !s_data_ptr) return nullptr;
    return PyModule_Create(&module);
}
