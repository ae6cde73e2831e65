// Host side of the operators that serve a batch of conversations (include/seoul_hip.h): checks of their arguments and
// the launches. Lengths, tables and slots are device memory, so what they hold is bounded in the kernels.
#include "../../include/seoul_hip.h"

#include <hip/hip_runtime.h>

#include <cfloat>
#include <climits>
#include <cmath>
#include <string>

#include "sh_ctx.h"
#include "sh_serve.h"

using namespace sh;

namespace {
// the calling thread's device is the context's while a call runs, and its own again afterwards
struct on_device {
    int before = -1;
    hipError_t e;
    explicit on_device(int device) {
        e = hipGetDevice(&before);
        if (e == hipSuccess && before != device) e = hipSetDevice(device);
        else before = -1;
    }
    ~on_device() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

int done(hipError_t e, const char* who) {
    return e == hipSuccess ? SH_OK : set_error(SH_E_HIP, std::string(who) + ": " + hipGetErrorString(e));
}
int bad(const char* who, const char* what) { return set_error(SH_E_ARG, std::string(who) + ": " + what); }

bool is_16(int type) { return type == SH_F16 || type == SH_BF16; }
bool off(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }
bool meet(const void* p, size_t np, const void* q, size_t nq) {
    const auto a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return np && nq && a < b + nq && b < a + np;
}

struct extent { const void* p; size_t n; };
// null when no output overlaps an input or another output
template <size_t I, size_t O> const char* overlap(const extent (&in)[I], const extent (&out)[O]) {
    for (size_t i = 0; i < O; i++) {
        for (auto& x : in)
            if (out[i].p && x.p && meet(out[i].p, out[i].n, x.p, x.n)) return "an output overlaps an input";
        for (size_t j = 0; j < i; j++)
            if (out[i].p && out[j].p && meet(out[i].p, out[i].n, out[j].p, out[j].n)) return "two outputs overlap";
    }
    return nullptr;
}

int page_log(int page) {
    for (int l = 4; l <= 8; l++)
        if (page == 1 << l) return l;
    return -1;
}

// null when the shape is one the kernels take
const char* shape_fault(const sh_page_shape* s) {
    if (!s) return "shape is null";
    if (s->n_kv < 1 || s->n_head < 1 || s->n_head % s->n_kv) return "n_head must be a positive multiple of n_kv";
    if (s->n_head > 65536) return "n_head is at most 65536";
    if (s->head_dim != 32 && s->head_dim != 64 && s->head_dim != 128) return "head_dim must be 32, 64 or 128";
    if (page_log(s->page) < 0) return "page must be 16, 32, 64, 128 or 256";
    if (!is_16(s->type)) return "type must be SH_F16 or SH_BF16";
    if (s->window < 0) return "window is negative";
    if (s->n_pages < 1 || s->n_pages > INT_MAX) return "n_pages must be at least 1 and fit 32 bits";
    if (!(s->scale >= 0.0f) || !std::isfinite(s->scale)) return "scale must be finite and not negative";
    if (!(s->eps >= 0.0f) || !std::isfinite(s->eps)) return "eps must be finite and not negative";
    return nullptr;
}

// sizes of an attention call into its argument block (the parts of the keys among them); null when they are in range
const char* attn_sizes(const sh_page_shape* s, int n, int rows, int max_rows, int prefix_len, int max_len, bool single, pattn_args& a) {
    if (const char* f = shape_fault(s)) return f;
    if (n < 1 || rows < 0 || max_rows < 1 || prefix_len < 0 || max_len < 0) return "a size is negative, or n or max_rows is 0";
    if (single && (rows != n || max_rows != 1)) return "without cu every request has one row (rows == n, max_rows == 1)";
    if ((long long)prefix_len + max_len > INT_MAX - 1024) return "prefix_len + max_len does not fit 32 bits";
    a.n = n;
    a.rows = rows;
    a.n_head = s->n_head;
    a.n_kv = s->n_kv;
    a.grp = s->n_head / s->n_kv;
    a.page_log = page_log(s->page);
    a.window = s->window < prefix_len + max_len ? s->window : 0;   // (a longer one leaves nothing out)
    a.max_rows = max_rows < rows ? max_rows : rows > 0 ? rows : 1;
    a.prefix_len = prefix_len;
    a.max_len = max_len;
    a.n_pages = (int)s->n_pages;
    a.c = std::fmax((s->scale > 0.0f ? s->scale : 1.0f / std::sqrt((float)s->head_dim)) * 1.44269504f, FLT_MIN);   // (0 times a masked -inf is NaN)
    if (!page_attn_split(s->head_dim, single, a)) return "more workgroups than one launch holds: fewer rows at once";
    return nullptr;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// bytes of the parts' sums, and behind them of their maxima and sums of weights
void attn_work(const pattn_args& a, int D, size_t* sums, size_t* all) {
    const size_t parts = a.sp + a.so > 1 ? (size_t)(a.sp + a.so) * a.rows * a.n_head : 0;
    *sums = align256(parts * D * sizeof(float));
    *all = *sums + align256(parts * sizeof(float2));
}
}  // namespace

#define SH_ENTRY try {
#define SH_ENTRY_END                                                        \
    }                                                                       \
    catch (...) {                                                           \
        return SH_E_NOMEM; /* the message of an error could not be made */  \
    }

extern "C" {

int sh_page_plan(sh_ctx* c, int n, const int32_t* held, const int32_t* add, int page, int32_t* table, int cols,
                 const int32_t* free_pages, int n_free, const int32_t* taken, int32_t* taken_out, int32_t* len, int32_t* cu,
                 int64_t* slots, int32_t* pos, int rows, int pos0) {
    SH_ENTRY
    const char* who = "sh_page_plan";
    if (!c || !held || !add || !taken || !taken_out || !len || !cu) return bad(who, "null");
    if (n < 1 || n > PLAN_MAX_N) return bad(who, "n must be 1 to 4096");
    if (page_log(page) < 0) return bad(who, "page must be 16, 32, 64, 128 or 256");
    if (cols < 0 || n_free < 0 || rows < 0 || pos0 < 0) return bad(who, "a size is negative");
    if ((cols && !table) || (n_free && !free_pages) || (rows && (!slots || !pos))) return bad(who, "null");
    const size_t in4 = (size_t)n * 4;
    const extent in[] = {{held, in4}, {add, in4}, {free_pages, (size_t)n_free * 4}, {taken, 4}},
                 out[] = {{table, (size_t)n * cols * 4}, {taken_out, 4}, {len, in4}, {cu, in4 + 4}, {slots, (size_t)rows * 8}, {pos, (size_t)rows * 4}};
    if (const char* f = overlap(in, out)) return bad(who, f);
    const on_device dev(c->device);
    if (dev.e != hipSuccess) return done(dev.e, who);
    plan_args a{};
    a.n = n;
    a.page_log = page_log(page);
    a.cols = cols;
    a.n_free = n_free;
    a.rows = rows;
    a.pos0 = pos0;
    a.held = held;
    a.add = add;
    a.free_pages = free_pages;
    a.taken = taken;
    a.table = table;
    a.taken_out = taken_out;
    a.len = len;
    a.cu = cu;
    a.slots = slots;
    a.pos = pos;
    return done(launch_page_plan(a, c->stream), who);
    SH_ENTRY_END
}

int sh_page_put(sh_ctx* c, const sh_page_shape* s, int rows, const void* qkv, long long ld, int src_type, const float* q_norm,
                const float* k_norm, const float* rope, int n_rope, const int32_t* pos, const int64_t* slots, void* q_out,
                void* keys, void* values) {
    SH_ENTRY
    const char* who = "sh_page_put";
    if (const char* f = shape_fault(s)) return bad(who, f);
    if (!c || rows < 0) return bad(who, "null context or negative rows");
    if (rows == 0) return SH_OK;
    if (!qkv || !slots || !keys || !values || (rope && !pos)) return bad(who, "null");
    if (src_type != SH_F32 && !is_16(src_type)) return bad(who, "src_type must be SH_F32, SH_F16 or SH_BF16");
    const long long heads = (long long)s->n_head + 2ll * s->n_kv;
    if (ld < heads * s->head_dim) return bad(who, "a row (ld) is shorter than its heads");
    if (rope && n_rope < 1) return bad(who, "n_rope must be positive");
    if ((rows * heads + 15) / 16 > most_blocks(256)) return bad(who, "more rows than one launch holds");
    if (off(qkv, src_type == SH_F32 ? 4 : 2)) return bad(who, "qkv is not aligned to its type");
    if (off(q_out, 16) || off(keys, 16) || off(values, 16)) return bad(who, "queries, keys and values start on 16 bytes");
    const size_t cache = (size_t)s->n_pages * s->n_kv * s->page * s->head_dim * 2, vec = (size_t)s->head_dim * 4;
    const extent in[] = {{qkv, ((size_t)(rows - 1) * ld + heads * s->head_dim) * (src_type == SH_F32 ? 4 : 2)}, {slots, (size_t)rows * 8}, {pos, (size_t)rows * 4},
                         {q_norm, vec}, {k_norm, vec}, {rope, rope ? (size_t)n_rope * vec : 0}},
                 out[] = {{q_out, (size_t)rows * s->n_head * s->head_dim * 2}, {keys, cache}, {values, cache}};
    if (const char* f = overlap(in, out)) return bad(who, f);
    const on_device dev(c->device);
    if (dev.e != hipSuccess) return done(dev.e, who);
    put_args a{};
    a.rows = rows;
    a.n_head = s->n_head;
    a.n_kv = s->n_kv;
    a.n_rope = n_rope;
    a.page_log = page_log(s->page);
    a.ld = ld;
    a.n_slots = s->n_pages * s->page;
    a.qkv = qkv;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.rope = reinterpret_cast<const float2*>(rope);
    a.pos = pos;
    a.slots = slots;
    a.q = q_out;
    a.keys = keys;
    a.values = values;
    a.eps = s->eps;
    return done(launch_page_put(s->head_dim, src_type, s->type, a, c->stream), who);
    SH_ENTRY_END
}

int sh_page_attn_work(const sh_page_shape* s, int n, int rows, int max_rows, int prefix_len, int max_len, size_t* bytes) {
    SH_ENTRY
    if (!bytes) return bad("sh_page_attn_work", "null");
    *bytes = 0;
    // (with or without cu: what either needs, of those that one launch holds)
    const char* fault = nullptr;
    bool any = false;
    for (const bool single : {false, true}) {
        if (single && (rows != n || max_rows != 1)) continue;
        pattn_args a{};
        if (const char* f = attn_sizes(s, n, rows, max_rows, prefix_len, max_len, single, a)) {
            fault = f;
            continue;
        }
        any = true;
        size_t sums, all;
        attn_work(a, s->head_dim, &sums, &all);
        if (all > *bytes) *bytes = all;
    }
    if (!any) return bad("sh_page_attn_work", fault);
    if (*bytes < 256) *bytes = 256;
    return SH_OK;
    SH_ENTRY_END
}

int sh_page_attn(sh_ctx* c, const sh_page_shape* s, int n, int rows, const int32_t* cu, int max_rows, const void* q, const void* keys,
                 const void* values, const int32_t* prefix, int prefix_len, const int32_t* table, int cols, const int32_t* len,
                 int max_len, const float* gate, void* out, float* lse, void* work, size_t work_bytes) {
    SH_ENTRY
    const char* who = "sh_page_attn";
    pattn_args a{};
    if (const char* f = attn_sizes(s, n, rows, max_rows, prefix_len, max_len, cu == nullptr, a)) return bad(who, f);
    if (!c) return bad(who, "null context");
    if (rows == 0) return SH_OK;
    if (!q || !keys || !values || !len || !out || (prefix_len && !prefix) || cols < 0 || (cols && !table)) return bad(who, "null, or cols negative");
    if (off(q, 16) || off(keys, 16) || off(values, 16) || off(out, 16)) return bad(who, "queries, keys, values and outputs start on 16 bytes");
    size_t sums, all;
    attn_work(a, s->head_dim, &sums, &all);
    if (all && (!work || work_bytes < all || off(work, 256))) return bad(who, "work is missing, smaller than sh_page_attn_work says, or not on 256 bytes");
    const size_t q_bytes = (size_t)rows * s->n_head * s->head_dim * 2, rh = (size_t)rows * s->n_head * sizeof(float),
                 cache = (size_t)s->n_pages * s->n_kv * s->page * s->head_dim * 2;
    const extent in[] = {{q, q_bytes}, {keys, cache}, {values, cache}, {gate, rh}, {len, (size_t)n * 4}, {table, (size_t)n * cols * 4}, {cu, ((size_t)n + 1) * 4},
                         {prefix, ((size_t)prefix_len + s->page - 1) / s->page * 4}},
                 to[] = {{out, q_bytes}, {lse, rh}, {work, all}};
    if (const char* f = overlap(in, to)) return bad(who, f);
    const on_device dev(c->device);
    if (dev.e != hipSuccess) return done(dev.e, who);
    a.cols = cols;
    a.cu = cu;
    a.prefix = prefix;
    a.table = table;
    a.len = len;
    a.q = q;
    a.keys = keys;
    a.values = values;
    a.gate = gate;
    a.out = out;
    a.lse = lse;
    a.part_o = static_cast<float*>(work);
    a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(work) + sums);
    return done(launch_page_attn(s->head_dim, s->type, a, c->stream), who);
    SH_ENTRY_END
}

int sh_sample_work(int rows, int vocab, size_t* bytes) {
    SH_ENTRY
    if (!bytes) return bad("sh_sample_work", "null");
    *bytes = 0;
    if (rows < 0 || vocab < 1 || vocab > SAMPLE_MAX_VOCAB) return bad("sh_sample_work", "rows is negative, or vocab not 1 to 524288");
    if (rows > most_blocks(1024)) return bad("sh_sample_work", "more rows than one launch holds");
    *bytes = 256;
    return SH_OK;
    SH_ENTRY_END
}

int sh_sample(sh_ctx* c, int rows, int vocab, const void* scores, long long ld, int type, const float* temp, const int32_t* top_k,
              const float* top_p, const float* min_p, const double* u, int32_t* ids, float* chance, void* work, size_t work_bytes) {
    SH_ENTRY
    const char* who = "sh_sample";
    size_t need = 0;
    if (!c) return bad(who, "null context");
    if (const int rc = sh_sample_work(rows, vocab, &need)) return rc;
    if (rows == 0) return SH_OK;
    if (!scores || !u || !ids) return bad(who, "null");
    if (type != SH_F32 && !is_16(type)) return bad(who, "type must be SH_F32, SH_F16 or SH_BF16");
    if (ld < vocab) return bad(who, "a row (ld) is shorter than vocab");
    if (off(scores, type == SH_F32 ? 4 : 2)) return bad(who, "scores are not aligned to their type");
    if (!work || work_bytes < need || off(work, 256)) return bad(who, "work is missing, smaller than sh_sample_work says, or not on 256 bytes");
    const size_t each = (size_t)rows * 4;
    const extent in[] = {{scores, ((size_t)(rows - 1) * ld + vocab) * (type == SH_F32 ? 4 : 2)}, {temp, each}, {top_k, each}, {top_p, each}, {min_p, each}, {u, each * 2}},
                 out[] = {{ids, each}, {chance, each}};
    if (const char* f = overlap(in, out)) return bad(who, f);
    const on_device dev(c->device);
    if (dev.e != hipSuccess) return done(dev.e, who);
    sample_args a{};
    a.rows = rows;
    a.vocab = vocab;
    a.type = type;
    a.ld = ld;
    a.scores = scores;
    a.temp = temp;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.u = u;
    a.ids = ids;
    a.chance = chance;
    return done(launch_sample(a, c->stream), who);
    SH_ENTRY_END
}

}  // extern "C"
