// The operators that serve a batch of conversations (include/seoul_hip.h: sh_page_plan, sh_page_put, sh_page_attn, sh_sample;
// for drafted words sh_tree_plan, sh_tree_attn, sh_word_probs, sh_tree_take, sh_page_keep): argument blocks and launchers of
// their kernels.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace sh {

enum { TY_F32 = 0, TY_F16 = 1, TY_BF16 = 30 };

constexpr int PLAN_MAX_N = 4096;   // requests of a step: their running sums live in LDS
constexpr int SAMPLE_MAX_VOCAB = 1 << 19;   // 2^44 times as many fits 64 bits
constexpr int TREE_MAX = 256;      // drafted words of a request
constexpr int PROBS_MAX_TOP = 64;  // alternatives of a row of scores

// the workgroups of so many threads that one launch holds (less than 2^32 threads)
constexpr long long most_blocks(int threads) { return 0xFFFFFFFFll / threads; }

struct plan_args {
    int n, page_log, cols, n_free, rows, pos0;
    const int32_t *held, *add, *free_pages, *taken;
    int32_t *table, *taken_out, *len, *cu, *pos;
    int64_t* slots;
};

struct put_args {
    int rows, n_head, n_kv, n_rope, page_log;
    long long ld, n_slots;
    const void* qkv;
    const float *q_norm, *k_norm;
    const float2* rope;        // [n_rope][D / 2]
    const int32_t* pos;
    const int64_t* slots;
    void *q, *keys, *values;
    float eps;
};

struct pattn_args {
    int n, rows, n_head, n_kv, grp, page_log, window, max_rows, prefix_len, max_len, cols;
    int n_pages;
    float c;                   // scale * log2(e): scores in powers of two
    const int32_t *cu, *prefix, *table, *len;
    const void *q, *keys, *values;
    const float* gate;
    void* out;
    float* lse;
    // parts: the shared positions in sp parts of pchunk keys (none: fused, each request reads them before its own), each
    // request's own in so parts of ochunk; own ones are counted from own_at
    int sp, so, pchunk, ochunk, own_at, shared_blocks, own_blocks;
    bool fused;
    float* part_o;             // [sp + so][rows][n_head][D] sums of weights times values, not divided
    float2* part_ml;           // [sp + so][rows][n_head] maximum (powers of two) and sum of weights
    // trees of drafted words alone: which words of its request a row sees
    const unsigned* mask;      // [rows][words]
    int words, nts, nto;       // words of a mask; column groups of a workgroup of the shared positions and of the own ones
};

struct sample_args {
    int rows, vocab, type;
    long long ld;
    const void* scores;
    const float* temp;
    const int32_t* top_k;
    const float *top_p, *min_p;
    const double* u;
    int32_t* ids;
    float* chance;
};

struct tree_plan_args {
    int n, rows, max_rows, words, pos0;
    const int32_t *cu, *parent, *held, *len;
    unsigned* mask;            // [rows][words]
    int32_t* pos;
};

struct tree_take_args {
    int n, rows;
    const int32_t *cu, *parent, *pos, *word, *pick, *held, *len;   // (pos: null where it is not asked)
    int32_t *path, *count, *next, *len_out;
    // pages that are free again; none where table is null
    int page_log, cols, n_free;
    const int32_t *table, *taken;
    int32_t *free_pages, *taken_out;
};

struct keep_args {
    int n, rows, n_kv, page_log, cols, n_pages;
    const int32_t *cu, *path, *len, *table;
    void *keys, *values;
};

// one part of a row of scores: its largest, how many have that value, the others' weights relative to it, and their sum times
// the distance (in powers of two)
struct probs_part { float top, ties, rest, dist; };

struct probs_args {
    int rows, vocab, type, n_words, n_top, parts, chunk;
    long long ld;
    const void* scores;
    const float* temp;
    const int32_t* words;      // [rows][n_words]
    float *logp, *entropy, *top_logp;
    int32_t* top_words;
    probs_part* part;          // [rows][parts]
    unsigned long long* best;  // [rows][parts][max(n_top, 1)] keys of the likeliest words, 0 where there are none
};

hipError_t launch_page_plan(const plan_args& a, hipStream_t s);
hipError_t launch_page_put(int D, int src_type, int type, const put_args& a, hipStream_t s);
// the parts of a call's keys, from sizes alone (sp, so, pchunk, ochunk of `a`); single: one row for each request (no cu).
// False when a launch would be too large
bool page_attn_split(int D, bool single, pattn_args& a);
hipError_t launch_page_attn(int D, int type, const pattn_args& a, hipStream_t s);
// the same with trees of drafted words (a.mask)
bool tree_attn_split(int D, pattn_args& a);
hipError_t launch_tree_attn(int D, int type, const pattn_args& a, hipStream_t s);
// the parts of a call joined; nothing where there is one
hipError_t launch_page_join(int D, int type, const pattn_args& a, hipStream_t s);
hipError_t launch_tree_plan(const tree_plan_args& a, hipStream_t s);
hipError_t launch_tree_take(const tree_take_args& a, hipStream_t s);
hipError_t launch_page_keep(int D, const keep_args& a, hipStream_t s);
// parts and chunk of a call, from its sizes
void word_probs_split(probs_args& a);
hipError_t launch_word_probs(const probs_args& a, hipStream_t s);
hipError_t launch_sample(const sample_args& a, hipStream_t s);
// the words of ids[n] (a word < 0: fallback's) to token[n] and, for conversation m, out[m * ld]
hipError_t launch_take(int n, const int32_t* ids, const int32_t* fallback, int32_t* token, int32_t* out, int ld, hipStream_t s);

}  // namespace sh
