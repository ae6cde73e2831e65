// The operators that serve a batch of conversations (include/seoul_hip.h: sh_page_plan, sh_page_put, sh_page_attn,
// sh_sample): argument blocks and launchers of their kernels.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace sh {

enum { TY_F32 = 0, TY_F16 = 1, TY_BF16 = 30 };

constexpr int PLAN_MAX_N = 4096;   // requests of a step: their running sums live in LDS
constexpr int SAMPLE_MAX_VOCAB = 1 << 19;   // 2^44 times as many fits 64 bits

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

hipError_t launch_page_plan(const plan_args& a, hipStream_t s);
hipError_t launch_page_put(int D, int src_type, int type, const put_args& a, hipStream_t s);
// the parts of a call's keys, from sizes alone (sp, so, pchunk, ochunk of `a`); single: one row for each request (no cu).
// False when a launch would be too large
bool page_attn_split(int D, bool single, pattn_args& a);
hipError_t launch_page_attn(int D, int type, const pattn_args& a, hipStream_t s);
hipError_t launch_sample(const sample_args& a, hipStream_t s);
// the words of ids[n] (a word < 0: fallback's) to token[n] and, for conversation m, out[m * ld]
hipError_t launch_take(int n, const int32_t* ids, const int32_t* fallback, int32_t* token, int32_t* out, int ld, hipStream_t s);

}  // namespace sh
