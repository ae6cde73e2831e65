// Pages of keys and values: the block tables and slot maps of a step (k_page_plan) and the write of its positions
// (k_page_put).
#include <hip/hip_runtime.h>

#include <climits>

#include "sh_device.h"
#include "sh_serve.h"

namespace sh {
namespace {

// ---------------------------------------------------------------- block tables and slot maps
// One launch. The running sums (rows before a request, pages opened before it) are short, so every workgroup forms them
// itself in LDS from the lengths rather than wait for another launch; then the workgroups share out the step's rows and
// its new pages, and find the request of each by bisection in LDS. Sums are formed in 64 bits and kept saturated at
// INT_MAX, which fits nothing. A decode step's plan (64 requests, one workgroup) takes 4.7 us, an empty launch about 3;
// 500 prompts with half a million rows 8.3 us: 489 workgroups, of which each spends about 5 on the lengths and sums before
// its first row. What bounds it is that chain of loads and barriers, not the 12 bytes a row.
constexpr int PLAN_T = 256;

struct plan_req {
    int have, need;      // pages held, pages opened (0 for a request that is refused for its lengths)
    bool ok;
};

__device__ __forceinline__ plan_req plan_need(const plan_args& a, int held, int add) {
    const int page = 1 << a.page_log;
    plan_req r{0, 0, held >= 0 && add >= 0};
    if (!r.ok) return r;
    const long long want = ((long long)held + add + page - 1) >> a.page_log;
    r.have = (int)(((long long)held + page - 1) >> a.page_log);
    r.ok = want <= a.cols && (long long)held + add <= INT_MAX;
    if (r.ok) r.need = (int)want - r.have;
    return r;
}

__device__ __forceinline__ int sat(long long v) { return v > INT_MAX ? INT_MAX : (int)v; }

// the last i in [0, n) with s[i] <= v (s[0] = 0 <= v)
__device__ __forceinline__ int last_at_most(const int* s, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (s[m] <= v) lo = m;
        else hi = m;
    }
    return lo;
}

// R: neighbouring rows a thread
template <int R> __global__ __launch_bounds__(PLAN_T) void k_page_plan(plan_args a) {
    extern __shared__ int lds[];
    int* cu_s = lds;                       // [n + 1] rows before each request
    int* st_s = lds + a.n + 1;             // [n + 1] pages opened before each request
    __shared__ long long wsum[2][PLAN_T / 64];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const int per = (a.n + PLAN_T - 1) / PLAN_T, i0 = t * per, i1 = min(a.n, i0 + per);
    long long rows = 0, pages = 0;
    for (int i = i0; i < i1; i++) {
        const int add = a.add[i];
        rows += max(add, 0);
        pages += plan_need(a, a.held[i], add).need;
    }
    // this thread's sums before it: a scan within the wave, then over the waves
    long long r_in = rows, p_in = pages;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long r = __shfl_up(r_in, o), p = __shfl_up(p_in, o);
        if (lane >= o) { r_in += r; p_in += p; }
    }
    if (lane == 63) { wsum[0][wv] = r_in; wsum[1][wv] = p_in; }
    __syncthreads();
    long long r_at = r_in - rows, p_at = p_in - pages;
    for (int w = 0; w < wv; w++) { r_at += wsum[0][w]; p_at += wsum[1][w]; }
    for (int i = i0; i < i1; i++) {
        const int add = a.add[i];
        cu_s[i] = sat(r_at);
        st_s[i] = sat(p_at);
        r_at += max(add, 0);
        p_at += plan_need(a, a.held[i], add).need;
    }
    if (t == PLAN_T - 1) { cu_s[a.n] = sat(r_at); st_s[a.n] = sat(p_at); }
    __syncthreads();
    const int taken = max(a.taken[0], 0), total = min(cu_s[a.n], a.rows);
    const int opened = min(st_s[a.n], max(a.n_free - taken, 0));   // (what lies behind fits no request)
    auto fits = [&](const plan_req& q, int i) {
        return q.ok && cu_s[i + 1] <= a.rows && cu_s[i + 1] < INT_MAX && (q.need == 0 || (long long)taken + st_s[i + 1] <= a.n_free);
    };
    // ---- per request: lengths and row starts (workgroup 0) ----
    if (blockIdx.x == 0) {
        long long out = taken;
        for (int i = t; i < a.n; i += PLAN_T) {
            const int held = a.held[i], add = a.add[i];
            const plan_req q = plan_need(a, held, add);
            const bool f = fits(q, i);
            a.cu[i] = cu_s[i];
            a.len[i] = f ? held + add : held;
            if (f && q.need) out = max(out, (long long)taken + st_s[i + 1]);
        }
        if (t == 0) a.cu[a.n] = cu_s[a.n];
        // pages are given out in order, so the last request that got some says how many are gone
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) out = max(out, __shfl_xor(out, o));
        if (lane == 0) wsum[0][wv] = out;   // (its sums were read before the last barrier)
        __syncthreads();
        if (t == 0) {
            for (int w = 1; w < PLAN_T / 64; w++) out = max(out, wsum[0][w]);
            a.taken_out[0] = (int)out;
        }
    }
    // ---- new pages ----
    for (long long p = (long long)blockIdx.x * PLAN_T + t; p < opened; p += (long long)gridDim.x * PLAN_T) {
        const int i = last_at_most(st_s, a.n, (int)p);
        const plan_req q = plan_need(a, a.held[i], a.add[i]);
        if (fits(q, i)) a.table[(size_t)i * a.cols + q.have + (int)p - st_s[i]] = a.free_pages[taken + (int)p];
    }
    // ---- new rows ----
    typedef int64_t slots_r __attribute__((ext_vector_type(R), aligned(8)));
    typedef int32_t pos_r __attribute__((ext_vector_type(R), aligned(4)));
    for (long long r0 = ((long long)blockIdx.x * PLAN_T + t) * R; r0 < total; r0 += (long long)gridDim.x * PLAN_T * R) {
        const int m = (int)min((long long)R, total - r0);
        int i = last_at_most(cu_s, a.n, (int)r0), of = -1, page = -1, id = -1, held = 0;
        plan_req q{};
        bool f = false;
        slots_r slot;
        pos_r pos;
#pragma unroll
        for (int e = 0; e < R; e++) {
            const int r = (int)min(r0 + e, total - 1ll);
            while (i + 1 < a.n && cu_s[i + 1] <= r) i++;
            if (i != of) {
                of = i;
                page = -1;
                held = a.held[i];
                q = plan_need(a, held, a.add[i]);
                f = fits(q, i);
            }
            const long long at = (long long)held + (r - cu_s[i]);
            slot[e] = -1;
            if (f) {
                const int j = (int)(at >> a.page_log);
                if (j != page) {
                    page = j;
                    id = j < q.have ? a.table[(size_t)i * a.cols + j] : a.free_pages[taken + st_s[i] + j - q.have];
                }
                if (id >= 0) slot[e] = ((int64_t)id << a.page_log) + (at & ((1 << a.page_log) - 1));
            }
            pos[e] = sat(a.pos0 + at);
        }
        if (m == R) {
            *(slots_r*)(a.slots + r0) = slot;
            *(pos_r*)(a.pos + r0) = pos;
        } else {
#pragma unroll
            for (int e = 0; e < R - 1; e++)
                if (e < m) { a.slots[r0 + e] = slot[e]; a.pos[r0 + e] = pos[e]; }
        }
    }
}

// ---------------------------------------------------------------- the write of a step's positions
// Sixteen lanes hold one head of one row, D / 16 neighbouring dimensions each: the sum of squares is four rotations
// within the 16 lanes, and the other half of a rotated pair (dimension + D / 2) sits 8 lanes on. Every value is read and
// written once, in vectors of a lane's share where rows start on them (VEC), one by one where not. Memory traffic bounds
// it: 8191 prompt rows of 16 + 2 x 4 heads of 128 (fp32 in, bf16 out) in 33 us, 4.6 TB/s of a copy's 5.1; a decode step of 64 rows
// takes 3 us, a launch.
template <class T> __device__ __forceinline__ float to_f(T v) { return (float)v; }

template <int CTRL> __device__ __forceinline__ float row16(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float sum16(float v) {
    v += row16<0x128>(v);   // row_ror:8, 4, 2, 1
    v += row16<0x124>(v);
    v += row16<0x122>(v);
    v += row16<0x121>(v);
    return v;
}

template <int N, class T> struct alignas(N * sizeof(T) > 16 ? 16 : N * sizeof(T)) packed { T v[N]; };

template <class S, class T, int D, bool VEC>
__global__ __launch_bounds__(256) void k_page_put(put_args a) {
    constexpr int E = D / 16;
    const int heads = a.n_head + 2 * a.n_kv, j = threadIdx.x & 15;
    const long long item = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (item >= (long long)a.rows * heads) return;   // (whole groups of 16 lanes leave)
    const int row = (int)(item / heads), h = (int)(item - (long long)row * heads);
    const bool is_q = h < a.n_head, is_v = h >= a.n_head + a.n_kv;
    if (is_q && !a.q) return;
    const S* src = (const S*)a.qkv + (size_t)row * a.ld + (size_t)h * D + j * E;
    float x[E];
    if constexpr (VEC) {
        const packed<E, S> p = *(const packed<E, S>*)src;
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = to_f(p.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = to_f(src[e]);
    }
    bool there = true;
    if (!is_v) {
        const float* w = is_q ? a.q_norm : a.k_norm;
        if (w) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) ss = fmaf(x[e], x[e], ss);
            const float s = 1.0f / sqrtf(sum16(ss) * (1.0f / D) + a.eps);
#pragma unroll
            for (int e = 0; e < E; e++) x[e] = x[e] * s * w[j * E + e];
        }
    }
    if (a.rope) {
        const int pos = a.pos[row];
        there = pos >= 0 && pos < a.n_rope;
        if (!is_v) {
            const float2* cs = a.rope + (size_t)(there ? pos : 0) * (D / 2) + (j & 7) * E;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float other = row16<0x128>(x[e]);   // the value 8 lanes on: dimension + or - D / 2
                const float2 t = cs[e];
                x[e] = j < 8 ? fmaf(x[e], t.x, -(other * t.y)) : fmaf(x[e], t.x, other * t.y);
            }
        }
    }
    packed<E, T> o;
#pragma unroll
    for (int e = 0; e < E; e++) o.v[e] = (T)(is_q && !there ? 0.0f : x[e]);   // the one rounding, to nearest
    if (is_q) {
        *(packed<E, T>*)((T*)a.q + ((size_t)row * a.n_head + h) * D + j * E) = o;
        return;
    }
    const int64_t slot = a.slots[row];
    if (slot < 0 || slot >= a.n_slots || !there) return;
    const int g = is_v ? h - a.n_head - a.n_kv : h - a.n_head;
    const size_t pg = (size_t)(slot >> a.page_log), at = (size_t)(slot & ((1 << a.page_log) - 1));
    T* dst = (T*)(is_v ? a.values : a.keys) + (((pg * a.n_kv + g) << a.page_log) + at) * D + j * E;
    *(packed<E, T>*)dst = o;
}

template <class S, class T, int D> hipError_t put_vec(const put_args& a, hipStream_t s) {
    const long long items = (long long)a.rows * (a.n_head + 2 * a.n_kv), grid = (items + 15) / 16;
    constexpr size_t bytes = alignof(packed<D / 16, S>);
    const bool vec = (uintptr_t)a.qkv % bytes == 0 && (size_t)a.ld * sizeof(S) % bytes == 0;
    if (vec) k_page_put<S, T, D, true><<<dim3((unsigned)grid), 256, 0, s>>>(a);
    else k_page_put<S, T, D, false><<<dim3((unsigned)grid), 256, 0, s>>>(a);
    return hipGetLastError();
}
template <class S, class T> hipError_t put_dim(int D, const put_args& a, hipStream_t s) {
    return D == 32 ? put_vec<S, T, 32>(a, s) : D == 64 ? put_vec<S, T, 64>(a, s) : put_vec<S, T, 128>(a, s);
}
template <class T> hipError_t put_src(int D, int src, const put_args& a, hipStream_t s) {
    return src == TY_F32 ? put_dim<float, T>(D, a, s) : src == TY_F16 ? put_dim<_Float16, T>(D, a, s) : put_dim<__bf16, T>(D, a, s);
}

}  // namespace

hipError_t launch_page_plan(const plan_args& a, hipStream_t s) {
    // a workgroup for 1024 rows, at most four per compute unit
    const long long want = ((long long)a.rows + 1023) / 1024;
    const int grid = want < 1 ? 1 : want > 1024 ? 1024 : (int)want;
    const size_t lds = 2 * ((size_t)a.n + 1) * sizeof(int);
    // Four neighbouring rows a thread from as many rows on as two turns of a workgroup, whatever their requests: rows
    // that share a request and its page look them up once, and threads have fewer bisections. Below, one row a thread: four
    // chains of loads one after the other take longer than what they save. us one by one and by fours, at n x rows a request:
    // 1 x 256 4.5 and 5.1, 8 x 32 4.9 and 5.6, 64 x 4 4.3 and 5.1, 500 x 1 6.5 and 7.4; 8 x 64 5.7 and 5.6, 64 x 8 5.3 and 5.1;
    // 1 x 1024 6.2 and 5.2, 500 x 2 8.9 and 6.7, 64 x 64 8.3 and 6.1, 4000 x 1 20.5 and 18.4
    if (a.rows >= 2 * PLAN_T) k_page_plan<4><<<grid, PLAN_T, lds, s>>>(a);
    else k_page_plan<1><<<grid, PLAN_T, lds, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_page_put(int D, int src_type, int type, const put_args& a, hipStream_t s) {
    return type == TY_F16 ? put_src<_Float16>(D, src_type, a, s) : put_src<__bf16>(D, src_type, a, s);
}

}  // namespace sh
