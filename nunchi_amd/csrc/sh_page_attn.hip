// Attention of a batch of conversations over keys and values in pages: positions that all requests share, read once as
// one matrix product for all query rows, and each request's own. Parts of the keys are taken by workgroups of their own
// (k_page_attn) and joined after them (k_page_join): with a part's maximum m, sum l of e^(s - m) and sum O of e^(s - m) v,
// two parts have m' = max(m1, m2), l' = l1 e^(m1 - m') + l2 e^(m2 - m'), O' likewise, and the result is O / l.
//
// What bounds it: one row a request, memory (256 requests of up to 2048 own positions, 8 kv heads of 64: 607 MB in 120 us,
// 5.05 TB/s, as a copy; the shared 8192 positions for all 8192 columns alone take 40 us, together with the own ones 159, and the
// join 7); many rows, the exponentials and masks between the two products (VALU instructions outlast the matrix ones
// two to one at head_dim 64); a few short requests, the launch (two behind 90 positions: 6.5 us of kernel).
#include <hip/hip_runtime.h>

#include <climits>

#include "sh_attend.h"

namespace sh {
namespace {

// waves per SIMD that the registers are to allow: two where a workgroup holds 32 columns of 128 or 64 of 64 (256 requests behind
// 8192 positions 166 us; 32 columns of 64 at three or four waves 185 to 190, as each key feeds half the products)
constexpr int waves_of(int D, int nts, int nto) { return nts > 1 || nto > 1 ? 2 : D > 64 ? 3 : 4; }

// Shared and own parts in one launch, eight workgroups of either in turn (one for each XCD): the shared ones wait for the
// matrix units and the VALU, the own ones for memory (166 us for both at 256 requests; 173 as two launches).
template <class T, int D, int NTS, int NTO>
__global__ __launch_bounds__(256, waves_of(D, NTS, NTO)) void k_page_attn(pattn_args a) {
    __shared__ __align__(16) union { join_space<D, NTO> own; join_space<D, NTS ? NTS : 1> shared; } js;
    int b = blockIdx.x;
    if constexpr (NTS > 0) {
        const long long grp = b >> 3, gs = (a.shared_blocks + 7) >> 3, all = gridDim.x >> 3;
        const long long before = grp * gs / all, next = (grp + 1) * gs / all;   // shared groups before this one, with it
        if (next > before) {
            b = (int)(before * 8) + (b & 7);
            if (b < a.shared_blocks) attend<T, D, NTS ? NTS : 1, true, false>(a, b, js.shared);
            return;
        }
        b = (int)((grp - before) * 8) + (b & 7);
        if (b >= a.own_blocks) return;
    }
    attend<T, D, NTO, false, false>(a, b, js.own);
}

// One wave per (row, query head), or all four for many parts: lanes take four dimensions each, as many parts at once as
// fit a wave. All four from 17 parts on: a wave alone reads them in turns that wait for each other. With few parts the
// other waves only cost. us a call of both kernels with one wave and with four, 32 heads of 64: one request 2 parts 8.3 and
// 8.5, 8 parts 8.4 and 8.6, 12 parts 8.7 and 8.6, 16 parts 9.1 and 8.8, 32 parts 10.1 and 9.6, 128 parts 44 and 32; 8 requests
// 4 parts 8.5 and 8.8, 16 parts 18.4 and 17.2; 256 requests of few parts: the join alone 7.3 and 14.
template <class T, int D, bool MANY>
__global__ __launch_bounds__(256) void k_page_join(pattn_args a) {
    constexpr int LP = D / 4, AT_ONCE = 64 / LP, WAVES = MANY ? 4 : 1;   // lanes per part, parts at once
    __shared__ f32x4 o_s[MANY ? 4 : 1][LP];
    __shared__ float l_s[4];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, parts = a.sp + a.so;
    const size_t rh = MANY ? (size_t)blockIdx.x : (size_t)blockIdx.x * 4 + wv, stride = (size_t)a.rows * a.n_head;
    if (rh >= stride) return;
    const int row = (int)(rh / a.n_head);
    if (a.cu) {   // rows behind the last request, and those past max_rows of theirs, have no parts
        const int k = request_of(a.cu, a.n, row), first = max(a.cu[k], 0);
        if (row < first || row >= a.cu[k + 1] || row - first >= a.max_rows) return;
    }
    float m = -INFINITY;
    for (int p = lane; p < parts; p += 64) {
        const float2 ml = a.part_ml[p * stride + rh];
        if (ml.y != 0.0f) m = fmaxf(m, ml.x);
    }
    m = wave_max(m);
    float l = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    const int d = (lane % LP) * 4;
#pragma unroll 4
    for (int p = (MANY ? wv * AT_ONCE : 0) + lane / LP; p < parts; p += WAVES * AT_ONCE) {
        const float2 ml = a.part_ml[p * stride + rh];
        if (ml.y == 0.0f) continue;
        const float f = exp2_(ml.x - m);
        l += ml.y * f;
        o += *(const f32x4*)(a.part_o + (p * stride + rh) * D + d) * f;
    }
#pragma unroll
    for (int k = LP; k < 64; k *= 2) {
        l += __shfl_xor(l, k);
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] += __shfl_xor(o[e], k);
    }
    if constexpr (MANY) {
        if (lane < LP) o_s[wv][lane] = o;
        if (lane == 0) l_s[wv] = l;
        __syncthreads();
        if (threadIdx.x >= LP) return;
        l = (l_s[0] + l_s[1]) + (l_s[2] + l_s[3]);
        o = (o_s[0][lane] + o_s[1][lane]) + (o_s[2][lane] + o_s[3][lane]);
    } else if (lane >= LP) {
        return;
    }
    float f = l == 0.0f ? 0.0f : 1.0f / l;
    if (a.gate) f *= 1.0f / (1.0f + expf(-a.gate[rh]));
    uint2 w = {0u, 0u};
    if (l != 0.0f) w = uint2{pack2<T>(o[0] * f, o[1] * f), pack2<T>(o[2] * f, o[3] * f)};
    *(uint2*)((T*)a.out + rh * D + d) = w;
    if (a.lse && d == 0) a.lse[rh] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

long long shared_tiles(const pattn_args& a, int nt) { return ((long long)a.rows * a.grp + 16 * nt - 1) / (16 * nt); }
long long own_tiles(const pattn_args& a, int nt, bool single) {
    return single ? (long long)a.n * ((a.grp + 16 * nt - 1) / (16 * nt)) : (long long)a.rows * a.grp / (16 * nt) + a.n;
}

template <class T, int D, int NTS, int NTO> hipError_t run_attn(const pattn_args& a, hipStream_t s) {
    const long long blocks = NTS ? ((a.shared_blocks + 7ll) / 8 + (a.own_blocks + 7ll) / 8) * 8 : a.own_blocks;
    k_page_attn<T, D, NTS, NTO><<<dim3((unsigned)blocks), 256, 0, s>>>(a);
    return hipGetLastError();
}
template <class T, int D> hipError_t run_join(const pattn_args& a, hipStream_t s) {
    if (a.sp + a.so == 1) return hipSuccess;
    const long long rh = (long long)a.rows * a.n_head;
    if (a.sp + a.so > 16) k_page_join<T, D, true><<<dim3((unsigned)rh), 256, 0, s>>>(a);
    else k_page_join<T, D, false><<<dim3((unsigned)((rh + 3) / 4)), 256, 0, s>>>(a);
    return hipGetLastError();
}
template <class T, int D> hipError_t run_all(const pattn_args& a, hipStream_t s) {
    constexpr int M = attn_many(D);
    const int nts = a.sp ? attn_col_groups(D, (long long)a.rows * a.grp) : 0, nto = attn_col_groups(D, (long long)a.max_rows * a.grp);
    hipError_t e;
    if (nts == 0) e = nto == 1 ? run_attn<T, D, 0, 1>(a, s) : run_attn<T, D, 0, M>(a, s);
    else if (nts == 1) e = run_attn<T, D, 1, 1>(a, s);   // (a request has no more columns than all of them)
    else e = nto == 1 ? run_attn<T, D, M, 1>(a, s) : run_attn<T, D, M, M>(a, s);
    return e == hipSuccess ? run_join<T, D>(a, s) : e;
}
template <class T> hipError_t run_dim(int D, const pattn_args& a, hipStream_t s) {
    return D == 32 ? run_all<T, 32>(a, s) : D == 64 ? run_all<T, 64>(a, s) : run_all<T, 128>(a, s);
}

void split(long long base, long long range, long long want, int* parts, int* chunk) {
    long long p = want / (base > 0 ? base : 1), most = (range + 255) / 256;
    if (p > most) p = most;
    if (p < 1) p = 1;
    const long long c = ((range + p - 1) / p + 127) / 128 * 128;
    *chunk = (int)(c < 128 ? 128 : c);
    *parts = (int)((range + *chunk - 1) / *chunk);
    if (*parts < 1) *parts = 1;
}

}  // namespace

// Which workgroups take the shared positions, and into how many parts the keys go: about four workgroups per compute
// unit (two for the shared positions), of 256 keys or more. With twice as many parts 48 requests of 4096 positions took 63 to
// 66 us instead of 62, the prompts below 76 instead of 40.
bool page_attn_split(int D, bool single, pattn_args& a) {
    const int nto = attn_col_groups(D, (long long)a.max_rows * a.grp);
    const long long own = own_tiles(a, nto, single), all = shared_tiles(a, attn_col_groups(D, (long long)a.rows * a.grp));
    a.own_at = (a.prefix_len + 31) / 32 * 32;
    // Requests whose columns fill their workgroups read the shared positions themselves: sharing would not save reads,
    // and nothing has to be joined (13 prompts of 300 rows behind 500 positions: 40 us, 138 apart). us fused and apart for 16
    // requests behind 1024 positions, 8 kv heads of 64: 16 rows each (own = 2 all) 22 and 28, 64 rows 26 and 57; 8 rows
    // (own = 3 all) 24 and 17.
    // So do few requests with few shared positions: own tiles times positions, one row each: 32 x 128 5.4 and 11.8, 4 x 1024
    // 8.6 and 8.6, 16 x 256 8.4 and 12.5. Past 4096 it depends on the columns: with 16 a workgroup it pays up to about 32768
    // (64 x 512 15.8 and 16.1, 64 x 1024 21.5 and 16.6), with 64 no longer at 6144 (16 requests of 8 rows behind 256: 15.6 and
    // 14.1), so the bound is what holds for both
    a.fused = a.prefix_len == 0 || own <= all * 2 || own * a.prefix_len <= 4096;
    a.sp = a.pchunk = 0;
    if (!a.fused) {
        const long long range = a.window && a.window + 31ll < a.prefix_len ? a.window + 31ll : a.prefix_len;
        split(all * a.n_kv, range, 512, &a.sp, &a.pchunk);
    }
    long long range = (a.fused ? a.own_at : 0ll) + a.max_len;
    if (a.window) {
        const long long rows = 16ll * nto / a.grp + 2, seen = a.window + 63ll + (rows < a.max_rows ? rows : a.max_rows);
        if (seen < range) range = seen;
    }
    split(own * a.n_kv, range, 1024, &a.so, &a.ochunk);
    const long long shared_blocks = all * a.n_kv * a.sp, own_blocks = own * a.n_kv * a.so;
    const long long rh = (long long)a.rows * a.n_head, join = a.sp + a.so == 1 ? 0 : a.sp + a.so > 16 ? rh : (rh + 3) / 4;
    // (columns of one kv head are counted in 32 bits in the kernel)
    if (shared_blocks + own_blocks + 16 > most_blocks(256) || join > most_blocks(256) || (long long)a.rows * a.grp > INT_MAX / 2) return false;
    a.shared_blocks = (int)shared_blocks;
    a.own_blocks = (int)own_blocks;
    return true;
}

hipError_t launch_page_join(int D, int type, const pattn_args& a, hipStream_t s) {
    if (type == TY_F16) return D == 32 ? run_join<_Float16, 32>(a, s) : D == 64 ? run_join<_Float16, 64>(a, s) : run_join<_Float16, 128>(a, s);
    return D == 32 ? run_join<__bf16, 32>(a, s) : D == 64 ? run_join<__bf16, 64>(a, s) : run_join<__bf16, 128>(a, s);
}

hipError_t launch_page_attn(int D, int type, const pattn_args& a, hipStream_t s) {
    return type == TY_F16 ? run_dim<_Float16>(D, a, s) : run_dim<__bf16>(D, a, s);
}

}  // namespace sh
