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

template <class T> __device__ __forceinline__ float of_bits(unsigned h) {
    return (float)__builtin_bit_cast(T, (unsigned short)h);
}

template <class F> __device__ __forceinline__ int over16(int v, F f) {   // the same value in the 16 lanes of a column group
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o));
    return v;
}

// what the four waves of a workgroup pass each other when they are joined: 16 NT columns of D sums (the pitch shifts
// columns by four banks), maxima and sums of weights, of two waves
template <int D, int NT> struct join_space {
    static constexpr int NC = 16 * NT, PITCH = D + 4;
    float o[2][NC * PITCH];
    float m[2][NC], l[2][NC];
};

// Keys are counted along one line: the shared positions, a gap to the next multiple of 32, the request's own.
// Columns: the (row, query head) pairs of one kv head, packed; a workgroup takes 16 NT of them and one part of the line,
// its four waves take blocks of 32 keys in turn. With K of 32 keys as rows of the first product (S^T = K Q^T) a lane
// holds the scores of one column, so maxima and sums stay in the lane; rows are dealt to the product so that a lane's
// eight scores are eight neighbouring keys, which are its operand of the second product (O^T = V^T P^T) as they are.
// V's operand is eight keys of one dimension: each lane loads the same D / 16 dimensions of eight keys and turns the
// block with byte permutes. Nothing passes through LDS before the waves are joined. Weights are rounded to the values'
// 16 bits for the second product, as the matrix units take them; their sum stays in 32 bits. They are relative to a
// maximum that is up to 2^SLACK behind the true one (the accumulators are rescaled only when a score passes it by more)
// and 2^LIFT below it: with f16's five bits of exponent, weights below 2^-25 of the largest would all be lost, and a
// hundred thousand of them are a part of the sum that shows.
// SHARED: the columns of all requests over the shared positions. Else one request's columns over its own positions, and
// over the shared ones before them where no SHARED part takes them (a.fused).
template <class T, int D, int NT, bool SHARED>
__device__ __forceinline__ void attend(const pattn_args& a, const int block, join_space<D, NT>& js) {
    constexpr int NC = 16 * NT, E = D / 16, CH = D / 32, VW = E / 2, PITCH = join_space<D, NT>::PITCH;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m16 = lane & 15, quad = lane >> 4;
    const int S = SHARED ? a.sp : a.so, per = a.n_kv * S;
    // (workgroups of the same keys are `per` apart: on one XCD where that is a multiple of 8)
    const int gs = block % per, g = gs % a.n_kv, part = gs / a.n_kv;
    const int tile = block / per;
    // ---- the workgroup's columns ----
    int i = 0, r0 = 0, r1, ct = tile;      // request, its rows, tile of columns within them
    if constexpr (SHARED) {
        r1 = a.cu ? min(max(a.cu[a.n], 0), a.rows) : a.rows;
    } else if (!a.cu) {
        const int tpr = (a.grp + NC - 1) / NC;
        i = tile / tpr;
        ct = tile - i * tpr;
        r0 = i;
        r1 = i + 1;
    } else {
        // request i owns the tiles first(i) .. first(i + 1) - 1, at least as many as its columns fill
        auto row_at = [&](int k) { return min(max(a.cu[k], 0), a.rows); };
        auto first = [&](int k) { return (int)((long long)row_at(k) * a.grp / NC) + k; };
        int lo = 0, hi = a.n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first(mid) <= tile) lo = mid;
            else hi = mid;
        }
        i = lo;
        ct = tile - first(i);
        r0 = row_at(i);
        r1 = min(row_at(i + 1), r0 + a.max_rows);
    }
    const int ncol = (r1 - r0) * a.grp, c0 = ct * NC;
    if (c0 < 0 || c0 >= ncol) return;
    // ---- what each column sees: keys lo .. hi - 1 of the line, the gap left out ----
    const int L0 = a.prefix_len, P = a.own_at;
    int row[NT], head[NT], lo[NT], hi[NT];
    bool live[NT];
    const int own_max = (int)min((long long)a.max_len, (long long)a.cols << a.page_log);
    int lo0 = INT_MAX, lo1 = 0, hi0 = INT_MAX, hi1 = 0;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int c = c0 + 16 * t + m16, cc = min(c, ncol - 1);
        live[t] = c < ncol;
        row[t] = r0 + cc / a.grp;
        head[t] = g * a.grp + cc % a.grp;
        int at = 0;                        // the row's own position, counted from the first that is not shared
        if (!SHARED || a.window) {
            const int k = !SHARED ? i : a.cu ? request_of(a.cu, a.n, row[t]) : row[t];
            const int first_row = a.cu ? a.cu[k] : k, rows_k = a.cu ? a.cu[k + 1] - first_row : 1;
            // (at most its last place: row starts that contradict each other lead nowhere else)
            at = (int)max(min(min(max(a.len[k], 0), own_max) - (long long)rows_k + (row[t] - first_row), own_max - 1ll), -1ll - a.rows);
        }
        // the first position of the line that a window leaves
        const int from = a.window ? (int)max(L0 + at + 1ll - a.window, 0ll) : 0;
        if constexpr (SHARED) {
            lo[t] = min(max(from, 0), L0);
            hi[t] = L0;
        } else {
            lo[t] = from >= L0 ? P + (from - L0) : a.fused ? max(from, 0) : P;
            hi[t] = at >= 0 ? P + at + 1 : a.fused ? L0 : P;
        }
        lo0 = min(lo0, lo[t]);
        lo1 = max(lo1, lo[t]);
        hi0 = min(hi0, hi[t]);
        hi1 = max(hi1, hi[t]);
    }
    auto mn = [](int x, int y) { return min(x, y); };
    auto mx = [](int x, int y) { return max(x, y); };
    lo0 = __builtin_amdgcn_readfirstlane(over16(lo0, mn));
    lo1 = __builtin_amdgcn_readfirstlane(over16(lo1, mx));
    hi0 = __builtin_amdgcn_readfirstlane(over16(hi0, mn));
    hi1 = __builtin_amdgcn_readfirstlane(over16(hi1, mx));
    // ---- the part: the first starts where the first column does; the last goes to the end ----
    const int chunk = SHARED ? a.pchunk : a.ochunk;
    const long long k0l = (long long)(lo0 & ~31) + (long long)part * chunk;
    const int k1 = part + 1 == S ? hi1 : (int)min((long long)hi1, k0l + chunk);
    const bool any = k0l < k1;
    const int k0 = any ? (int)k0l : 0;

    f32x4 o[E][NT];
    float m[NT], l[NT];
    u32x4 qf[CH][NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        m[t] = -INFINITY;
        l[t] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) o[e][t] = f32x4{0, 0, 0, 0};
    }
    if (any) {
        const T* qp = (const T*)a.q;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int c = 0; c < CH; c++)
                qf[c][t] = *(const u32x4*)(qp + ((size_t)row[t] * a.n_head + head[t]) * D + c * 32 + quad * 8);
        const int32_t* own = SHARED ? nullptr : a.table + (size_t)i * a.cols;
        const int pl = a.page_log, pm = (1 << pl) - 1;
        const size_t page_sz = ((size_t)a.n_kv << pl) * D;
        const T* kp = (const T*)a.keys + ((size_t)g << pl) * D;
        const T* vp = (const T*)a.values + ((size_t)g << pl) * D;
        const int koff = ((m16 >> 2) << 3) + (m16 & 3);
        for (int kt = k0 + 32 * wv; kt < k1; kt += 128) {
            // a block of 32 keys lies in one page, or in two of 16; behind `last` of its table there are none
            const bool in_shared = SHARED || kt < P;
            const int32_t* tab = in_shared ? a.prefix : own;
            const int k_at = in_shared ? kt : kt - P, last = in_shared ? L0 - 1 : hi1 - 1 - P, ahead = last - k_at;
            if (!SHARED && ahead < 0) continue;   // (the gap alone)
            const int id0 = tab[k_at >> pl], id1 = pl == 4 ? tab[min(k_at + 16, last) >> 4] : id0;
            const bool ok0 = (unsigned)id0 < (unsigned)a.n_pages, ok1 = (unsigned)id1 < (unsigned)a.n_pages;
            const size_t b0 = (ok0 ? (size_t)id0 : 0) * page_sz, b1 = (ok1 ? (size_t)id1 : 0) * page_sz;
            auto at = [&](int off) {       // place of key kt + off (the last one where it is past the end)
                const int f = min(off, ahead);
                return pl == 4 ? ((f & 16) ? b1 : b0) + (size_t)(f & 15) * D : b0 + (size_t)((k_at & pm) + f) * D;
            };
            u32x4 kf[2][CH];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const T* p = kp + at(koff + 4 * t) + quad * 8;
#pragma unroll
                for (int c = 0; c < CH; c++) kf[t][c] = *(const u32x4*)(p + c * 32);
            }
            unsigned vw[8][VW];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const T* p = vp + at(quad * 8 + k) + m16 * E;
                if constexpr (VW == 4) *(u32x4*)vw[k] = *(const u32x4*)p;
                else if constexpr (VW == 2) *(uint2*)vw[k] = *(const uint2*)p;
                else vw[k][0] = *(const unsigned*)p;
            }
            const bool full = kt >= lo1 && kt + 32 <= hi0 && ahead >= 31 && ok0 && ok1;
            const bool mine = quad >= 2 ? ok1 : ok0;
            const int end = kt + ahead + 1;
            unsigned pw[NT][4];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                float x[8];
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    f32x4 s = {0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < CH; c++) s = mat<T>::mul(kf[b][c], qf[c][t], s);
#pragma unroll
                    for (int r = 0; r < 4; r++) x[4 * b + r] = s[r];
                }
                if (!full) {
                    const int stop = min(hi[t], end);
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const int key = kt + quad * 8 + k;
                        x[k] = mine && key >= lo[t] && key < stop ? x[k] : -INFINITY;
                    }
                }
                float top = x[0];          // (NaN is passed over)
#pragma unroll
                for (int k = 1; k < 8; k++) top = fmaxf(top, x[k]);
                top *= a.c;
                if (__any(top > m[t] + (mat<T>::SLACK + mat<T>::LIFT))) {
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float to = fmaxf(m[t], top - mat<T>::LIFT), f = rescale(m[t], to);
                    l[t] *= f;
#pragma unroll
                    for (int e = 0; e < E; e++) o[e][t] *= f;
                    m[t] = to;
                }
                const float ref = m[t] == -INFINITY ? 0.0f : m[t];
                float sum = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    x[k] = exp2_(fmaf(x[k], a.c, -ref));
                    sum += x[k];
                }
                l[t] += sum;
#pragma unroll
                for (int k = 0; k < 4; k++) pw[t][k] = pack2<T>(x[2 * k], x[2 * k + 1]);
            }
            if (!full) {
                bool odd = false;          // infinities or NaN among the values of a block that columns see in part
                const int stop = min(hi1, end);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int key = kt + quad * 8 + k;
                    const bool seen = mine && key >= lo0 && key < stop;
#pragma unroll
                    for (int w = 0; w < VW; w++) {
                        vw[k][w] = seen ? vw[k][w] : 0u;
                        odd |= (vw[k][w] & mat<T>::EXP) == mat<T>::EXP || ((vw[k][w] >> 16) & mat<T>::EXP) == mat<T>::EXP;
                    }
                }
                if (__any(odd)) {
                    // A weight of 0 times an infinity would reach columns that do not see the key: such values are
                    // left out of the product and added to the columns that do, key by key
#pragma unroll
                    for (int k = 0; k < 8; k++) {
#pragma unroll
                        for (int w = 0; w < VW; w++) {
                            if ((vw[k][w] & mat<T>::EXP) == mat<T>::EXP) vw[k][w] &= 0xFFFF0000u;
                            if (((vw[k][w] >> 16) & mat<T>::EXP) == mat<T>::EXP) vw[k][w] &= 0x0000FFFFu;
                        }
                        for (int kq = 0; kq < 4; kq++) {
                            const int key = kt + kq * 8 + k;
                            const bool there = (kq >= 2 ? ok1 : ok0) && key < stop;
                            const T* p = vp + at(kq * 8 + k) + quad * 4 * E;   // this lane's dimensions of O
#pragma unroll
                            for (int t = 0; t < NT; t++) {
                                const unsigned two = __shfl(pw[t][k >> 1], kq * 16 + m16);
                                const float w = of_bits<T>(k & 1 ? two >> 16 : two & 0xFFFFu);
                                if (!there || key < lo[t] || key >= hi[t]) continue;
#pragma unroll
                                for (int r = 0; r < 4; r++)
#pragma unroll
                                    for (int e = 0; e < E; e++) {
                                        const float v = (float)p[r * E + e];
                                        if (!(fabsf(v) < INFINITY)) o[e][t][r] += w * v;
                                    }
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < E; e++) {  // dimension m16 * E + e of eight keys
                const unsigned sel = (e & 1) ? 0x07060302u : 0x05040100u;
                u32x4 vf;
#pragma unroll
                for (int k = 0; k < 4; k++) vf[k] = __builtin_amdgcn_perm(vw[2 * k + 1][e >> 1], vw[2 * k][e >> 1], sel);
#pragma unroll
                for (int t = 0; t < NT; t++) o[e][t] = mat<T>::mul(vf, u32x4{pw[t][0], pw[t][1], pw[t][2], pw[t][3]}, o[e][t]);
            }
        }
    }
    // ---- the four waves joined: 2 and 3 into 0 and 1, then 1 into 0 ----
#pragma unroll
    for (int t = 0; t < NT; t++) {
        l[t] += __shfl_xor(l[t], 16);
        l[t] += __shfl_xor(l[t], 32);
    }
#pragma unroll
    for (int step = 2; step > 0; step >>= 1) {
        if (k0 + 32 * step >= k1) continue;   // (waves from `step` on had no block)
        if (wv >= step && wv < 2 * step) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const int c = 16 * t + m16;
                if (quad == 0) {
                    js.m[wv - step][c] = m[t];
                    js.l[wv - step][c] = l[t];
                }
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int e = 0; e < E; e++) js.o[wv - step][c * PITCH + (quad * 4 + r) * E + e] = o[e][t][r];
            }
        }
        __syncthreads();
        if (wv < step) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const int c = 16 * t + m16;
                const float m2 = js.m[wv][c], l2 = js.l[wv][c];
                const float to = fmaxf(m[t], m2), f1 = rescale(m[t], to), f2 = rescale(m2, to);
                m[t] = to;
                l[t] = l[t] * f1 + l2 * f2;
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int e = 0; e < E; e++)
                        o[e][t][r] = o[e][t][r] * f1 + js.o[wv][c * PITCH + (quad * 4 + r) * E + e] * f2;
            }
        }
        __syncthreads();
    }
    if (wv) return;
    const bool alone = a.sp + a.so == 1;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        if (!live[t]) continue;
        const size_t rh = (size_t)row[t] * a.n_head + head[t];
        if (alone) {
            float f = l[t] == 0.0f ? 0.0f : 1.0f / l[t];
            if (a.gate) f *= 1.0f / (1.0f + expf(-a.gate[rh]));
            unsigned* dst = (unsigned*)((T*)a.out + rh * D + quad * 4 * E);
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const float x = o[e][t][r], y = o[e + 1][t][r];
                    dst[(r * E + e) / 2] = l[t] == 0.0f ? 0u : pack2<T>(x * f, y * f);
                }
            if (a.lse && quad == 0) a.lse[rh] = l[t] == 0.0f ? -INFINITY : (m[t] + log2f(l[t])) * 0.69314718055994531f;
        } else {
            const size_t at = (size_t)(SHARED ? part : a.sp + part) * a.rows * a.n_head + rh;
            if (quad == 0) a.part_ml[at] = make_float2(m[t], l[t]);
            if (any) {
                float* dst = a.part_o + at * D + quad * 4 * E;
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int e = 0; e < E; e++) dst[r * E + e] = o[e][t][r];
            }
        }
    }
}

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
            if (b < a.shared_blocks) attend<T, D, NTS ? NTS : 1, true>(a, b, js.shared);
            return;
        }
        b = (int)((grp - before) * 8) + (b & 7);
        if (b >= a.own_blocks) return;
    }
    attend<T, D, NTO, false>(a, b, js.own);
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

// column groups of 16 a workgroup takes: one, or as many as the registers hold (prompts of 300 rows, head_dim 128: 40 us
// in tiles of 32 columns, 84 in tiles of 16, which read every key twice as often)
constexpr int many(int D) { return D > 64 ? 2 : 4; }
int col_groups(int D, long long cols) { return cols <= 16 ? 1 : many(D); }

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
    constexpr int M = many(D);
    const int nts = a.sp ? col_groups(D, (long long)a.rows * a.grp) : 0, nto = col_groups(D, (long long)a.max_rows * a.grp);
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
    const int nto = col_groups(D, (long long)a.max_rows * a.grp);
    const long long own = own_tiles(a, nto, single), all = shared_tiles(a, col_groups(D, (long long)a.rows * a.grp));
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
