// One workgroup's part of attention over keys and values in pages (sh_page_attn.hip, sh_tree_attn.hip): a tile of the
// (row, query head) columns of one kv head against a stretch of the shared positions or of a request's own.
#pragma once
#include <hip/hip_runtime.h>

#include <climits>

#include "sh_device.h"
#include "sh_serve.h"

namespace sh {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <class T> struct mat;
template <> struct mat<_Float16> {
    static constexpr unsigned EXP = 0x7C00u;   // the exponent bits of one value: all set in infinities and NaN
    static constexpr float SLACK = 4.0f, LIFT = 11.0f;   // weights up to 2^15; their last place is 2^-35 of the largest
    static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <> struct mat<__bf16> {
    static constexpr unsigned EXP = 0x7F80u;
    static constexpr float SLACK = 8.0f, LIFT = 0.0f;    // (eight bits of exponent hold any weight)
    static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <class T> __device__ __forceinline__ unsigned pack2(float x, float y) {
    typedef T t2 __attribute__((ext_vector_type(2)));
    const t2 v = {(T)x, (T)y};   // to nearest
    return __builtin_bit_cast(unsigned, v);
}
template <class T> __device__ __forceinline__ float of_bits(unsigned h) {
    return (float)__builtin_bit_cast(T, (unsigned short)h);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// e^(from - to) in powers of two for maxima that may be -inf (nothing seen yet)
__device__ __forceinline__ float rescale(float from, float to) { return from == -INFINITY ? 0.0f : exp2_(from - to); }

template <class F> __device__ __forceinline__ int over16(int v, F f) {   // the same value in the 16 lanes of a column group
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o));
    return v;
}
// the request whose rows hold `row` (the last k with cu[k] <= row)
__device__ __forceinline__ int request_of(const int32_t* cu, int n, int row) {
    int x = 0, y = n;
    while (y - x > 1) {
        const int mid = (x + y) >> 1;
        if (cu[mid] <= row) x = mid;
        else y = mid;
    }
    return x;
}

// what the four waves of a workgroup pass each other when they are joined: 16 NT columns of D sums (the pitch shifts
// columns by four banks), maxima and sums of weights, of two waves
template <int D, int NT> struct join_space {
    static constexpr int NC = 16 * NT, PITCH = D + 4;
    float o[2][NC * PITCH];
    float m[2][NC], l[2][NC];
};

// eight bits from bit `from` on of a row's mask; what lies before the first word is set, what lies behind the last one is not
__device__ __forceinline__ unsigned tree_bits(const pattn_args& a, int row, int from) {
    if (from <= -8) return 0xFFu;
    const unsigned* mask = a.mask + (size_t)row * a.words;
    if (from < 0) return ((mask[0] << -from) | ((1u << -from) - 1)) & 0xFFu;
    const int w = from >> 5;
    unsigned long long bits = 0;
    if (w < a.words) bits = mask[w];
    if (w + 1 < a.words) bits |= (unsigned long long)mask[w + 1] << 32;
    return (unsigned)(bits >> (from & 31)) & 0xFFu;
}

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
// TREE: a request's last positions are the words of a tree, one for each of its rows. A row sees all positions before them and
// the words whose bits are set in its mask, and its own position is the last one before them plus the bits that are set.
template <class T, int D, int NT, bool SHARED, bool TREE>
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
    [[maybe_unused]] int words_at = 0;     // TREE: place of the request's first tree word on the line
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
        int sure = INT_MAX;                // (below here the row sees every key from lo on)
        if constexpr (TREE) {
            const int k = SHARED ? request_of(a.cu, a.n, row[t]) : i;
            const long long first_row = a.cu[k], rows_k = a.cu[k + 1] - first_row, nth = row[t] - first_row;
            const int held = min(max(a.len[k], 0), own_max);
            const int base = (int)max(held - rows_k, 0ll);   // the tree's first word
            const unsigned* mask = a.mask + (size_t)row[t] * a.words;
            const bool node = held >= rows_k && nth >= 0 && nth < 32ll * a.words && (mask[nth >> 5] >> (nth & 31) & 1);
            int from = 0, first_word = 0;
            if (node && a.window) {
                int depth = -1;
                for (int w = 0; w < a.words; w++) depth += __popc(mask[w]);
                at = base + depth;
                from = (int)max(L0 + at + 1ll - a.window, 0ll);
                int drop = depth + 1 - a.window;   // of the words that it follows the window leaves the last ones
                for (int w = 0; w < a.words && drop > 0; w++) {
                    unsigned bits = mask[w];
                    const int n = __popc(bits);
                    if (n < drop) {
                        drop -= n;
                        continue;
                    }
                    for (; drop > 0; drop--) {
                        first_word = 32 * w + __ffs(bits);
                        bits &= bits - 1;
                    }
                }
            }
            if constexpr (SHARED) {
                lo[t] = node ? min(from, L0) : L0;
                hi[t] = L0;
            } else {
                words_at = P + base;
                lo[t] = first_word ? words_at + first_word : from >= L0 ? P + (from - L0) : a.fused ? from : P;
                hi[t] = node ? P + held : lo[t];
                sure = node ? words_at : 0;
            }
        } else {
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
        }
        lo0 = min(lo0, lo[t]);
        lo1 = max(lo1, lo[t]);
        hi0 = min(hi0, min(hi[t], sure));
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
                    unsigned bits = 0xFFu;         // of the lane's eight keys those that are before the tree, or in the row's branch
                    if constexpr (TREE && !SHARED)
                        if (!in_shared) bits = tree_bits(a, row[t], kt + quad * 8 - words_at);
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const int key = kt + quad * 8 + k;
                        x[k] = mine && key >= lo[t] && key < stop && (bits >> k & 1) ? x[k] : -INFINITY;
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
                                if constexpr (TREE && !SHARED)
                                    if (!in_shared && !(tree_bits(a, row[t], key - words_at) & 1)) continue;
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

// column groups of 16 a workgroup takes: one, or as many as the registers hold (prompts of 300 rows, head_dim 128: 40 us
// in tiles of 32 columns, 84 in tiles of 16, which read every key twice as often)
constexpr int attn_many(int D) { return D > 64 ? 2 : 4; }
inline int attn_col_groups(int D, long long cols) { return cols <= 16 ? 1 : attn_many(D); }

}  // namespace
}  // namespace sh
