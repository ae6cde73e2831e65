// One word for each row of scores: temperature, top-k, top-p, min-p and a given random number (include/seoul_hip.h:
// sh_sample).
//
// With w(x) = e^((x - max) / temp) the kept words are, in the order (score descending, index ascending), a beginning cut
// by count (top-k) or by weight (top-p), of which min-p leaves those above a score: all of them the words above one score
// t, some of the words equal to t (the first r by index), above another. So nothing is sorted: t is found by histograms,
// the first over the weights' exponent (64 powers of two in 2048 bins), the next over the bits of the scores inside the
// bin that holds the cut, until one score is left. The pick is a search for the running sum in index order, first over
// the sums of 64-lane blocks, then within one.
// Weights are summed as integers, in 2^-44ths of the largest: sums do not depend on their order, so neither atomics nor
// the layout change a result. A weight is formed from the score's distance in double (its rounding in single would move
// it by up to 1e-6) with the hardware's 2^x, exact to 2^-23.
#include <hip/hip_runtime.h>

#include "sh_device.h"
#include "sh_serve.h"

namespace sh {
namespace {

constexpr int ST = 1024, SW = ST / 64;     // threads and waves per row
constexpr int BINS = 2048;
constexpr int MAX_BLOCKS = SAMPLE_MAX_VOCAB / 256;   // blocks of a wave's neighbouring words (64 lanes of 4 or 8)

typedef unsigned long long u64;

// scores as numbers that sort like them
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x);
    return b ^ ((int)b < 0 ? 0xFFFFFFFFu : 0x80000000u);
}

template <class T> struct score;
template <> struct score<float> {
    static constexpr int V = 4;
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    static __device__ __forceinline__ void unpack(const vec& v, float* x) {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = v[e];
    }
};
template <class T> struct score16 {
    static constexpr int V = 8;
    typedef T vec __attribute__((ext_vector_type(8), aligned(2)));
    static __device__ __forceinline__ void unpack(const vec& v, float* x) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)v[e];
    }
};
template <> struct score<_Float16> : score16<_Float16> {};
template <> struct score<__bf16> : score16<__bf16> {};

struct row_shared {
    unsigned cnt[2][BINS];     // words per bin: [0] the first histogram, [1] the finer ones
    u64 mass[2][BINS];         // and their weights
    u64 blocks[MAX_BLOCKS];    // sums of blocks of neighbouring words
    u64 wsum[2][SW];
    float wmax[SW];
    int widx[SW];
    unsigned kmin, kmax;
    u64 found[4];
};

// inclusive sum over the workgroup of two numbers per thread
__device__ __forceinline__ void scan2(row_shared& s, u64& a, u64& b) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 x = __shfl_up(a, o), y = __shfl_up(b, o);
        if (lane >= o) { a += x; b += y; }
    }
    if (lane == 63) { s.wsum[0][wv] = a; s.wsum[1][wv] = b; }
    __syncthreads();
    u64 pa = 0, pb = 0;
    for (int w = 0; w < wv; w++) { pa += s.wsum[0][w]; pb += s.wsum[1][w]; }
    a += pa;
    b += pb;
    __syncthreads();
}

template <class T>
__global__ __launch_bounds__(ST) void k_sample(sample_args a) {
    constexpr int V = score<T>::V;
    typedef typename score<T>::vec vec;
    extern __shared__ __align__(16) char lds_raw[];
    row_shared& s = *reinterpret_cast<row_shared*>(lds_raw);
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const T* x = (const T*)a.scores + (size_t)row * a.ld;
    auto load = [&](int at, float* v) {    // V neighbouring scores (-inf past the end, NaN as -inf, -0 as 0)
        if (at + V <= a.vocab) {
            score<T>::unpack(*(const vec*)(x + at), v);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = at + e < a.vocab ? (float)x[at + e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = v[e] != v[e] ? -INFINITY : v[e] + 0.0f;
    };
    auto each = [&](auto f) {
        for (int at = t * V; at - lane * V < a.vocab; at += ST * V) {   // (whole waves)
            float v[V];
            load(at, v);
            f(v, at);
        }
    };
    // ---- the maximum, and where it first is ----
    float top = -INFINITY;
    int first = 0x7FFFFFFF;
    each([&](const float* v, int at) {
#pragma unroll
        for (int e = 0; e < V; e++)
            if (v[e] > top) { top = v[e]; first = at + e; }
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(top, o);
        const int i2 = __shfl_xor(first, o);
        if (m2 > top || (m2 == top && i2 < first)) { top = m2; first = i2; }
    }
    if (lane == 0) { s.wmax[wv] = top; s.widx[wv] = first; }
    __syncthreads();
    for (int w = 0; w < SW; w++) {
        const float m2 = s.wmax[w];
        const int i2 = s.widx[w];
        if (m2 > top || (m2 == top && i2 < first)) { top = m2; first = i2; }
    }
    const float temp = a.temp ? a.temp[row] : 1.0f;
    const bool none = top == -INFINITY || !(temp >= 0.0f);
    if (none || temp == 0.0f) {
        if (t == 0) {
            a.ids[row] = none ? -1 : first;
            if (a.chance) a.chance[row] = none ? 0.0f : 1.0f;
        }
        return;
    }
    // ---- weights ----
    const double c = 1.4426950408889634 / (double)temp;
    const bool inf = top == INFINITY;
    auto valid = [&](float v) { return inf ? v == top : v > -INFINITY; };
    auto dist = [&](float v) { return v == top ? 0.0 : ((double)top - (double)v) * c; };   // -log2 of the weight
    auto weight = [&](double d) {
        const float hi = (float)d, lo = (float)(d - (double)hi);
        const float w = __builtin_amdgcn_exp2f(-hi);
        return hi < 126.0f ? w - w * (lo * 0.69314718f) : 0.0f;
    };
    auto fixed = [&](float w) {
        const float h = w * 4096.0f;
        const unsigned hi = (unsigned)h;
        return ((u64)hi << 32) | (unsigned)((h - (float)hi) * 4294967296.0f);
    };
    auto bin_of = [&](double d) { return d < 64.0 ? (int)(d * 32.0) : BINS - 1; };
    // ---- the cut: words above key tau, and the first r of the n_eq words equal to it ----
    const int top_k = a.top_k ? a.top_k[row] : 0;
    float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f;
    if (!(top_p < 1.0f)) top_p = 1.0f;
    if (top_p < 0.0f) top_p = 0.0f;
    const bool by_k = top_k > 0, by_p = top_p < 1.0f;
    unsigned tau = 0;          // (0: below every score's key)
    unsigned cut = 0xFFFFFFFFu;   // words equal to tau are kept up to this index

    // the first index at which the running sum of f over the words passes `target`, and that word's place in s.found;
    // f gives a u64 per word
    auto locate = [&](auto f, auto target_of) {
        const int nb = (a.vocab + 64 * V - 1) / (64 * V);
        each([&](const float* v, int at) {
            u64 sum = 0;
#pragma unroll
            for (int e = 0; e < V; e++) sum += f(v[e], at + e);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
            if (lane == 0) s.blocks[at / (64 * V)] = sum;
        });
        __syncthreads();
        constexpr int PER = MAX_BLOCKS / ST;
        u64 mine = 0, unused = 0;
        for (int k = 0; k < PER; k++)
            if (t * PER + k < nb) mine += s.blocks[t * PER + k];
        u64 up = mine;
        scan2(s, up, unused);
        if (t == ST - 1) s.found[0] = up;
        __syncthreads();
        const u64 total = s.found[0], target = target_of(total);
        u64 at = up - mine;
        if (at <= target && target < up) {   // one thread's blocks hold it
            int b = t * PER;
            while (at + s.blocks[b] <= target) at += s.blocks[b++];
            s.found[1] = (u64)b;
            s.found[2] = at;
        }
        __syncthreads();
        const int b = (int)s.found[1];
        u64 before = s.found[2];
        __syncthreads();
        int got = -1;
        if (wv == 0) {
            float v[V];
            const int w0 = (b * 64 + lane) * V;
            load(w0, v);
            u64 own = 0;
#pragma unroll
            for (int e = 0; e < V; e++) own += f(v[e], w0 + e);
            u64 in = own;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const u64 y = __shfl_up(in, o);
                if (lane >= o) in += y;
            }
            before += in - own;
            if (before <= target && target < before + own) {
                int e = 0;
                while (before + f(v[e], w0 + e) <= target) before += f(v[e], w0 + e), e++;
                got = w0 + e;
                s.found[3] = (u64)got;
            }
        }
        __syncthreads();
        return (int)s.found[3];
    };

    if (by_k || by_p) {
        auto clear = [&](int k) {
            for (int b = t; b < BINS; b += ST) { s.cnt[k][b] = 0; s.mass[k][b] = 0; }
            __syncthreads();
        };
        clear(0);
        each([&](const float* v, int) {
#pragma unroll
            for (int e = 0; e < V; e++) {
                if (!valid(v[e])) continue;
                const double d = dist(v[e]);
                const int b = bin_of(d);
                atomicAdd(&s.cnt[0][b], 1u);
                const u64 w = fixed(weight(d));
                if (w) atomicAdd(&s.mass[0][b], w);
            }
        });
        __syncthreads();
        // the first bin at which `reached(count, mass)` holds for the sums up to it; what lies before it
        u64 n_before = 0, m_before = 0, n_bin = 0;
        auto find = [&](int k, auto reached) {
            constexpr int PER = BINS / ST;
            u64 n = 0, m = 0;
            for (int j = 0; j < PER; j++) { n += s.cnt[k][t * PER + j]; m += s.mass[k][t * PER + j]; }
            u64 nu = n, mu = m;
            scan2(s, nu, mu);
            if (t == 0) s.found[0] = BINS;
            __syncthreads();
            u64 na = n_before + nu - n, ma = m_before + mu - m;
            if (n && reached(na + n, ma + m) && !(nu > n && reached(na, ma))) {
                int b = t * PER;
                while (!(s.cnt[k][b] && reached(na + s.cnt[k][b], ma + s.mass[k][b]))) {
                    na += s.cnt[k][b];
                    ma += s.mass[k][b];
                    b++;
                }
                s.found[0] = (u64)b;
                s.found[1] = na;
                s.found[2] = ma;
                s.found[3] = s.cnt[k][b];
            }
            __syncthreads();
            const int b = (int)s.found[0];
            if (b < BINS) { n_before = s.found[1]; m_before = s.found[2]; n_bin = s.found[3]; }
            __syncthreads();
            return b;
        };
        // the cut's key: the first histogram's bin, then finer ones over the keys inside
        auto descend = [&](auto reached) {
            n_before = m_before = 0;
            const int b0 = find(0, reached);
            if (b0 == BINS) return 0u;
            if (t == 0) { s.kmin = 0xFFFFFFFFu; s.kmax = 0; }
            __syncthreads();
            each([&](const float* v, int) {
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (valid(v[e]) && bin_of(dist(v[e])) == b0) {
                        atomicMin(&s.kmin, key_of(v[e]));
                        atomicMax(&s.kmax, key_of(v[e]));
                    }
            });
            __syncthreads();
            unsigned lo = s.kmin, hi = s.kmax;
            __syncthreads();
            while (lo < hi) {
                int shift = 0;
                while (((hi - lo) >> shift) >= BINS) shift++;
                clear(1);
                each([&](const float* v, int) {
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        const unsigned k = key_of(v[e]);
                        if (!valid(v[e]) || k < lo || k > hi) continue;
                        const int b = (int)((hi - k) >> shift);
                        atomicAdd(&s.cnt[1][b], 1u);
                        const u64 w = fixed(weight(dist(v[e])));
                        if (w) atomicAdd(&s.mass[1][b], w);
                    }
                });
                __syncthreads();
                const int b = find(1, reached);
                hi -= (unsigned)b << shift;
                const unsigned width = 1u << shift;
                lo = hi - lo >= width ? hi - width + 1 : lo;
            }
            return hi;
        };
        u64 r = 0;
        double p_of = -1.0;    // the sum that top-p takes its share of: of the words that top-k left
        if (by_k) {
            tau = descend([&](u64 n, u64) { return n >= (u64)top_k; });
            if (tau) {
                r = (u64)top_k - n_before;
                const float v = __uint_as_float(tau & 0x80000000u ? tau ^ 0x80000000u : ~tau);
                p_of = (double)(m_before + r * fixed(weight(dist(v))));
            }
        }
        if (by_p) {
            if (p_of < 0.0) {
                u64 n = 0, m = 0;
                for (int b = t; b < BINS; b += ST) { n += s.cnt[0][b]; m += s.mass[0][b]; }
                scan2(s, n, m);
                if (t == ST - 1) s.found[0] = m;
                __syncthreads();
                p_of = (double)s.found[0];
                __syncthreads();
            }
            const double share = (double)top_p * p_of;
            const unsigned at = descend([&](u64, u64 m) { return (double)m >= share; });
            if (at) {
                const float v = __uint_as_float(at & 0x80000000u ? at ^ 0x80000000u : ~at);
                const u64 w = fixed(weight(dist(v)));
                const double left = share - (double)m_before;   // words equal to it are kept while the sum before is below
                u64 rp = w && left > 0.0 ? (u64)ceil(left / (double)w) : 1;
                if (rp < 1) rp = 1;
                if (rp > n_bin) rp = n_bin;
                if (!(tau == at && r < rp)) r = rp;
                tau = at;
            }
        }
        if (tau && r < n_bin) cut = (unsigned)locate([&](float v, int) { return (u64)(valid(v) && key_of(v) == tau); }, [&](u64) { return r - 1; });
    }
    // ---- the pick ----
    const double lim = min_p > 0.0f ? fmax(0.0, -log2((double)min_p)) : INFINITY;
    auto kept = [&](float v, int i) -> u64 {
        if (!valid(v)) return 0;
        const unsigned k = key_of(v);
        if (k < tau || (k == tau && (unsigned)i > cut)) return 0;
        const double d = dist(v);
        return d <= lim ? fixed(weight(d)) : 0;
    };
    const double u = a.u[row];
    u64 sum = 0;
    const int pick = locate(kept, [&](u64 total) {
        sum = total;
        const double at = u > 0.0 ? u * (double)total : 0.0;
        return at < (double)(total - 1) ? (u64)at : total - 1;
    });
    if (t == 0) {
        a.ids[row] = pick;
        if (a.chance) a.chance[row] = (float)((double)weight(dist((float)x[pick])) * 17592186044416.0 / (double)sum);
    }
}

template <class T> hipError_t run(const sample_args& a, hipStream_t s) {
    const hipError_t e = hipFuncSetAttribute((const void*)k_sample<T>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(row_shared));
    if (e != hipSuccess) return e;
    k_sample<T><<<a.rows, ST, sizeof(row_shared), s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_sample(const sample_args& a, hipStream_t s) {
    return a.type == TY_F32 ? run<float>(a, s) : a.type == TY_F16 ? run<_Float16>(a, s) : run<__bf16>(a, s);
}

}  // namespace sh
