// One word for each row of scores: temperature, top-k, top-p, min-p and a given random number (include/seoul_hip.h:
// sh_sample).
//
// With w(x) = e^((x - max) / temp) the kept words are, in the order (score descending, index ascending), a beginning cut
// by count (top-k) or by weight (top-p), of which min-p leaves those above a score: all of them the words above one score
// t, some of the words equal to t (the first r by index), above another. So nothing is sorted. A histogram over the
// weights' exponent (-log2 w in 64ths of a power of two, 4096 bins in LDS) tells the bin that holds the cut; its words,
// a few dozen, are listed and each counts those before it. The pick is a search for the running sum in index order,
// first over the sums of blocks of 64 lanes' words, then within one.
// Weights are summed as integers, in 2^-44ths of the largest, in histograms and blocks alike: sums do not depend on the
// order of the atomics, a block's is exactly its words', and a row's word is the same every time. (Blocks summed in single
// precision, as before, lost words of 2^-24 of a block; the integers cost 3 to 4 us of the figures below.)
//
// A workgroup holds a row in registers: it is read from memory once (256 rows of 97496 fp32 scores: 20 us at 5 TB/s), and
// every pass over it after that costs instructions, which bound it: 256 such rows take 22 us at temperature 0, 31 with
// top-k 50, 35 with no filter, 55 to 65 with top-p 0.9, 62 mixed; one row 21. Up to 32768 32-bit words 1024 threads hold 32
// each (61 rows of 32003 bf16 scores 19 us with top-p; 71 where each pass read them again). Up to 98304 words 512 threads
// hold 192 each, as many as the registers leave: 1024 threads would have 128 registers a thread and spill. Above, and for
// the rare rows that need it (+inf among the scores, more than 4096 words listed by top-k or 512 in the cut's bin, scores
// further apart than 2^64 in weight at the cut), every step reads the row again, which the caches hold by then
// (sample_again; top-k 5000 of 97496: 265 us for 256 rows).
#include <hip/hip_runtime.h>

#include "sh_device.h"
#include "sh_serve.h"

namespace sh {
namespace {

constexpr int BINS = 4096;                // 64 to a power of two
constexpr int MAX_BLOCKS = SAMPLE_MAX_VOCAB / 256;   // blocks of a wave's neighbouring words (64 lanes of 4 or 8)
constexpr int HELD_WORDS = 98304;          // 32-bit words of a row that a workgroup holds at most

typedef unsigned long long u64;

// scores as numbers that sort like them
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);   // (-0 as 0)
    return b ^ ((int)b < 0 ? 0xFFFFFFFFu : 0x80000000u);
}

// 2^-d, d in double: its rounding to single and the rest apart (without the rest the result would be off by d 2^-25)
__device__ __forceinline__ float weight_of(double d) {
    const float hi = (float)d, lo = (float)(d - (double)hi), w = __builtin_amdgcn_exp2f(-hi);
    return hi < 126.0f ? w - w * (lo * 0.69314718f) : 0.0f;
}
// the score of a key
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
// a weight (at most 1, or a rounding above) in 2^-44ths
__device__ __forceinline__ u64 fixed(float w) {
    const float h = w * 4096.0f;
    return ((u64)(unsigned)h << 32) | (unsigned)(__builtin_amdgcn_fractf(h) * 4294967296.0f);
}
// the same as two numbers of 22 bits whose sums over a block (512 words at most) fit 32: a word's cost no carries
struct halves {
    unsigned hi = 0, lo = 0;
    __device__ __forceinline__ void add(float w) {
        const float h = w * 4194304.0f;
        hi += (unsigned)h;
        lo += (unsigned)(__builtin_amdgcn_fractf(h) * 4194304.0f);
    }
    __device__ __forceinline__ u64 sum() const { return ((u64)hi << 22) + lo; }
};
// of n equal words of weight w each, those before which the sum is still below `left`: one at least
__device__ __forceinline__ u64 words_left(double left, u64 w, u64 n) {
    const u64 r = w && left > 0.0 ? (u64)ceil(left / (double)w) : 1;
    return r < 1 ? 1 : r > n ? n : r;
}
// u times the sum as the running sum that has to be passed, the last word's at most
__device__ __forceinline__ u64 target(double u, u64 total) {
    const double at = u > 0.0 ? u * (double)total : 0.0;
    return at < (double)(total - 1) ? (u64)at : total - 1;
}

template <class T> struct score;
template <> struct score<float> {
    static constexpr int V = 4;
    static constexpr unsigned NONE = 0xFF800000u;   // 32 bits of -inf
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
template <> struct score<_Float16> : score16<_Float16> { static constexpr unsigned NONE = 0xFC00FC00u; };
template <> struct score<__bf16> : score16<__bf16> { static constexpr unsigned NONE = 0xFF80FF80u; };

constexpr int LIST = 4096;                 // words at and above a top-k cut that are listed
constexpr int NEAR = 512;                  // words of the bin at a cut that are ordered one by one

struct word {
    float x;
    int i;
    u64 m;                     // its weight
};

constexpr int MAX_WAVES = 16;
struct row_shared {
    unsigned cnt[BINS];        // words per bin of their weights' exponent
    u64 mass[BINS];            // and their weights
    union {
        struct {               // a row that is held
            u64 blocks[HELD_WORDS / 256];   // sums of blocks of neighbouring words
            float list_x[LIST];
            int list_i[LIST];
            word near[NEAR];
        };
        struct {               // a row that is read again
            u64 all_blocks[MAX_BLOCKS];
            unsigned fine_cnt[BINS];   // bins of the keys inside a bin
            u64 fine_mass[BINS];
        };
    };
    // what the threads tell each other, in two buffers taken in turn: who writes one has passed a barrier since it was read
    u64 wsum[2][2][MAX_WAVES];
    u64 found[2][4];
    float wmax[MAX_WAVES];
    unsigned kmin, kmax, n_list, n_near;
    int first;
};

// one step of a scan over a wave: `from` lanes over, 0 where there is none (row_shr, then row_bcast 15 and 31)
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned moved(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ u64 moved(u64 v) {
    return ((u64)moved<CTRL, ROWS>((unsigned)(v >> 32)) << 32) | moved<CTRL, ROWS>((unsigned)v);
}
template <int CTRL, int ROWS> __device__ __forceinline__ double moved(double v) {
    return __longlong_as_double((long long)moved<CTRL, ROWS>((u64)__double_as_longlong(v)));
}
template <int CTRL, int ROWS> __device__ __forceinline__ float moved(float v) { return __uint_as_float(moved<CTRL, ROWS>(__float_as_uint(v))); }
// inclusive sums over the lanes of a wave; lane 63 has the whole
template <class N> __device__ __forceinline__ N wave_scan(N v) {
    v += moved<0x111, 0xF>(v);
    v += moved<0x112, 0xF>(v);
    v += moved<0x114, 0xF>(v);
    v += moved<0x118, 0xF>(v);
    v += moved<0x142, 0xA>(v);
    v += moved<0x143, 0xC>(v);
    return v;
}

__device__ __forceinline__ u64 lane_of(u64 v, int lane) {   // (lane: the same in the whole wave)
    return ((u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}
// inclusive sums over the workgroup of two numbers per thread, and the whole sums
template <int ST> __device__ __forceinline__ void scan2(u64 (&wsum)[2][MAX_WAVES], u64& a, u64& b, u64& all_a, u64& all_b) {
    constexpr int SW = ST / 64;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    a = wave_scan(a);
    b = wave_scan(b);
    if (lane == 63) { wsum[0][wv] = a; wsum[1][wv] = b; }
    __syncthreads();
    // (every wave adds up the waves' sums itself, one a lane)
    const u64 x = wave_scan(lane < SW ? wsum[0][lane] : 0), y = wave_scan(lane < SW ? wsum[1][lane] : 0);
    all_a = lane_of(x, SW - 1);
    all_b = lane_of(y, SW - 1);
    if (wv) { a += lane_of(x, wv - 1); b += lane_of(y, wv - 1); }
}

// What one row needs of its filters
struct row_filter {
    int top_k;                 // 0: all
    float top_p, min_p;        // 1 and 0: all
    double u;
};

// The bins and sums of one row: searches that every path shares (ST threads)
template <int ST> struct row_search {
    row_shared& s;
    u64 n_before = 0, m_before = 0, n_bin = 0;   // words and weights before the bin that was found, words in it
    u64 m_all = 0;                               // all weights of the histogram that was searched
    int turn = 0;                                // the buffer in use

    __device__ __forceinline__ void clear(unsigned* cnt, u64* mass) {
        for (int b = threadIdx.x; b < BINS; b += ST) { cnt[b] = 0; mass[b] = 0; }
        __syncthreads();
    }
    // the first bin that holds something and at which reached(words, weights, all weights) holds for the sums up to it;
    // BINS if none. Presence is a word or, where only weights were summed, a weight
    template <class F> __device__ __forceinline__ int find(const unsigned* cnt, const u64* mass, bool words, F reached) {
        constexpr int PER = BINS / ST;
        const int t = threadIdx.x;
        u64 c[PER], g[PER], n = 0, m = 0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            g[j] = mass[t * PER + j];
            c[j] = words ? cnt[t * PER + j] : (g[j] != 0);
            n += c[j];
            m += g[j];
        }
        u64 nu = n, mu = m, all_n, all_m;
        u64 (&found)[4] = s.found[turn];
        if (t == 0) found[0] = BINS;
        scan2<ST>(s.wsum[turn], nu, mu, all_n, all_m);
        turn ^= 1;
        all_m += m_before;
        u64 na = n_before + nu - n, ma = m_before + mu - m;
        bool past = nu > n && reached(na, ma, all_m);   // (before this thread's bins)
#pragma unroll
        for (int j = 0; j < PER; j++) {
            if (!past && c[j] && reached(na + c[j], ma + g[j], all_m)) {
                found[0] = (u64)(t * PER + j);
                found[1] = na;
                found[2] = ma;
                found[3] = c[j];
                past = true;
            }
            na += c[j];
            ma += g[j];
        }
        __syncthreads();
        const int b = (int)found[0];
        if (b < BINS) { n_before = found[1]; m_before = found[2]; n_bin = found[3]; }
        m_all = all_m;
        return b;
    }
    // the key at which `reached` first holds among the words that `inside` accepts (a bin's): finer and finer bins of
    // their keys. each(f) calls f(score) for every word it knows; weight(score) is its weight in 2^-44ths
    template <class E, class I, class W, class F>
    __device__ __forceinline__ unsigned refine(E each, I inside, W weight, F reached) {
        const int t = threadIdx.x;
        if (t == 0) { s.kmin = 0xFFFFFFFFu; s.kmax = 0; }
        __syncthreads();
        each([&](float x) {
            if (!inside(x)) return;
            atomicMin(&s.kmin, key_of(x));
            atomicMax(&s.kmax, key_of(x));
        });
        __syncthreads();
        unsigned lo = s.kmin, hi = s.kmax;
        bool one = lo == hi;
        do {   // (also once where all are equal: it counts them)
            int shift = 0;
            while (((hi - lo) >> shift) >= BINS) shift++;
            clear(s.fine_cnt, s.fine_mass);
            each([&](float x) {
                const unsigned k = key_of(x);
                if (!inside(x) || k < lo || k > hi) return;
                const int b = (int)((hi - k) >> shift);
                atomicAdd(&s.fine_cnt[b], 1u);
                const u64 w = weight(x);
                if (w) atomicAdd(&s.fine_mass[b], w);
            });
            __syncthreads();
            const int b = find(s.fine_cnt, s.fine_mass, true, reached);
            hi -= (unsigned)b << shift;
            const unsigned width = 1u << shift;
            lo = hi - lo >= width ? hi - width + 1 : lo;
            one = lo == hi && shift == 0;
        } while (!one);
        return hi;
    }
    // the first word, in index order, at which the running sum passes target(total): blocks hold the sums of nb blocks of
    // 64 V words, of(lane's V words) -> their kept weights. `sum` gets the total
    template <int V, class L, class W, class G>
    __device__ __forceinline__ int pick(const u64* blocks, int nb, L load, W of, G target_of, u64& sum) {
        const int t = threadIdx.x, lane = t & 63, per = (nb + ST - 1) / ST;
        u64 mine = 0, unused = 0;
        for (int k = 0; k < per; k++)
            if (t * per + k < nb) mine += blocks[t * per + k];
        u64 up = mine, unused2;
        u64 (&found)[4] = s.found[turn];
        scan2<ST>(s.wsum[turn], up, unused, sum, unused2);
        turn ^= 1;
        const u64 target = target_of(sum);
        u64 at = up - mine;
        if (at <= target && target < up) {   // one thread's blocks hold it
            int b = t * per;
            while (at + blocks[b] <= target) at += blocks[b++];
            found[1] = (u64)b;
            found[2] = at;
        }
        __syncthreads();
        if (t < 64) {
            float v[V];
            u64 w[V], own = 0;
            const int w0 = ((int)found[1] * 64 + lane) * V;
            load(w0, v);
#pragma unroll
            for (int e = 0; e < V; e++) own += w[e] = of(v[e], w0 + e);
            u64 before = found[2] + wave_scan(own) - own;
            // The block's sum is its words': one lane holds the target, at a word of some weight. (Unless the row is written to
            // meanwhile: then a word of the block, so that nothing is read outside the row)
            if (lane == 0) found[3] = (u64)w0;
            if (before <= target && target < before + own) {
                int e = 0;
                while (before + w[e] <= target) before += w[e++];
                found[3] = (u64)(w0 + e);
            }
        }
        __syncthreads();
        return (int)found[3];
    }
};

template <class T, int ST> struct row_words {
    static constexpr int V = score<T>::V;
    const T* x;
    int vocab;
    // V neighbouring scores (-inf past the end)
    __device__ __forceinline__ typename score<T>::vec raw(int at) const {
        typename score<T>::vec v;
        if (at + V <= vocab) return *(const typename score<T>::vec*)(x + at);
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = at + e < vocab ? x[at + e] : (T)-INFINITY;
        return v;
    }
    __device__ __forceinline__ void load(int at, float* v) const { score<T>::unpack(raw(at), v); }
    // every word, read from memory, by whole waves: f(V scores, index of the first)
    template <class F> __device__ __forceinline__ void each(F f) const {
        const int lane = threadIdx.x & 63;
        for (int at = threadIdx.x * V; at - lane * V < vocab; at += ST * V) {
            float v[V];
            load(at, v);
            f(v, at);
        }
    }
};

// A row whose words do not fit the registers, holds +inf, or has too many words at its cut to list them: every step reads
// the row again, which the caches hold by then
template <int ST, class T> __device__ __forceinline__ int sample_again(row_shared& s, const row_words<T, ST>& words, float top, double c, const row_filter& q, u64& sum, float& won) {
    constexpr int V = score<T>::V;
    const int lane = threadIdx.x & 63;
    const bool inf = top == INFINITY;
    auto valid = [&](float v) { return inf ? v == top : v > -INFINITY; };
    auto dist = [&](float v) { return v == top ? 0.0 : ((double)top - (double)v) * c; };   // -log2 of the weight
    auto mass = [&](float v) { return fixed(weight_of(dist(v))); };
    auto bin_of = [&](float v) { const double d = dist(v); return d < 64.0 ? (int)(d * (BINS / 64)) : BINS - 1; };
    auto each = [&](auto f) {
        words.each([&](const float* v, int) {
#pragma unroll
            for (int e = 0; e < V; e++)
                if (valid(v[e])) f(v[e]);
        });
    };
    row_search<ST> w{s};
    unsigned tau = 0, cut = 0xFFFFFFFFu;
    const int nb = (words.vocab + 64 * V - 1) / (64 * V);
    // block sums of f over the words
    auto blocks = [&](auto f) {
        __syncthreads();
        words.each([&](const float* v, int at) {
            u64 t = 0;
#pragma unroll
            for (int e = 0; e < V; e++) t += f(v[e], at + e);
            t = wave_scan(t);
            if (lane == 63) s.all_blocks[at / (64 * V)] = t;
        });
        __syncthreads();
    };
    auto load = [&](int at, float* v) { words.load(at, v); };
    if (q.top_k || q.top_p < 1.0f) {
        __syncthreads();
        w.clear(s.cnt, s.mass);
        each([&](float v) {
            const int b = bin_of(v);
            atomicAdd(&s.cnt[b], 1u);
            const u64 m = mass(v);
            if (m) atomicAdd(&s.mass[b], m);
        });
        __syncthreads();
        u64 r = 0;
        double p_of = -1.0;    // the sum that top-p takes its share of: of the words that top-k left
        auto cut_at = [&](auto reached) {
            w.n_before = w.m_before = 0;
            const int b0 = w.find(s.cnt, s.mass, true, reached);
            return b0 == BINS ? 0u : w.refine(each, [&](float v) { return bin_of(v) == b0; }, mass, reached);
        };
        if (q.top_k) {
            tau = cut_at([&](u64 n, u64, u64) { return n >= (u64)q.top_k; });
            if (tau) {
                r = (u64)q.top_k - w.n_before;
                p_of = (double)(w.m_before + r * mass(of_key(tau)));
            }
        }
        if (q.top_p < 1.0f) {
            if (p_of < 0.0) {
                u64 n = 0, m = 0, all_n, all_m;
                for (int b = threadIdx.x; b < BINS; b += ST) m += s.mass[b];
                scan2<ST>(s.wsum[w.turn], n, m, all_n, all_m);
                w.turn ^= 1;
                p_of = (double)all_m;
            }
            const double share = (double)q.top_p * p_of;
            const unsigned at = cut_at([&](u64, u64 m, u64) { return (double)m >= share; });
            if (at) {
                const u64 rp = words_left(share - (double)w.m_before, mass(of_key(at)), w.n_bin);
                if (!(tau == at && r < rp)) r = rp;
                tau = at;
            }
        }
        if (tau && r < w.n_bin) {
            auto equal = [&](float v, int) -> u64 { return valid(v) && key_of(v) == tau; };
            blocks(equal);
            u64 all;
            cut = (unsigned)w.template pick<V>(s.all_blocks, nb, load, equal, [&](u64) { return r - 1; }, all);
            __syncthreads();
        }
    }
    const double lim = q.min_p > 0.0f ? fmax(0.0, -log2((double)q.min_p)) : INFINITY;
    auto kept = [&](float v, int i) -> u64 {
        if (!valid(v)) return 0;
        const unsigned k = key_of(v);
        if (k < tau || (k == tau && (unsigned)i > cut)) return 0;
        return dist(v) <= lim ? mass(v) : 0;
    };
    blocks(kept);
    const int id = w.template pick<V>(s.all_blocks, nb, load, kept, [&](u64 total) { return target(q.u, total); }, sum);
    won = weight_of(dist((float)words.x[id]));
    return id;
}

// A workgroup holds a row's words in registers, 32 NP words of 32 bits a thread (NP 0: none, the row is read again and
// again). Loops over them index the registers, so that their code stays small: unrolled, a pass over 96 of them is more
// code than the instruction cache holds, and fetching it took longer than running it.
template <class T, int ST, int NP>
__global__ __launch_bounds__(ST) void k_sample(sample_args a) {
    constexpr int V = score<T>::V, SW = ST / 64, SLABS = 8;   // (vectors of a part of 32 registers)
    typedef typename score<T>::vec vec;
    typedef unsigned part_regs __attribute__((ext_vector_type(32)));
    extern __shared__ __align__(16) char lds_raw[];
    row_shared& s = *reinterpret_cast<row_shared*>(lds_raw);
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const row_words<T, ST> words{(const T*)a.scores + (size_t)row * a.ld, a.vocab};
    part_regs held[NP > 0 ? NP : 1];
#pragma unroll
    for (int p = 0; p < NP; p++)
#pragma unroll
        for (int j = 0; j < SLABS; j++) {
            const int k = p * SLABS + j;
            u32x4 v = {score<T>::NONE, score<T>::NONE, score<T>::NONE, score<T>::NONE};
            if (k * ST * V < a.vocab) v = __builtin_bit_cast(u32x4, words.raw((k * ST + t) * V));
#pragma unroll
            for (int e = 0; e < 4; e++) held[p][4 * j + e] = v[e];
        }
    const float temp = a.temp ? a.temp[row] : 1.0f;
    row_filter q{a.top_k ? a.top_k[row] : 0, a.top_p ? a.top_p[row] : 1.0f, a.min_p ? a.min_p[row] : 0.0f, a.u[row]};
    if (q.top_k < 0 || q.top_k >= a.vocab) q.top_k = 0;
    if (!(q.top_p < 1.0f)) q.top_p = 1.0f;
    if (q.top_p <= 0.0f) { q.top_k = 1; q.top_p = 1.0f; }   // (one word at least: the first)
    const int slabs = (a.vocab + ST * V - 1) / (ST * V);
    auto each = [&](auto f) {              // f(V scores, index of the first, slab), by whole waves
        if constexpr (NP > 0) {
#pragma unroll
            for (int p = 0; p < NP; p++) {
                const int n = min(slabs - p * SLABS, SLABS);
#pragma nounroll
                for (int j = 0; j < n; j += 2) {   // (two at a time: one's steps fill the other's waits)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int o = 4 * (j + h), k = p * SLABS + j + h;
                        const u32x4 w = {held[p][o], held[p][o + 1], held[p][o + 2], held[p][o + 3]};
                        float v[V];
                        score<T>::unpack(__builtin_bit_cast(vec, w), v);
                        f(v, (k * ST + t) * V, k);
                    }
                }
            }
        } else {
            words.each([&](const float* v, int at) { f(v, at, 0); });
        }
    };
    auto each_at_once = [&](auto f) {      // f(V scores, vector), unrolled: for short passes
#pragma unroll
        for (int k = 0; k < NP * SLABS; k++) {
            if (k >= slabs) break;
            const int p = k / SLABS, o = 4 * (k % SLABS);
            const u32x4 w = {held[p][o], held[p][o + 1], held[p][o + 2], held[p][o + 3]};
            float v[V];
            score<T>::unpack(__builtin_bit_cast(vec, w), v);
            f(v, k);
        }
    };
    // ---- the maximum, and that of each group of vectors ----
    constexpr int GROUPS = NP == 1 ? SLABS : NP;
    float mine = -INFINITY, best[GROUPS > 0 ? GROUPS : 1];
    if constexpr (NP > 0) {
#pragma unroll
        for (int g = 0; g < GROUPS; g++) best[g] = -INFINITY;
        each_at_once([&](const float* v, int k) {   // (each word as it arrives)
#pragma unroll
            for (int e = 0; e < V; e++) best[k * GROUPS / (NP * SLABS)] = fmaxf(best[k * GROUPS / (NP * SLABS)], v[e]);   // (NaN is passed over)
        });
#pragma unroll
        for (int g = 0; g < GROUPS; g++) mine = fmaxf(mine, best[g]);
    } else {
        each([&](const float* v, int, int) {
#pragma unroll
            for (int e = 0; e < V; e++) mine = fmaxf(mine, v[e]);
        });
    }
    float top = wave_max(mine);
    if (lane == 0) s.wmax[wv] = top;
    if (t == 0) { s.first = 0x7FFFFFFF; s.n_list = s.n_near = 0; }
    for (int b = t; b < BINS; b += ST) { s.cnt[b] = 0; s.mass[b] = 0; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SW; w++) top = fmaxf(top, s.wmax[w]);
    const bool none = top == -INFINITY || !(temp >= 0.0f);
    if (none || temp == 0.0f) {
        if (!none) {
            if (mine == top) {
                int first = 0x7FFFFFFF;
                each([&](const float* v, int at, int) {
#pragma unroll
                    for (int e = V - 1; e >= 0; e--)
                        if (v[e] == top) first = min(first, at + e);
                });
                atomicMin(&s.first, first);
            }
            __syncthreads();
        }
        if (t == 0) {
            a.ids[row] = none ? -1 : s.first;
            if (a.chance) a.chance[row] = none ? 0.0f : 1.0f;
        }
        return;
    }
    const double c = 1.4426950408889634 / (double)temp;
    u64 sum = 0;
    int id = -1;
    float won = 0.0f;
    bool again = NP == 0 || top == INFINITY || !(c < 1e30) || !(c > 1e-30);
    if constexpr (NP > 0) {
        if (!again) {
            // weights 2^-far(x), far = (top - x) c with c in two parts: its rounding alone would move them by up to 1e-6. It
            // grows as x falls, step by step of x: d ch grows by more than the rounding of d cl takes. Beyond 2^-64, and
            // for -inf and NaN, it stays there: such words have no weight in 2^-44ths
            const float ch = (float)c, cl = (float)(c - (double)ch), least = -3.402823466e38f;
            auto far = [&](float x) { const float d = top - x; return fminf(fmaf(d, ch, d * cl), 63.99f); };
            auto weight = [&](float x) { return __builtin_amdgcn_exp2f(-far(x)); };
            auto mass = [&](float x) { return fixed(weight(x)); };
            auto bin_of = [&](float x) { return (int)(far(x) * (float)(BINS / 64)); };
            // a score below all of bin b, by a little more than roundings
            auto below = [&](int b) { return b >= BINS - 1 ? least : top - (float)(b + 1) / (ch * (float)(BINS / 64)) * 1.00001f - fabsf(top) * 1e-6f; };
            row_search<ST> w{s};
            float tau = least;             // kept: above, or equal with an index up to cut
            int cut = 0x7FFFFFFF;
            if (q.min_p > 0.0f) {          // the lowest score whose weight is at least min_p
                const double lim = fmax(0.0, -log2((double)q.min_p));
                auto enough = [&](float x) { return x <= top && ((double)top - (double)x) * c <= lim; };
                float x = (float)fmax((double)top - lim / c, (double)least);
                while (!enough(x)) x = nextafterf(x, INFINITY);
                while (x > least && enough(nextafterf(x, -INFINITY))) x = nextafterf(x, -INFINITY);
                tau = x;
            }
            const float low = tau;
            bool by_k = q.top_k > 0;
            const bool by_p = q.top_p < 1.0f;
            double share = 0.0;
            int b0 = -1;                   // the bin at the cut: none
            const int nb = (a.vocab + 64 * V - 1) / (64 * V);
            // A pass marks words; the few that are marked are listed after it, so that the pass itself has no branches
            unsigned marks[V == 4 ? NP : 2 * NP] = {};   // a bit a word
            auto mark = [&](int k, unsigned bits) {
#pragma unroll
                for (int p = 0; p < NP; p++)
                    if (k / SLABS == p) {
                        if (V == 4) marks[p] |= bits << (4 * (k & 7));
                        else if (k & 4) marks[2 * p + 1] |= bits << (8 * (k & 3));
                        else marks[2 * p] |= bits << (8 * (k & 3));
                    }
            };
            auto list_marked = [&](unsigned* count, int room, auto put) {   // put(place, index of the word)
                unsigned n = 0;
#pragma unroll
                for (unsigned m : marks) n += __popc(m);
                const unsigned in = wave_scan(n);
                unsigned k = 0;
                if (lane == 63 && in) k = atomicAdd(count, in);
                k = (unsigned)__builtin_amdgcn_readlane((int)k, 63) + in - n;
#pragma unroll
                for (int p = 0; p < (V == 4 ? NP : 2 * NP); p++)
                    for (unsigned m = marks[p]; m; m &= m - 1, k++) {
                        const int bit = __ffs((int)m) - 1;
                        if (k < (unsigned)room) put(k, ((p * (32 / V) + bit / V) * ST + t) * V + bit % V);
                    }
                __syncthreads();
                again = *count > (unsigned)room;
            };
            auto list_from = [&](float from) {   // all words from a score on
                each_at_once([&](const float* v, int k) {
                    unsigned bits = 0;
#pragma unroll
                    for (int e = 0; e < V; e++) bits |= v[e] >= from ? 1u << e : 0u;
                    mark(k, bits);
                });
                list_marked(&s.n_list, LIST, [&](unsigned k, int i) { s.list_i[k] = i; });
                if (!again)
                    for (int k = t; k < (int)s.n_list; k += ST) s.list_x[k] = (float)words.x[s.list_i[k]];
                __syncthreads();
            };
            if (by_k || by_p) {
                auto by_words = [&](u64 n, u64, u64) { return n >= (u64)q.top_k; };
                bool counted = by_k, from_list = false;
                if (by_k && q.top_k <= ST * GROUPS) {
                    // the largest words of as many groups as top_k: what lies below their bins is not among the first top_k
#pragma unroll
                    for (int g = 0; g < GROUPS; g++)
                        if (best[g] >= least) atomicAdd(&s.cnt[bin_of(best[g])], 1u);
                    __syncthreads();
                    const int b = w.find(s.cnt, s.mass, true, by_words);
                    w.n_before = w.m_before = 0;
                    for (int k = t; k < BINS; k += ST) s.cnt[k] = 0;
                    from_list = b < BINS - 1;
                    if (from_list) list_from(below(b));
                    else __syncthreads();
                }
                if (!again) {
                    if (from_list) {
                        for (int k = t; k < (int)s.n_list; k += ST) {
                            const float x = s.list_x[k];
                            atomicAdd(&s.cnt[bin_of(x)], 1u);
                            if (by_p) atomicAdd(&s.mass[bin_of(x)], mass(x));
                        }
                    } else {               // (-inf and NaN: no word, no weight, in the last bin)
                        if (by_k)
                            each([&](const float* v, int, int) {
#pragma unroll
                                for (int e = 0; e < V; e++) atomicAdd(&s.cnt[bin_of(v[e])], v[e] >= least ? 1u : 0u);
                            });
                        if (by_p)
                            each([&](const float* v, int, int) {
#pragma unroll
                                for (int e = 0; e < V; e++) atomicAdd(&s.mass[bin_of(v[e])], mass(v[e]));
                            });
                    }
                    __syncthreads();
                    if (by_k) {
                        b0 = w.find(s.cnt, s.mass, true, by_words);
                        by_k = b0 < BINS;  // (fewer words than top_k: all of them)
                    }
                    if (!by_k && by_p) {
                        b0 = w.find(s.cnt, s.mass, counted, [&](u64, u64 m, u64 all) { return (double)m >= (double)q.top_p * (double)all; });
                        share = (double)q.top_p * (double)w.m_all;
                    }
                    if (b0 == BINS) b0 = -1;
                    again = b0 == BINS - 1;    // (its words are further apart than a bin is wide)
                    if (!by_k && bin_of(low) < b0) b0 = -1;   // (min-p alone decides)
                }
                if (!again && by_k && !from_list) list_from(below(b0));
            }
            if (!again) {
                if (by_k) {
                    for (int b = t; b < nb; b += ST) s.blocks[b] = 0;
                } else {
                    // the weights above the cut's bin summed up by blocks, the words of the bin listed
                    halves sums;           // lane k: the sum of the wave's words of slab k
                    auto put = [&](halves part, int k) {
                        const unsigned hi = (unsigned)__builtin_amdgcn_readlane((int)wave_scan(part.hi), 63);
                        const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)wave_scan(part.lo), 63);
                        sums.hi = lane == k ? hi : sums.hi;
                        sums.lo = lane == k ? lo : sums.lo;
                    };
                    if (b0 < 0) {
                        each([&](const float* v, int, int k) {
                            halves part;
#pragma unroll
                            for (int e = 0; e < V; e++) part.add(v[e] >= low ? weight(v[e]) : 0.0f);
                            put(part, k);
                        });
                    } else {
                        const float f0 = (float)b0 * (64.0f / BINS), f1 = (float)(b0 + 1) * (64.0f / BINS);   // (exact)
                        each([&](const float* v, int, int k) {
                            halves part;
                            unsigned bits = 0;
#pragma unroll
                            for (int e = 0; e < V; e++) {
                                const float d = top - v[e], f = fmaf(d, ch, d * cl);
                                const bool above = f < f0;
                                part.add(above ? __builtin_amdgcn_exp2f(-f) : 0.0f);
                                bits |= f < f1 && !above ? 1u << e : 0u;
                            }
                            mark(k, bits);
                            put(part, k);
                        });
                    }
                    if (lane * SW + wv < nb) s.blocks[lane * SW + wv] = sums.sum();
                    if (b0 >= 0) {
                        list_marked(&s.n_near, NEAR, [&](unsigned k, int i) { s.near[k].i = i; });
                        if (!again)
                            for (int k = t; k < (int)s.n_near; k += ST) {
                                const float x = (float)words.x[s.near[k].i];
                                s.near[k].x = x;
                                s.near[k].m = mass(x);
                            }
                        __syncthreads();
                    }
                }
            }
            // the words of bin b among those listed
            auto near_of = [&](int b) {
                for (int k = t; k < (int)s.n_list; k += ST) {
                    const float x = s.list_x[k];
                    if (bin_of(x) != b) continue;
                    const unsigned j = atomicAdd(&s.n_near, 1u);
                    if (j < NEAR) s.near[j] = word{x, s.list_i[k], mass(x)};
                }
                __syncthreads();
                again = s.n_near > NEAR;
            };
            // the words of the bin in their order: the last one kept is the one that last(words before it, weights before it,
            // its own weight) accepts. As many threads share a word's comparisons as there are
            u64 to_cut = 0;
            auto order = [&](auto last) {
                const int n = (int)s.n_near;
                int share_log = 4;
                while (share_log && (n << share_log) > ST) share_log--;
                const int per = 1 << share_log, k = t >> share_log;
                u64 (&found)[4] = s.found[w.turn];
                w.turn ^= 1;
                if (k < n) {
                    const word me = s.near[k];
                    u64 mb = 0;
                    unsigned nb = 0, after = 0;
                    for (int j = t & (per - 1); j < n; j += per) {
                        const word o = s.near[j];
                        const bool same = o.x == me.x, first = o.x > me.x || (same && o.i < me.i);
                        nb += first ? 1u : 0u;
                        mb += first ? o.m : 0u;
                        after |= same && o.i > me.i;
                    }
                    for (int o = 1; o < per; o <<= 1) {
                        nb += __shfl_xor(nb, o);
                        mb += __shfl_xor(mb, o);
                        after |= __shfl_xor(after, o);
                    }
                    nb += (unsigned)w.n_before;
                    mb += w.m_before;
                    if ((t & (per - 1)) == 0 && last((u64)nb, mb, me.m)) {
                        found[0] = __float_as_uint(me.x);
                        found[1] = after ? (u64)me.i : 0x7FFFFFFFu;   // (no equal word behind it: none to leave out)
                        found[2] = mb + me.m;
                    }
                }
                __syncthreads();
                const float x = __uint_as_float((unsigned)found[0]);
                cut = (int)found[1];
                to_cut = found[2];
                if (x >= low) tau = x;
                else { tau = low; cut = 0x7FFFFFFF; }
            };
            if (!again && by_k) {
                near_of(b0);
                if (!again) {
                    order([&](u64 n, u64, u64) { return n == (u64)q.top_k - 1; });
                    if (by_p) {            // the share of what top-k left, by the same histogram
                        share = (double)q.top_p * (double)to_cut;
                        w.n_before = w.m_before = 0;
                        const int b1 = w.find(s.cnt, s.mass, true, [&](u64, u64 m, u64) { return (double)m >= share; });
                        if (b1 != b0) {
                            if (t == 0) s.n_near = 0;
                            __syncthreads();
                            near_of(b1);
                        }
                    }
                }
            }
            if (!again && by_p && b0 >= 0) order([&](u64, u64 m, u64 own) { return (double)m < share && (double)(m + own) >= share; });
            if (!again) {
                auto kept = [&](float x, int i) { return x > tau || (x == tau && i <= cut); };
                if (by_k) {
                    for (int k = t; k < (int)s.n_list; k += ST)
                        if (kept(s.list_x[k], s.list_i[k])) atomicAdd(&s.blocks[s.list_i[k] / (64 * V)], mass(s.list_x[k]));
                } else if (b0 >= 0) {
                    for (int k = t; k < (int)s.n_near; k += ST)
                        if (kept(s.near[k].x, s.near[k].i)) atomicAdd(&s.blocks[s.near[k].i / (64 * V)], s.near[k].m);
                }
                __syncthreads();
                id = w.template pick<V>(s.blocks, nb, [&](int at, float* v) { words.load(at, v); },
                                        [&](float x, int i) -> u64 { return kept(x, i) ? mass(x) : 0; },
                                        [&](u64 total) { return target(q.u, total); }, sum);
                won = weight_of(((double)top - (double)(float)words.x[id]) * c);
            }
        }
    }
    if (again) id = sample_again<ST, T>(s, words, top, c, q, sum, won);
    if (t == 0) {
        a.ids[row] = id;
        if (a.chance) a.chance[row] = (float)((double)won * 17592186044416.0 / (double)sum);
    }
}

template <class T, int ST, int NP> hipError_t run_held(const sample_args& a, hipStream_t s) {
    const hipError_t e = hipFuncSetAttribute((const void*)k_sample<T, ST, NP>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(row_shared));
    if (e != hipSuccess) return e;
    k_sample<T, ST, NP><<<a.rows, ST, sizeof(row_shared), s>>>(a);
    return hipGetLastError();
}
template <class T> hipError_t run(const sample_args& a, hipStream_t s) {
    const int per = 4 / sizeof(T), words = (a.vocab + per - 1) / per;
    return words <= 1024 * 32 ? run_held<T, 1024, 1>(a, s) : words <= HELD_WORDS ? run_held<T, 512, 6>(a, s) : run_held<T, 1024, 0>(a, s);
}

__global__ void k_take(int n, const int32_t* ids, const int32_t* fallback, int32_t* token, int32_t* out, int ld) {
    const int m = threadIdx.x;
    if (m >= n) return;
    const int id = ids[m] < 0 ? fallback[m] : ids[m];
    token[m] = id;
    out[(size_t)m * ld] = id;
}

}  // namespace

hipError_t launch_take(int n, const int32_t* ids, const int32_t* fallback, int32_t* token, int32_t* out, int ld, hipStream_t s) {
    k_take<<<1, 64, 0, s>>>(n, ids, fallback, token, out, ld);
    return hipGetLastError();
}

hipError_t launch_sample(const sample_args& a, hipStream_t s) {
    return a.type == TY_F32 ? run<float>(a, s) : a.type == TY_F16 ? run<_Float16>(a, s) : run<__bf16>(a, s);
}

}  // namespace sh
