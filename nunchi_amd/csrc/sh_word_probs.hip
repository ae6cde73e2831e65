// Log probabilities of given words, entropy and the likeliest words of rows of scores (include/seoul_hip.h: sh_word_probs).
//
// With z = (x - max) / temp, L = sum e^z and S = sum e^z z a word's log probability is z - log L and the entropy log L - S / L.
// A row is cut into parts that workgroups of their own read once (k_probs_part): each keeps its part in registers, and sums
// relative to its own largest score, of which two parts' join as in a running softmax (k_probs_join). The largest score's own
// weight, 1, is counted apart from the others' sum (the rest): log L = log1p(rest) keeps its digits where one word has nearly
// everything, and the entropy is a sum of two numbers that are not negative.
// The likeliest words of a part: with the scores in groups, the n-th largest of the groups' largest scores is no larger than the
// n-th largest score, so the few dozen scores from there up hold them all; these are ordered by counting, for each, those before
// it. No histogram, no sort. A word's place in the order is one 64-bit key: its score as a number that sorts like it, and its
// index turned round.
//
// What bounds it: many rows, memory (256 rows of 97496 fp32 scores, 100 MB: 23.3 us for the parts, 4.3 TB/s of 5.0, and 4.8 for the join; a
// call 27.2. In 16 bits, 50 MB, a call takes 25: as many words, each with its exponential); few rows, the two launches that wait for each
// other (one such row 6.0 and 3.5 us of kernels, 11.4 a call).
#include <hip/hip_runtime.h>

#include <climits>

#include "sh_device.h"
#include "sh_serve.h"

namespace sh {
namespace {

constexpr int PT = 256;                    // threads of a part
constexpr int LISTED = 1024;               // words of a part that may be listed
constexpr int GROUPS = 256, PAST = 4;      // groups of words; how many more than asked for a cut may leave
// keys that a row's parts may have, and those of them that a cut of their groups can leave at most
constexpr int JOINED = SAMPLE_MAX_VOCAB / (32 * PT) * PROBS_MAX_TOP, LEFT = ((PROBS_MAX_TOP + PAST) * (JOINED / GROUPS) + 63) / 64 * 64;

template <class T> struct score_vec {
    static constexpr int V = 8;
    typedef T vec __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct score_vec<float> {
    static constexpr int V = 4;
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
};

typedef unsigned long long u64;

// scores as numbers that sort like them (-0 as 0); above NONE: a score that is more than -inf
__device__ __forceinline__ unsigned order_of(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return b ^ ((int)b < 0 ? 0xFFFFFFFFu : 0x80000000u);
}
constexpr unsigned NONE = 0x007FFFFFu;     // order_of(-inf)
__device__ __forceinline__ float of_order(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ u64 key_of(float x, int i) { return (u64)order_of(x) << 32 | (unsigned)~i; }

template <int CTRL, class V> __device__ __forceinline__ V by_dpp(V v) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
template <class V> __device__ __forceinline__ V of_lane(V v, int lane) {
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
// the same value in every lane (the wave fully active): within each 16 lanes by DPP, then the four of them
template <class V> __device__ __forceinline__ V wave_all(V v, V (*f)(V, V)) {
    v = f(v, by_dpp<DPP_XOR1>(v));
    v = f(v, by_dpp<DPP_XOR2>(v));
    v = f(v, by_dpp<DPP_MIRROR8>(v));
    v = f(v, by_dpp<DPP_MIRROR16>(v));
    return f(f(of_lane(v, 0), of_lane(v, 16)), f(of_lane(v, 32), of_lane(v, 48)));
}
__device__ __forceinline__ int add_i(int x, int y) { return x + y; }
__device__ __forceinline__ float add_f(float x, float y) { return x + y; }
__device__ __forceinline__ float most_f(float x, float y) { return fmaxf(x, y); }

// A number that at least n of the wave's keys (N a lane) reach, and at most a few more than n: the n-th largest bit by bit, until
// that is so.
template <class K, int N> __device__ __forceinline__ K reached_by(const K (&key)[N], int n) {
    K at = 0;
#pragma unroll 1
    for (K bit = (K)1 << (8 * sizeof(K) - 1); bit; bit >>= 1) {
        int c = 0;
#pragma unroll
        for (int e = 0; e < N; e++) c += __popcll(__ballot(key[e] >= (at | bit)));
        if (c >= n) at |= bit;
        if (c >= n && c <= n + PAST) break;
    }
    return at;
}

// The want largest of n keys in LDS, in order, to best[0 .. want); 0 behind them. By NT threads: t is one's number among them.
template <int NT> __device__ __forceinline__ void order_keys(const u64* key, int n, int want, u64* best, int t) {
    if (n <= 64) {                         // one a lane of the first wave, told to all lanes one after the other
        if (t < 64) {
            const u64 mine = t < n ? key[t] : 0;
            const int hi = (int)(mine >> 32), lo = (int)(unsigned)mine;
            int before = 0;
            for (int o = 0; o < n; o++) {
                const u64 x = (u64)(unsigned)__builtin_amdgcn_readlane(hi, o) << 32 | (unsigned)__builtin_amdgcn_readlane(lo, o);
                before += x > mine;
            }
            if (t < n && before < want) best[before] = mine;
        }
    } else {
        for (int k = t; k < n; k += NT) {
            const u64 mine = key[k];
            int before = 0;
#pragma unroll 8
            for (int o = 0; o < n; o++) before += key[o] > mine;
            if (before < want) best[before] = mine;
        }
    }
    for (int k = n + t; k < want; k += NT) best[k] = 0;
}

// two parts' sums as one, relative to the larger of their largest (c: powers of two a unit of score)
__device__ __forceinline__ probs_part joined(const probs_part& a, const probs_part& b, float c) {
    const float top = fmaxf(a.top, b.top);
    probs_part r{top, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const probs_part& q = k ? b : a;
        if (q.top == top) {
            r.ties += q.ties;
            r.rest += q.rest;
            r.dist += q.dist;
        } else if (q.top > -INFINITY && top < INFINITY) {
            const float d = fmaxf((q.top - top) * c, -200.0f), f = __builtin_amdgcn_exp2f(d), all = q.ties + q.rest;
            r.rest += all * f;
            r.dist += (q.dist + all * d) * f;
        }
    }
    return r;
}

// log2 e over the temperature, inside the range so that 0 times it is 0 (a row without a temperature above 0 has no sums)
__device__ __forceinline__ float per_score(float temp) { return temp > 0.0f ? fminf(1.44269504f / temp, 3e38f) : 1.0f; }

struct join_shared {
    u64 key[LEFT > LISTED ? LEFT : LISTED], best[PROBS_MAX_TOP];
    float log_sum, top;
};

// A row's parts joined, by NT threads: one wave puts the likeliest words in order, another adds up the sums.
template <class T, int NT> __device__ __forceinline__ void join_row(const probs_args& a, const int row, join_shared& s) {
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const float temp = a.temp ? a.temp[row] : 1.0f;
    const int want = a.n_top > 0 ? a.n_top : 1;
    if (wv == 0) {
        // The keys in groups, four a lane: the want-th largest of the groups' largest, and the few dozen from there up hold them all. (A part's
        // keys are in order, so a group is to take few keys of each part.)
        const u64* best = a.best + (size_t)row * a.parts * want;
        const int all = a.parts * want;
        u64 most[4] = {0, 0, 0, 0};
        for (int k = lane; k < all; k += GROUPS) {
            u64 x[4];
#pragma unroll
            for (int g = 0; g < 4; g++) x[g] = k + 64 * g < all ? best[k + 64 * g] : 0;
#pragma unroll
            for (int g = 0; g < 4; g++) most[g] = max(most[g], x[g]);
        }
        const u64 cut = max(reached_by(most, want), 1ull);
        int n = 0;
#pragma unroll 4
        for (int k = 0; k < all; k += 64) {
            const u64 mine = k + lane < all ? best[k + lane] : 0;
            const u64 who = __ballot(mine >= cut);
            const int at = n + __popcll(who & ((1ull << lane) - 1));
            if (mine >= cut && at < LEFT) s.key[at] = mine;
            n += __popcll(who);
        }
        wave_lds();
        if (n > 128) {                     // (many parts and many words: once more, among the keys themselves)
            u64 mine[LEFT / 64];
#pragma unroll
            for (int e = 0; e < LEFT / 64; e++) mine[e] = 64 * e + lane < n ? s.key[64 * e + lane] : 0;
            const u64 from = reached_by(mine, want);
            wave_lds();
            n = 0;
#pragma unroll
            for (int e = 0; e < LEFT / 64; e++) {
                const u64 who = __ballot(mine[e] >= from);
                if (mine[e] >= from) s.key[n + __popcll(who & ((1ull << lane) - 1))] = mine[e];
                n += __popcll(who);
            }
            wave_lds();
        }
        order_keys<64>(s.key, n, want, s.best, lane);
    } else if (wv == 1) {
        const probs_part* p = a.part + (size_t)row * a.parts;
        const float c = per_score(temp);
        probs_part q{-INFINITY, 0.0f, 0.0f, 0.0f};
        for (int k = lane; k < a.parts; k += 64) q = joined(q, p[k], c);
        const float top = wave_all(q.top, most_f);
        if (q.top < top) {
            const probs_part at_top{top, 0.0f, 0.0f, 0.0f};
            q = joined(q, at_top, c);
        }
        const float ties = wave_all(q.ties, add_f), rest = wave_all(q.rest, add_f), dist = wave_all(q.dist, add_f);
        if (lane == 0) {
            const float log_sum = ties > 1.0f ? logf(ties + rest) : log1pf(rest);
            s.log_sum = log_sum;
            s.top = top;
            if (a.entropy) {
                float h = 0.0f;
                if (temp > 0.0f && top > -INFINITY) h = log_sum - dist * 0.69314718f / (ties + rest);
                else if (!(temp >= 0.0f)) h = NAN;
                a.entropy[row] = h;
            }
        }
    }
    __syncthreads();
    const float top = s.top, log_sum = s.log_sum;
    const int first = (int)~(unsigned)s.best[0];
    auto logp = [&](float x, int i) {
        if (!(temp >= 0.0f)) return (float)NAN;
        if (!(x > -INFINITY)) return -INFINITY;
        if (temp == 0.0f) return i == first ? 0.0f : -INFINITY;
        if (x == top) return -log_sum;
        if (top == INFINITY) return -INFINITY;
        return (x - top) / temp - log_sum;
    };
    for (int k = t; k < a.n_top; k += NT) {
        const u64 b = s.best[k];
        const size_t at = (size_t)row * a.n_top + k;
        if (a.top_words) a.top_words[at] = b ? (int)~(unsigned)b : -1;
        if (a.top_logp) a.top_logp[at] = b ? logp(of_order((unsigned)(b >> 32)), (int)~(unsigned)b) : temp >= 0.0f ? -INFINITY : (float)NAN;
    }
    for (int k = t; k < a.n_words; k += NT) {
        const int w = a.words[(size_t)row * a.n_words + k];
        const float x = w >= 0 && w < a.vocab ? (float)((const T*)a.scores)[(size_t)row * a.ld + w] : -INFINITY;
        a.logp[(size_t)row * a.n_words + k] = logp(x, w);
    }
}

// A part: PT * VPT words of a row, VPT a thread. A row that is one part is finished here.
template <class T, int VPT> __global__ __launch_bounds__(PT) void k_probs_part(probs_args a) {
    typedef score_vec<T> sv;
    constexpr int V = sv::V, N = VPT / V, WAVES = PT / 64;
    __shared__ join_shared js;
    u64* const key_s = js.key;
    __shared__ unsigned lane_s[PT], cut_s;
    __shared__ probs_part part_s[WAVES];
    __shared__ int n_s, count_s[WAVES];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const int first = part * (PT * VPT);
    const T* src = (const T*)a.scores + (size_t)row * a.ld;
    const float c = per_score(a.temp ? a.temp[row] : 1.0f);
    // ---- the part's scores, behind the row's end -inf: all loads before the first is waited for ----
    // (a vector that would pass the end is taken from the row's last words, of which those before its place do not count)
    auto place = [&](int l) { return first + (l * PT + t) * V; };
    auto from = [&](int l) { return max(min(place(l), a.vocab - V), 0); };
    float x[VPT];
    if (a.vocab >= V) {
        typename sv::vec v[N];
#pragma unroll
        for (int l = 0; l < N; l++) v[l] = *(const typename sv::vec*)(src + from(l));
#pragma unroll
        for (int l = 0; l < N; l++)
#pragma unroll
            for (int e = 0; e < V; e++) x[l * V + e] = (float)v[l][e];
    } else {
#pragma unroll
        for (int l = 0; l < N; l++)
#pragma unroll
            for (int e = 0; e < V; e++) x[l * V + e] = (float)src[min(e, a.vocab - 1)];
    }
    if (first + PT * VPT > a.vocab) {
#pragma unroll
        for (int l = 0; l < N; l++)
#pragma unroll
            for (int e = 0; e < V; e++)
                if (from(l) + e < place(l) || from(l) + e >= a.vocab) x[l * V + e] = -INFINITY;
    }
    float mine = -INFINITY;                // (NaN is passed over here and in every comparison below)
#pragma unroll
    for (int e = 0; e < VPT; e++) mine = fmaxf(mine, x[e]);
    lane_s[t] = order_of(mine);
    const float top = wave_all(mine, most_f);
    // ---- sums of the wave relative to its largest ----
    float rest[2] = {0, 0}, dist[2] = {0, 0};
    int ties = 0;
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int e = 0; e < VPT; e++) {
        const bool same = x[e] == ref;
        ties += same;
        // (at -200 a weight is 0; scores at the largest are counted, not summed. +inf less +inf is NaN, which the maximum drops)
        const float z = same ? -200.0f : fmaxf((x[e] - ref) * c, -200.0f);
        const float w = __builtin_amdgcn_exp2f(z);
        rest[e & 1] += w;
        dist[e & 1] = fmaf(w, z, dist[e & 1]);
    }
    ties = wave_all(ties, add_i);
    const float rest_w = wave_all(rest[0] + rest[1], add_f), dist_w = wave_all(dist[0] + dist[1], add_f);
    if (lane == 0) part_s[wv] = probs_part{top, top == -INFINITY ? 0.0f : (float)ties, rest_w, dist_w};
    if (t == 0) n_s = 0;
    __syncthreads();
    // ---- where the likeliest begin: a group is a thread's words ----
    const int want = a.n_top > 0 ? a.n_top : 1;
    if (wv == 0) {
        unsigned k[4];
#pragma unroll
        for (int w = 0; w < WAVES; w++) k[w] = lane_s[64 * w + lane];
        const unsigned cut = reached_by(k, want);
        if (lane == 0) cut_s = max(cut, NONE + 1);
    } else if (t == 64) {
        probs_part p = part_s[0];
        for (int w = 1; w < WAVES; w++) p = joined(p, part_s[w], c);
        a.part[(size_t)row * a.parts + part] = p;
    }
    __syncthreads();
    const float cut = of_order(cut_s);
    auto index = [&](int e) { return from(e / V) + e % V; };
    if (mine >= cut) {
#pragma unroll
        for (int e = 0; e < VPT; e++)
            if (x[e] >= cut) {
                const int at = atomicAdd(&n_s, 1);
                if (at < LISTED) key_s[at] = key_of(x[e], index(e));
            }
    }
    __syncthreads();
    int n = n_s;
    if (n > LISTED) {
        // Rare (many equal scores, or most of the likeliest with few threads): the key of the last word that counts, bit by bit
        // over all words. 64 turns of two barriers: one row of 97496 equal scores 48 us (one of different ones 11), 256 such rows 178 (27)
        u64 at = 0;
#pragma unroll 1
        for (u64 bit = 1ull << 63; bit; bit >>= 1) {
            int k = 0;
#pragma unroll
            for (int e = 0; e < VPT; e++) k += x[e] >= cut && key_of(x[e], index(e)) >= (at | bit);
            k = wave_all(k, add_i);
            __syncthreads();
            if (lane == 0) count_s[wv] = k;
            __syncthreads();
            if (count_s[0] + count_s[1] + count_s[2] + count_s[3] >= want) at |= bit;
        }
        if (t == 0) n_s = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VPT; e++)
            if (x[e] >= cut && key_of(x[e], index(e)) >= at) key_s[atomicAdd(&n_s, 1) & (LISTED - 1)] = key_of(x[e], index(e));
        __syncthreads();
        n = min(n_s, LISTED);
    }
    order_keys<PT>(key_s, n, want, a.best + ((size_t)row * a.parts + part) * want, t);
    if (a.parts == 1) {
        __syncthreads();
        join_row<T, PT>(a, row, js);
    }
}

constexpr int JOIN_T = 128;

template <class T> __global__ __launch_bounds__(JOIN_T) void k_probs_join(probs_args a) {
    __shared__ join_shared s;
    join_row<T, JOIN_T>(a, blockIdx.x, s);
}

template <class T> hipError_t run_probs(const probs_args& a, hipStream_t s) {
    const dim3 grid((unsigned)((long long)a.rows * a.parts));
    if (a.chunk == PT * 8) k_probs_part<T, 8><<<grid, PT, 0, s>>>(a);
    else k_probs_part<T, 32><<<grid, PT, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.parts > 1) k_probs_join<T><<<dim3((unsigned)a.rows), JOIN_T, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

// Parts of 8192 words, 32 a thread: as many as the registers hold, so that a row of up to 8192 words is one part and one launch is all
// (8000 words: 10.2 us, in parts of 2048 12.4). us by parts of 2048 and 8192, rows of f32 scores: 256 of 97496 35 and 26, one with its
// 5 likeliest words 12.3 and 11.9, with 20 14.6 and 12.7, with 64 32.6 and 22.7. 2048 words are one part of 8 a thread.
void word_probs_split(probs_args& a) {
    a.chunk = a.vocab <= 8 * PT ? 8 * PT : 32 * PT;
    a.parts = (a.vocab + a.chunk - 1) / a.chunk;
}

hipError_t launch_word_probs(const probs_args& a, hipStream_t s) {
    return a.type == TY_F32 ? run_probs<float>(a, s) : a.type == TY_F16 ? run_probs<_Float16>(a, s) : run_probs<__bf16>(a, s);
}

}  // namespace sh
