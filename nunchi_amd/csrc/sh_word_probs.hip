// Log probabilities of given words, entropy and the likeliest words of rows of scores (include/seoul_hip.h: sh_word_probs).
//
// With z = (x - max) / temp, L = sum e^z and S = sum e^z z a word's log probability is z - log L and the entropy log L - S / L.
// A row is cut into parts that workgroups of their own read once (k_probs_part): each keeps its part in registers, and sums
// relative to its own largest score, of which two parts' join as in a running softmax (k_probs_join). The largest score's own
// weight, 1, is counted apart from the others' sum (the rest): log L = log1p(rest) keeps its digits where one word has nearly
// everything, and the entropy is a sum of two numbers that are not negative.
// The likeliest words of a part: the n-th largest of its lanes' largest scores is no larger than its n-th largest score, so a few
// dozen scores from there up hold them all; these are ordered by counting, for each, those before it. No histogram, no sort.
#include <hip/hip_runtime.h>

#include <climits>

#include "sh_device.h"
#include "sh_serve.h"

namespace sh {
namespace {

constexpr int PT = 256;                    // threads of a part
constexpr int LISTED = 1024;               // scores that may be listed

template <class T> struct score_vec {
    static constexpr int V = 8;
    typedef T vec __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct score_vec<float> {
    static constexpr int V = 4;
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
};

// scores as numbers that sort like them (-0 as 0)
__device__ __forceinline__ unsigned order_of(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return b ^ ((int)b < 0 ? 0xFFFFFFFFu : 0x80000000u);
}
// whether word a comes before word b among the likeliest
__device__ __forceinline__ bool ahead(float xa, int ia, float xb, int ib) { return xa > xb || (xa == xb && ia < ib); }

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_most(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// the n-th largest of a wave's 64 keys (1 <= n <= 64), bit by bit
__device__ __forceinline__ unsigned nth_of_wave(unsigned key, int n) {
    unsigned at = 0;
#pragma unroll 1
    for (unsigned bit = 0x80000000u; bit; bit >>= 1) {
        const int c = __popcll(__ballot(key >= (at | bit)));
        if (c >= n) at |= bit;
        if (c == n) break;                 // (the keys from here up are the ones)
    }
    return at;
}

struct part_shared {
    float x[LISTED];
    int i[LISTED];
    unsigned cut[PT / 64];
    probs_part part[PT / 64];
    int n, equal[PT / 64];
};

// the parts' sums as one, relative to the largest (each lane the same parts)
__device__ __forceinline__ probs_part joined(const probs_part& a, const probs_part& b, float c) {
    const bool first = a.top >= b.top;
    const probs_part &hi = first ? a : b, &lo = first ? b : a;
    probs_part r = hi;
    if (lo.top == -INFINITY) return r;
    if (lo.top == hi.top) {
        r.ties += lo.ties;
        r.rest += lo.rest;
        r.dist += lo.dist;
        return r;
    }
    if (hi.top == INFINITY) return r;
    const float d = fmaxf((lo.top - hi.top) * c, -1000.0f), f = __builtin_amdgcn_exp2f(d), all = lo.ties + lo.rest;
    r.rest += all * f;
    r.dist += (lo.dist + all * d) * f;
    return r;
}

// A part: `chunk` words of a row. VPT: words a thread
template <class T, int VPT> __global__ __launch_bounds__(PT) void k_probs_part(probs_args a) {
    typedef score_vec<T> sv;
    constexpr int V = sv::V, N = VPT / V;
    __shared__ part_shared s;
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const int first = part * a.chunk;
    const T* src = (const T*)a.scores + (size_t)row * a.ld;
    const float temp = a.temp ? a.temp[row] : 1.0f;
    // ---- the part's scores: words that are none (NaN, past the row) are -inf ----
    float x[VPT];
#pragma unroll
    for (int l = 0; l < N; l++) {
        const int at = first + (l * PT + t) * V;
        if (at + V <= a.vocab) {
            const typename sv::vec v = *(const typename sv::vec*)(src + at);
#pragma unroll
            for (int e = 0; e < V; e++) x[l * V + e] = fmaxf((float)v[e], -INFINITY);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) x[l * V + e] = at + e < a.vocab ? fmaxf((float)src[at + e], -INFINITY) : -INFINITY;
        }
    }
    float mine = x[0];
#pragma unroll
    for (int e = 1; e < VPT; e++) mine = fmaxf(mine, x[e]);
    const float top = wave_most(mine);
    // ---- sums of the wave relative to its largest ----
    // (log2 e over the temperature, held inside the range so that 0 times it is 0; a row without one has no sums)
    const float c = temp > 0.0f ? fminf(1.44269504f / temp, 3e38f) : 1.0f;
    float rest[4] = {0, 0, 0, 0}, dist[4] = {0, 0, 0, 0};
    int ties = 0;
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int e = 0; e < VPT; e++) {
        const bool same = x[e] == ref;
        ties += __popcll(__ballot(same));
        // (at -200 a weight is 0; scores at the largest are counted, not summed. +inf less +inf is NaN, which the maximum drops)
        const float z = same ? -200.0f : fmaxf((x[e] - ref) * c, -200.0f);
        const float w = __builtin_amdgcn_exp2f(z);
        rest[e & 3] += w;
        dist[e & 3] = fmaf(w, z, dist[e & 3]);
    }
    const float rest_w = wave_sum((rest[0] + rest[1]) + (rest[2] + rest[3])), dist_w = wave_sum((dist[0] + dist[1]) + (dist[2] + dist[3]));
    if (lane == 0) s.part[wv] = probs_part{top, top == -INFINITY ? 0.0f : (float)ties, rest_w, dist_w};
    // ---- where the likeliest begin ----
    const int want = a.n_top > 0 ? a.n_top : 1;
    const unsigned none = order_of(-INFINITY);
    const unsigned cut_w = nth_of_wave(order_of(mine), want);
    if (lane == 0) s.cut[wv] = cut_w;
    if (t == 0) s.n = 0;
    __syncthreads();
    if (t == 0) {
        probs_part p = s.part[0];
        for (int w = 1; w < PT / 64; w++) p = joined(p, s.part[w], c);
        a.part[(size_t)row * a.parts + part] = p;
    }
    unsigned cut = none + 1;
#pragma unroll
    for (int w = 0; w < PT / 64; w++) cut = max(cut, s.cut[w]);
    auto index = [&](int e) { return first + ((e / V) * PT + t) * V + e % V; };
    if (order_of(mine) >= cut) {
#pragma unroll
        for (int e = 0; e < VPT; e++)
            if (order_of(x[e]) >= cut) {
                const int at = atomicAdd(&s.n, 1);
                if (at < LISTED) {
                    s.x[at] = x[e];
                    s.i[at] = index(e);
                }
            }
    }
    __syncthreads();
    int n = s.n;
    if (n > LISTED) {
        // Rare (many equal scores, or many words of few lanes): the score of the last word that counts, bit by bit over all
        // words, then the index behind the last of those equal to it
        auto total = [&](auto&& test) {
            int k = 0;
#pragma unroll
            for (int e = 0; e < VPT; e++) k += __popcll(__ballot(test(e)));
            __syncthreads();
            if (lane == 0) s.equal[wv] = k;
            __syncthreads();
            int all = 0;
            for (int w = 0; w < PT / 64; w++) all += s.equal[w];
            return all;
        };
        unsigned at = 0;
#pragma unroll 1
        for (unsigned bit = 0x80000000u; bit; bit >>= 1)
            if (total([&](int e) { return order_of(x[e]) >= (at | bit); }) >= want) at |= bit;
        const int above = total([&](int e) { return order_of(x[e]) > at; });
        int behind = 0;                    // of the equal ones those before this index count
#pragma unroll 1
        for (int bit = 1 << 30; bit; bit >>= 1)
            if (total([&](int e) { return order_of(x[e]) == at && index(e) < (behind | bit); }) <= want - above) behind |= bit;
        if (t == 0) s.n = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VPT; e++)
            if (order_of(x[e]) > at || (order_of(x[e]) == at && index(e) < behind)) {
                const int to = atomicAdd(&s.n, 1);
                if (to < LISTED) {
                    s.x[to] = x[e];
                    s.i[to] = index(e);
                }
            }
        __syncthreads();
        n = min(s.n, LISTED);
    }
    // ---- in their order ----
    word_score* best = a.best + ((size_t)row * a.parts + part) * want;
    for (int k = t; k < n; k += PT) {
        const float xk = s.x[k];
        const int ik = s.i[k];
        int before = 0;
        for (int o = 0; o < n; o++) before += ahead(s.x[o], s.i[o], xk, ik);
        if (before < want) best[before] = word_score{xk, ik};
    }
    for (int k = n + t; k < want; k += PT) best[k] = word_score{-INFINITY, -1};
}

constexpr int JOIN_T = 256;

// A row's parts joined, its words' log probabilities
template <class T> __global__ __launch_bounds__(JOIN_T) void k_probs_join(probs_args a) {
    __shared__ float x_s[LISTED];
    __shared__ int i_s[LISTED];
    __shared__ int n_s;
    __shared__ unsigned cut_s[JOIN_T / 64];
    __shared__ word_score best_s[PROBS_MAX_TOP];
    __shared__ double log_s;
    __shared__ float top_s;
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const float temp = a.temp ? a.temp[row] : 1.0f;
    const int want = a.n_top > 0 ? a.n_top : 1;
    // ---- the sums, by the first wave, in 64 bits ----
    if (wv == 0) {
        const probs_part* p = a.part + (size_t)row * a.parts;
        float top = -INFINITY;
        for (int k = lane; k < a.parts; k += 64) top = fmaxf(top, p[k].top);
        top = wave_most(top);
        double ties = 0.0, rest = 0.0, dist = 0.0;
        if (top > -INFINITY && temp > 0.0f) {
            const float c = fminf(1.44269504f / temp, 3e38f);
            for (int k = lane; k < a.parts; k += 64) {
                const probs_part q = p[k];
                if (q.top == top) {
                    ties += q.ties;
                    if (top < INFINITY) {
                        rest += q.rest;
                        dist += q.dist;
                    }
                } else if (q.top > -INFINITY && top < INFINITY) {
                    const double d = fmax((double)(q.top - top) * c, -1000.0), f = exp2(d), all = (double)q.ties + q.rest;
                    rest += all * f;
                    dist += (q.dist + all * d) * f;
                }
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            ties += __shfl_xor(ties, o);
            rest += __shfl_xor(rest, o);
            dist += __shfl_xor(dist, o);
        }
        if (lane == 0) {
            const double log_sum = ties > 1.0 ? log(ties + rest) : log1p(rest);
            log_s = log_sum;
            top_s = top;
            if (a.entropy) {
                float h = 0.0f;
                if (temp > 0.0f && top > -INFINITY) h = (float)(log_sum - dist * 0.6931471805599453 / (ties + rest));
                else if (!(temp >= 0.0f)) h = NAN;
                a.entropy[row] = h;
            }
        }
    }
    // ---- the likeliest words of all parts: from the largest of the parts' last ones up ----
    const word_score* best = a.best + (size_t)row * a.parts * want;
    unsigned cut = order_of(-INFINITY) + 1;
    for (int k = t; k < a.parts; k += JOIN_T) cut = max(cut, order_of(best[(size_t)k * want + want - 1].x));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) cut = max(cut, (unsigned)__shfl_xor((int)cut, o));
    if (lane == 0) cut_s[wv] = cut;
    if (t == 0) n_s = 0;
    if (t < want) best_s[t] = word_score{-INFINITY, -1};
    __syncthreads();
#pragma unroll
    for (int w = 0; w < JOIN_T / 64; w++) cut = max(cut, cut_s[w]);
    for (int k = t; k < a.parts * want; k += JOIN_T) {
        const word_score b = best[k];
        if (order_of(b.x) >= cut) {
            const int at = atomicAdd(&n_s, 1);
            if (at < LISTED) {
                x_s[at] = b.x;
                i_s[at] = b.i;
            }
        }
    }
    __syncthreads();
    const int listed = n_s;
    if (listed <= LISTED) {
        for (int k = t; k < listed; k += JOIN_T) {
            const float xk = x_s[k];
            const int ik = i_s[k];
            int before = 0;
            for (int o = 0; o < listed; o++) before += ahead(x_s[o], i_s[o], xk, ik);
            if (before < want) best_s[before] = word_score{xk, ik};
        }
    } else {
        // (many parts whose words are equal)
        for (int k = t; k < a.parts * want; k += JOIN_T) {
            const word_score b = best[k];
            if (order_of(b.x) < cut) continue;
            int before = 0;
            for (int o = 0; o < a.parts * want && before < want; o++) before += best[o].i >= 0 && ahead(best[o].x, best[o].i, b.x, b.i);
            if (before < want) best_s[before] = b;
        }
    }
    __syncthreads();
    const float top = top_s;
    const int first = best_s[0].i;
    auto logp = [&](float x, int i) {
        if (!(temp >= 0.0f)) return (float)NAN;
        if (!(x > -INFINITY)) return -INFINITY;
        if (temp == 0.0f) return i == first ? 0.0f : -INFINITY;
        if (top == INFINITY && x < top) return -INFINITY;
        const double z = x == top ? 0.0 : ((double)x - top) / temp;
        return (float)(z - log_s);
    };
    for (int k = t; k < a.n_top; k += JOIN_T) {
        const word_score b = best_s[k];
        if (a.top_words) a.top_words[(size_t)row * a.n_top + k] = b.i;
        if (a.top_logp) a.top_logp[(size_t)row * a.n_top + k] = logp(b.x, b.i);
    }
    for (int k = t; k < a.n_words; k += JOIN_T) {
        const int w = a.words[(size_t)row * a.n_words + k];
        const float x = w >= 0 && w < a.vocab ? (float)((const T*)a.scores)[(size_t)row * a.ld + w] : -INFINITY;
        a.logp[(size_t)row * a.n_words + k] = logp(x, w);
    }
}

template <class T> hipError_t run_probs(const probs_args& a, hipStream_t s) {
    const dim3 grid((unsigned)((long long)a.rows * a.parts));
    if (a.chunk == PT * 8) k_probs_part<T, 8><<<grid, PT, 0, s>>>(a);
    else k_probs_part<T, 32><<<grid, PT, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    k_probs_join<T><<<dim3((unsigned)a.rows), JOIN_T, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

// Parts of 8192 words, or of 2048 where the rows are too few to fill the compute units with those.
void word_probs_split(probs_args& a) {
    a.chunk = (long long)a.rows * ((a.vocab + 8191) / 8192) >= 512 ? 8192 : 2048;
    a.parts = (a.vocab + a.chunk - 1) / a.chunk;
}

hipError_t launch_word_probs(const probs_args& a, hipStream_t s) {
    return a.type == TY_F32 ? run_probs<float>(a, s) : a.type == TY_F16 ? run_probs<_Float16>(a, s) : run_probs<__bf16>(a, s);
}

}  // namespace sh
