// Trees of drafted words: their masks and positions (k_tree_plan), the branch that the picked words agree with (k_tree_take)
// and the pages that are free again after it (k_tree_free), and the branch's keys and values at their places (k_page_keep).
//
// All are bound by latency: 256 requests of 64 words read and write 1 MB (plan), 0.3 MB (take), 16 MB (keep, of up to 15 moved
// words); a kernel with its dependent loads takes 2.6 to 6.4 us, and the calling thread 8 to 10 us for each call that it makes.
#include <hip/hip_runtime.h>

#include <climits>

#include "sh_device.h"
#include "sh_serve.h"

namespace sh {
namespace {

// A request's rows, when its row starts and lengths say the same: its words are all there behind the positions held before.
struct tree_rows {
    int r0, m;
    bool sound;
};
__device__ __forceinline__ tree_rows rows_of(const int32_t* cu, const int32_t* held, const int32_t* len, int i, int rows, int most) {
    const int c0 = cu[i], c1 = cu[i + 1], h = held[i];
    const long long m = (long long)c1 - c0;
    tree_rows t;
    t.sound = c0 >= 0 && c1 <= rows && m >= 0 && m <= most && h >= 0 && h + m == len[i];
    t.r0 = min(max(c0, 0), rows);
    t.m = max(min(c1, rows), t.r0) - t.r0;
    return t;
}

// ---------------------------------------------------------------- masks and positions
// One workgroup a request, one thread a word. Each turn a word takes over the bits of the word it points to and points to where
// that one did, so the words known to be before it double: six turns for 64 words in one chain, eight for 256.
template <int NT> __global__ __launch_bounds__(NT) void k_tree_plan(tree_plan_args a) {
    constexpr int W = NT / 32;
    __shared__ unsigned bits_s[NT][W + 1];
    __shared__ int up_s[NT];
    __shared__ bool bad_s[NT];
    const int i = blockIdx.x, j = threadIdx.x;
    const tree_rows t = rows_of(a.cu, a.held, a.len, i, a.rows, a.max_rows);
    if (!t.sound) {
        for (int r = j; r < t.m; r += NT) {
            for (int w = 0; w < a.words; w++) a.mask[(size_t)(t.r0 + r) * a.words + w] = 0;
            a.pos[t.r0 + r] = -1;
        }
        return;
    }
    int up = -1;
    bool bad = false;
    unsigned bits[W];
#pragma unroll
    for (int w = 0; w < W; w++) bits[w] = w == j >> 5 ? 1u << (j & 31) : 0u;
    if (j < t.m) {
        up = a.parent[t.r0 + j];
        bad = up < -1 || up >= j;          // (no word before it)
        if (bad) up = -1;
    }
    for (;;) {
#pragma unroll
        for (int w = 0; w < W; w++) bits_s[j][w] = bits[w];
        up_s[j] = up;
        bad_s[j] = bad;
        if (!__syncthreads_or(up >= 0)) break;
        if (up >= 0) {
#pragma unroll
            for (int w = 0; w < W; w++) bits[w] |= bits_s[up][w];
            bad |= bad_s[up];
            up = up_s[up];
        }
        __syncthreads();
    }
    if (j >= t.m) return;
    int depth = -1;
#pragma unroll
    for (int w = 0; w < W; w++) {
        depth += __popc(bits[w]);
        if (w < a.words) a.mask[(size_t)(t.r0 + j) * a.words + w] = bad ? 0u : bits[w];
    }
    a.pos[t.r0 + j] = bad ? -1 : (int)min((long long)a.pos0 + a.held[i] + depth, (long long)INT_MAX);
}

// ---------------------------------------------------------------- the branch that is kept
// One wave a request, four words a lane at most. Each turn of the walk asks all words at once whether they are the picked child
// and goes on with the first.
constexpr int PER = TREE_MAX / 64;

__device__ __forceinline__ void take_branch(const tree_take_args& a, const int i, const int lane) {
    const tree_rows t = rows_of(a.cu, a.held, a.len, i, a.rows, a.pos ? INT_MAX : TREE_MAX);
    // Nothing was written for a first row without a position, nor behind it: the plan refused the request, or the row has a parent among
    // the rows, or none that there is
    const bool whole = t.sound && t.m > 0, planned = whole && a.parent[t.r0] == -1 && (!a.pos || a.pos[t.r0] >= 0) && t.m <= TREE_MAX;
    if (!planned) {
        for (int r = lane; r < t.m; r += 64) a.path[t.r0 + r] = -1;
        if (lane == 0) {
            a.count[i] = 0;
            a.next[i] = -1;
            a.len_out[i] = whole ? a.held[i] : a.len[i];
        }
        return;
    }
    int up[PER], word[PER], pick[PER], path[PER];
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int j = 64 * e + lane, r = t.r0 + min(j, t.m - 1);
        up[e] = j < t.m ? a.parent[r] : -1;
        if (up[e] >= j) up[e] = -1;        // (not before it)
        word[e] = a.word[r];
        pick[e] = a.pick[r];
        path[e] = -1;
    }
    int at = 0, count = 0, want;
    for (;;) {
#pragma unroll
        for (int e = 0; e < PER; e++)
            if (count == 64 * e + lane) path[e] = at;
        count++;
        int mine = pick[0];
#pragma unroll
        for (int e = 1; e < PER; e++)
            if (at >> 6 == e) mine = pick[e];
        want = __builtin_amdgcn_readlane(mine, at & 63);
        if (want < 0) break;
        int found = -1;
#pragma unroll
        for (int e = PER - 1; e >= 0; e--) {
            const unsigned long long hit = __ballot(up[e] == at && word[e] == want);
            if (hit) found = 64 * e + __ffsll((long long)hit) - 1;
        }
        if (found < 0) break;
        at = found;
    }
#pragma unroll
    for (int e = 0; e < PER; e++)
        if (64 * e + lane < t.m) a.path[t.r0 + 64 * e + lane] = path[e];
    if (lane == 0) {
        a.count[i] = count;
        a.next[i] = want;
        a.len_out[i] = a.held[i] + count;
    }
}

// Pages behind the new lengths go back to the list of free ones, in the order of the requests. One workgroup.
constexpr int FREE_T = 1024;

__device__ __forceinline__ void free_pages_behind(const tree_take_args& a, long long (&sum_s)[FREE_T / 64]) {
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const int per = (a.n + FREE_T - 1) / FREE_T, i0 = min(a.n, t * per), i1 = min(a.n, i0 + per);
    auto pages = [&](int len) { return (int)min(((long long)max(len, 0) + (1 << a.page_log) - 1) >> a.page_log, (long long)a.cols); };
    long long back = 0;
    for (int i = i0; i < i1; i++) back += max(pages(a.len[i]) - pages(a.len_out[i]), 0);
    long long in = back;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long x = __shfl_up(in, o);
        if (lane >= o) in += x;
    }
    if (lane == 63) sum_s[wv] = in;
    __syncthreads();
    long long before = in - back, all = 0;
    for (int w = 0; w < FREE_T / 64; w++) {
        if (w < wv) before += sum_s[w];
        all += sum_s[w];
    }
    const int taken = min(max(a.taken[0], 0), a.n_free);
    const int left = (int)max(taken - all, 0ll);
    long long to = left + before;
    for (int i = i0; i < i1; i++)
        for (int p = pages(a.len_out[i]), p1 = pages(a.len[i]); p < p1; p++, to++)
            if (to < taken) a.free_pages[to] = a.table[(size_t)i * a.cols + p];
    if (t == 0) a.taken_out[0] = left;
}

__global__ __launch_bounds__(256) void k_tree_take(tree_take_args a) {
    const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i < a.n) take_branch(a, i, threadIdx.x & 63);
}
__global__ __launch_bounds__(FREE_T) void k_tree_free(tree_take_args a) {
    __shared__ long long sum_s[FREE_T / 64];
    free_pages_behind(a, sum_s);
}
// both, for requests so few that one workgroup's waves walk them
__global__ __launch_bounds__(FREE_T) void k_tree_take_free(tree_take_args a) {
    __shared__ long long sum_s[FREE_T / 64];
    for (int i = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); i < a.n; i += FREE_T / 64) take_branch(a, i, threadIdx.x & 63);
    __syncthreads();
    free_pages_behind(a, sum_s);
}

// ---------------------------------------------------------------- keys and values of the branch
// A thread moves 16 bytes of one head of the keys or the values for all the words of a request, eight loads before their
// stores. A word moves towards the front, and the words are in the order of their places: what a later word is read from lies
// behind all places that were written.
template <int D> __global__ __launch_bounds__(256) void k_page_keep(keep_args a) {
    __shared__ size_t from_s[TREE_MAX], to_s[TREE_MAX];
    __shared__ int sum_s[4];
    const int i = blockIdx.x, t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const int c0 = a.cu[i], c1 = a.cu[i + 1], len = a.len[i];
    const long long m = (long long)c1 - c0, base = len - m;
    if (c0 < 0 || c1 > a.rows || m < 1 || m > TREE_MAX || base < 0) return;
    // the places of word t
    bool moves = false;
    size_t from = 0, to = 0;
    if (t < m) {
        const int j = a.path[c0 + t];
        moves = j > t && j < m;
        if (moves) {
            const long long f = base + j, g = base + t;
            const long long fp = f >> a.page_log, gp = g >> a.page_log;
            moves = fp < a.cols;
            if (moves) {
                const int fi = a.table[(size_t)i * a.cols + fp], gi = a.table[(size_t)i * a.cols + gp];
                moves = fi >= 0 && fi < a.n_pages && gi >= 0 && gi < a.n_pages;
                const int pm = (1 << a.page_log) - 1;
                from = (((size_t)fi * a.n_kv << a.page_log) + (f & pm)) * D;
                to = (((size_t)gi * a.n_kv << a.page_log) + (g & pm)) * D;
            }
        }
    }
    const unsigned long long who = __ballot(moves);
    if (lane == 0) sum_s[wv] = __popcll(who);
    __syncthreads();
    int at = __popcll(who & ((1ull << lane) - 1)), count = 0;
    for (int w = 0; w < 4; w++) {
        if (w < wv) at += sum_s[w];
        count += sum_s[w];
    }
    if (moves) {
        from_s[at] = from;
        to_s[at] = to;
    }
    __syncthreads();
    const int c = blockIdx.y * 256 + t, per = a.n_kv * (D / 8);
    if (c >= 2 * per) return;
    const int h = c < per ? c : c - per;
    const size_t off = ((size_t)(h / (D / 8)) << a.page_log) * D + h % (D / 8) * 8;
    unsigned short* x = (unsigned short*)(c < per ? a.keys : a.values) + off;
    for (int b = 0; b < count; b += 8) {
        u32x4 v[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (b + e < count) v[e] = *(const u32x4*)(x + from_s[b + e]);
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (b + e < count) *(u32x4*)(x + to_s[b + e]) = v[e];
    }
}

}  // namespace

// A wave a request where it holds the largest tree, so that a turn waits for no other wave: us by 64 and 256 threads, trees of 64 words,
// 256 requests 8.5 and 8.7, 4096 8.0 and 12.3
hipError_t launch_tree_plan(const tree_plan_args& a, hipStream_t s) {
    if (a.max_rows <= 64) k_tree_plan<64><<<a.n, 64, 0, s>>>(a);
    else k_tree_plan<TREE_MAX><<<a.n, TREE_MAX, 0, s>>>(a);
    return hipGetLastError();
}

// One launch where a wave walks two requests at most: us by one and two launches, requests of up to 64 words: 2 10.6 and 12.7, 32 10.1
// and 12.6, 64 12.1 and 12.5 (of up to 256 words 13.8 and 12.0), 128 20.6 and 12.2
constexpr int FEW = 2 * FREE_T / 64;

hipError_t launch_tree_take(const tree_take_args& a, hipStream_t s) {
    if (a.table && a.n <= FEW) {
        k_tree_take_free<<<1, FREE_T, 0, s>>>(a);
        return hipGetLastError();
    }
    k_tree_take<<<(a.n + 3) / 4, 256, 0, s>>>(a);
    if (a.table) k_tree_free<<<1, FREE_T, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_page_keep(int D, const keep_args& a, hipStream_t s) {
    const dim3 grid((unsigned)a.n, (unsigned)((2ll * a.n_kv * (D / 8) + 255) / 256));
    if (D == 32) k_page_keep<32><<<grid, 256, 0, s>>>(a);
    else if (D == 64) k_page_keep<64><<<grid, 256, 0, s>>>(a);
    else k_page_keep<128><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace sh
