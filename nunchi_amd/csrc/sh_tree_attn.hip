// Attention of a batch whose requests try a tree of drafted words each (sh_tree_attn): every word sees the shared positions, its
// request's own before the tree and the words that it follows. Parts of the keys are taken by workgroups of their own and
// joined after them by sh_page_attn.hip's kernel.
//
// With a column's reference r, its sum l of e^(s - r) and its sums O of e^(s - r) v over the keys that it sees, two waves or parts have
// r' = max(r1, r2), l' = l1 e^(r1 - r') + l2 e^(r2 - r'), O' likewise, and the result is O / l (0 where nothing is seen).
//
// What bounds it (us a call, calls in a row over three inputs in turn): many columns, issue: 64 requests of up to 64 words over 2048
// shared and up to 2048 own positions (8 kv heads of 64, 54 GFLOP) 124 us, 440 TFLOP/s of 1139, of which the exponentials, conversions
// and masks take as long as the products, and 2.1 rounds of workgroups over the compute units; few columns over long keys, memory: 64
// requests x 4 words over the same positions (156 MB) 46.5, 3.4 TB/s of 5.0, and 35.7 where the same input comes again and the last
// cache still has it; one request, the chain of loads in front of the first product (ids, keys, 5 us) and the join of its parts (6 us
// of 27 for 32749 positions); short ones, the launch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "sh_attend.h"

namespace sh {
namespace {

constexpr int MASK_WORDS = TREE_MAX / 32;

template <int D, int NT> struct tree_space {
    static constexpr int PITCH = D + 4;        // (shifts columns by four banks)
    union {
        float o[16 * NT * PITCH];              // a wave's sums
        unsigned short keys[32 * (D + 8)];     // its block of keys (the pitch shifts rows by four banks)
    } wave[4];
    f32x4 m[16 * NT], l[16 * NT];              // the waves' references and sums of weights
    unsigned mask[16 * NT][MASK_WORDS + 1];    // the columns' masks, and a word without bits
    int lo[16 * NT], hi[16 * NT];              // what a column sees (below)
    float top[4][16 * NT];                     // the largest score of each wave's first block
};

// four bits from bit `from` on of a column's mask; what lies before the first word is set
__device__ __forceinline__ unsigned tree_bits(const unsigned* mask, int words, int from) {
    if (from <= -4) return 0xFu;
    if (from < 0) return ((mask[0] << -from) | ((1u << -from) - 1)) & 0xFu;
    const int w = min(from >> 5, words);
    const unsigned long long two = mask[w] | (unsigned long long)mask[min(w + 1, words)] << 32;
    return (unsigned)(two >> (from & 31)) & 0xFu;
}

// the largest of the wave's first 16 lanes
__device__ __forceinline__ int most_of_16(int x) {
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x128, 0xF, 0xF, false));   // row_ror:8, 4, 2, 1
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x124, 0xF, 0xF, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x122, 0xF, 0xF, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x121, 0xF, 0xF, false));
    return __builtin_amdgcn_readfirstlane(x);
}
// the bits of a lane's 16
__device__ __forceinline__ unsigned any_of_16(unsigned x) {
    x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xF, 0xF, false);
    x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xF, 0xF, false);
    x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xF, 0xF, false);
    x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xF, 0xF, false);
    return x;
}
// the largest of four lanes 16 apart
__device__ __forceinline__ float over_quads(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// A request, its row starts and its length, and which of its tiles of columns a workgroup takes.
struct tile_of_request {
    int k, cu0, cu1, len, tile;
};

// Tile `at` of all requests': request k has the tiles first(k) .. first(k + 1) - 1, at least as many as its columns fill. A wave
// looks at 63 requests at a time. (Longest requests first, so that the last workgroups to start are the shortest: no gain.)
__device__ __forceinline__ tile_of_request find_tile(const pattn_args& a, int at, int lane, int nc) {
    auto row_at = [&](int cu) { return min(max(cu, 0), a.rows); };
    auto first = [&](int cu, int k) { return (int)((long long)row_at(cu) * a.grp / nc) + k; };
    int lo = 0, hi = a.n;
    for (;;) {
        const int step = (hi - lo + 62) / 63, k = lo + lane * step;
        const int cu = a.cu[min(k, a.n)], len = a.len[min(k, a.n - 1)];
        const int there = max(__popcll(__ballot(k < hi && first(cu, k) <= at)), 1);
        lo += (there - 1) * step;
        if (step == 1) {
            const int cu0 = __builtin_amdgcn_readlane(cu, there - 1);
            return {lo, cu0, __builtin_amdgcn_readlane(cu, there), __builtin_amdgcn_readlane(len, there - 1), at - first(cu0, lo)};
        }
        hi = min(hi, lo + step);
    }
}

// Keys are counted along one line: the shared positions, a gap to the next multiple of 32, the request's own, of which the last
// are its tree's words. Columns: the (row, query head) pairs of one kv head, packed; a workgroup takes 16 NT of them and one part
// of the line, its four waves take blocks of 32 keys in turn. With K of 32 keys as rows of the first product (S^T = K Q^T) a
// lane holds the scores of one column, so maxima and sums stay in the lane: four of either half of the block's keys, which are its
// operand of the second product (O^T = V^T P^T) as they are, if V's rows are dealt the same way. V's operand is eight keys of one
// dimension: each lane loads the same D / 16 dimensions of its eight keys and turns the block with byte permutes. A load takes
// rows of one half, so its address is the wave's and a lane's place in it never changes. Keys are asked for as soon as the first
// product has read those before them, values as soon as the second has: loads are in flight all the time without registers of
// their own.
// Weights are rounded to the values' 16 bits for the second product; their sum stays in 32 bits. They are relative to a maximum
// that is up to 2^SLACK behind the true one and 2^LIFT below it (sh_page_attn.hip says why). Each column is rescaled by its own
// scores alone, but its tile's other columns decide whether its first reference is four waves' or its own wave's, and under a window
// which wave and part takes which key: the same call gives the same bits, a row beside other rows may round elsewhere.
// SHARED: the columns of all requests over the shared positions. Else one request's columns over its own positions, and over the
// shared ones before them where no SHARED part takes them (a.fused).
template <class T, int D, int NT, bool SHARED>
__device__ __forceinline__ void attend(const pattn_args& a, const int block, tree_space<D, NT>& s) {
    constexpr int NC = 16 * NT, E = D / 16, CH = D / 32, VW = E / 2, PITCH = tree_space<D, NT>::PITCH;
    // (f16 with a lift of 2^8 and 2^7 of slack rescales less often and is no more than 3 % faster, 64 requests with up to 64 words over
    // 2048 and 2048 positions 120.9 and 122.4 us, but weights of 2^-25.5 are then off by up to half a percent)
    constexpr float LIFT = mat<T>::LIFT, SLACK = mat<T>::SLACK;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m16 = lane & 15, quad = lane >> 4;
    const int S = SHARED ? a.sp : a.so, per = a.n_kv * S;
    // (workgroups of the same keys are `per` apart: on one XCD where that is a multiple of 8)
    const int gs = block % per, g = gs % a.n_kv, part = gs / a.n_kv;
    const int tile = block / per;
    // ---- the workgroup's columns ----
    int i = 0, r0 = 0, r1, ct = tile;      // request, its rows, tile of columns within them
    [[maybe_unused]] tile_of_request mine{};
    if constexpr (SHARED) {
        r1 = min(max(a.cu[a.n], 0), a.rows);
    } else {
        mine = find_tile(a, tile, lane, NC);
        i = mine.k;
        ct = mine.tile;
        r0 = min(max(mine.cu0, 0), a.rows);
        r1 = min(min(max(mine.cu1, 0), a.rows), r0 + a.max_rows);
    }
    const int ncol = (r1 - r0) * a.grp, c0 = ct * NC;
    if (c0 < 0 || c0 >= ncol) return;
    // (a column's row and head: within a tile small numbers are divided)
    const int row0 = c0 / a.grp, over0 = c0 - row0 * a.grp, last = ncol - 1 - c0, by = a.grp < 64 ? 65536 / a.grp + 1 : 0;
    auto rows_on = [&](int c) {
        const int x = over0 + min(c, last);
        return a.grp < 64 ? (x * by) >> 16 : x >= a.grp ? 1 : 0;
    };
    auto row_of = [&](int c) { return r0 + row0 + rows_on(c); };
    auto head_of = [&](int c) { return g * a.grp + over0 + min(c, last) - rows_on(c) * a.grp; };
    {
        constexpr int PER = 256 / NC;      // threads a column
        const int c = threadIdx.x / PER;
        const unsigned* from = a.mask + (size_t)row_of(c) * a.words;
        for (int w = threadIdx.x % PER; w <= a.words; w += PER) s.mask[c][w] = w < a.words ? from[w] : 0u;
    }
    u32x4 qf[CH][NT];
    auto load_queries = [&](int t) {
#pragma unroll
        for (int c = 0; c < CH; c++)
            qf[c][t] = *(const u32x4*)((const T*)a.q + ((size_t)row_of(16 * t + m16) * a.n_head + head_of(16 * t + m16)) * D + c * 32 + quad * 8);
    };
#pragma unroll
    for (int t = 0; t < NT; t++) load_queries(t);
    __syncthreads();
    // ---- what each column sees: of keys lo .. hi - 1 all before words_at, and the words there whose bits its mask has ----
    const int L0 = a.prefix_len, P = a.own_at;
    const int own_max = (int)min((long long)a.max_len, (long long)a.cols << a.page_log);
    int words_at = L0;
    int lo0 = INT_MAX, lo1 = 0, hi0 = INT_MAX, hi1 = 0;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int c = 16 * t + m16, row = row_of(c);
        const unsigned* mask = s.mask[c];
        const int k = SHARED ? request_of(a.cu, a.n, row) : i;
        const long long first_row = SHARED ? a.cu[k] : mine.cu0, rows_k = (SHARED ? a.cu[k + 1] : mine.cu1) - first_row, nth = row - first_row;
        const int held = min(max(SHARED ? a.len[k] : mine.len, 0), own_max);
        const int base = (int)max(held - rows_k, 0ll);   // the tree's first word
        const bool node = held >= rows_k && nth >= 0 && nth < 32ll * a.words && (mask[nth >> 5] >> (nth & 31) & 1);
        int from = 0, first_word = 0;
        if (node && a.window) {
            // (bits behind the request's rows are no words of its)
            auto bits_of = [&](int w) { return mask[w] & (rows_k - 32 * w >= 32 ? ~0u : rows_k <= 32 * w ? 0u : (1u << (rows_k - 32 * w)) - 1); };
            int depth = -1;
            for (int w = 0; w < a.words; w++) depth += __popc(bits_of(w));
            from = (int)max(L0 + base + depth + 1ll - a.window, 0ll);
            int drop = depth + 1 - a.window;   // of the words that it follows the window leaves the last ones
            for (int w = 0; w < a.words && drop > 0; w++) {
                unsigned bits = bits_of(w);
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
        int lo = node ? min(from, L0) : L0, hi = L0, sure = L0;
        if constexpr (!SHARED) {
            words_at = P + base;
            lo = first_word ? words_at + first_word : from >= L0 ? P + (from - L0) : a.fused ? from : P;
            hi = node ? P + held : lo;
            sure = node ? words_at : 0;
        }
        if (wv == 0 && quad == 0) {
            s.lo[c] = lo;
            s.hi[c] = hi;
        }
        lo0 = min(lo0, lo);
        lo1 = max(lo1, lo);
        hi0 = min(hi0, sure);
        hi1 = max(hi1, hi);
    }
    __syncthreads();
    lo0 = -most_of_16(-lo0);
    lo1 = most_of_16(lo1);
    hi0 = -most_of_16(-hi0);
    hi1 = most_of_16(hi1);
    if constexpr (!SHARED) words_at = __builtin_amdgcn_readfirstlane(words_at);
    // ---- the part: the first starts where the first column does; the last goes to the end ----
    const int chunk = SHARED ? a.pchunk : a.ochunk;
    const long long k0l = (long long)(lo0 & ~31) + (long long)part * chunk;
    const int k1 = part + 1 == S ? hi1 : (int)min((long long)hi1, k0l + chunk);
    const bool any = k0l < k1;
    const int k0 = any ? (int)k0l : 0;

    f32x4 o[E][NT];
    // each column's reference, turned round (0 before there is one), its sum of weights and the score from which on it is rescaled
    float nref[NT], l[NT], thr[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        thr[t] = -INFINITY;
        nref[t] = l[t] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) o[e][t] = f32x4{0, 0, 0, 0};
    }
    int kt = k0 + 32 * wv;
    if (any && kt < k1) {
        const int32_t* own = SHARED ? nullptr : a.table + (size_t)i * a.cols;
        const int pl = a.page_log, pm = (1 << pl) - 1;
        // A block of 32 keys is two halves of 16, each in one page. Pages are whole, so that no key of theirs is out of reach; what
        // lies behind the last one is masked
        auto place_of = [&](int kt) { return SHARED || kt < P ? kt : kt - P; };
        auto id_of = [&](int kt, int half) {
            const bool in_shared = SHARED || kt < P;
            const int last = in_shared ? L0 - 1 : hi1 - 1 - P;
            return (in_shared ? a.prefix : own)[min(place_of(kt) + 16 * half, last) >> pl];
        };
        auto known = [&](int id) { return (unsigned)id < (unsigned)a.n_pages; };
        // a half's place in the cache, counted in halves (of 1 KB and more: 32 bits reach 4 TB)
        auto half_of = [&](int kt, int half, int id) {
            return ((known(id) ? (unsigned)id : 0u) * (unsigned)a.n_kv + (unsigned)g) * (unsigned)((pm + 1) >> 4) + (unsigned)(((place_of(kt) + 16 * half) & pm) >> 4);
        };
        // whether every column sees every key of a block (of pages id0, id1)
        auto is_full = [&](int kt, int id0, int id1) {
            return kt >= lo1 && kt + 32 <= hi0 && (SHARED || kt < P ? L0 : hi1) - kt >= 32 && known(id0) && known(id1);
        };
        constexpr int RL = D / 8, RI = 64 / RL, KI = 32 / RI;  // lanes that load a row, rows that the wave loads at once
        u32x4 kr[KI], kf[2][CH];
        unsigned vw[8][VW];
        const unsigned k_lane = lane * 16, v_lane = quad * (4 * D * 2) + m16 * (E * 2);
        auto load_keys = [&](unsigned half0, unsigned half1) {
#pragma unroll
            for (int n = 0; n < KI; n++) {
                const char* p = (const char*)a.keys + (size_t)(n * RI / 16 ? half1 : half0) * (32 * D) + (n * RI % 16) * (D * 2);
                kr[n] = *(const u32x4*)(p + k_lane);
            }
        };
        unsigned short* const kw = s.wave[wv].keys + lane / RL * (D + 8) + lane % RL * 8;
        const unsigned short* const ks = s.wave[wv].keys + m16 * (D + 8) + quad * 8;
        auto turn_keys = [&]() {
#pragma unroll
            for (int n = 0; n < KI; n++) *(u32x4*)(kw + n * RI * (D + 8)) = kr[n];
            wave_lds();
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int c = 0; c < CH; c++) kf[h][c] = *(const u32x4*)(ks + h * 16 * (D + 8) + c * 32);
            wave_lds();
        };
        auto load_values = [&](unsigned half0, unsigned half1) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const char* p = (const char*)a.values + (size_t)(h ? half1 : half0) * (32 * D);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const char* q = p + v_lane + k * (D * 2);
                    if constexpr (VW == 4) *(u32x4*)vw[4 * h + k] = *(const u32x4*)q;
                    else if constexpr (VW == 2) *(uint2*)vw[4 * h + k] = *(const uint2*)q;
                    else vw[4 * h + k][0] = *(const unsigned*)q;
                }
            }
        };
        auto scores = [&](int t, float (&x)[8]) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                f32x4 c4 = {0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < CH; c++) c4 = mat<T>::mul(kf[h][c], qf[c][t], c4);
#pragma unroll
                for (int r = 0; r < 4; r++) x[4 * h + r] = c4[r];
            }
        };
        auto largest = [&](const float (&x)[8]) {      // (NaN where one is: the column is NaN then, whatever its reference)
            float y = x[0];
#pragma unroll
            for (int k = 1; k < 8; k++) y = __builtin_elementwise_maximum(y, x[k]);
            return y;
        };
        auto refer_to = [&](int t, float top) {
            nref[t] = LIFT - top * a.c;
            thr[t] = (SLACK + LIFT - nref[t]) / a.c;
        };
        // a column's new reference where its largest score passes the old one's slack
        auto move_to = [&](int t, float top) {
            const float y = over_quads(top);
            if (y > thr[t]) {
                const float old = nref[t];
                const bool none = thr[t] == -INFINITY;
                refer_to(t, y);
                const float f = none ? 0.0f : exp2_(nref[t] - old);
                l[t] *= f;
#pragma unroll
                for (int e = 0; e < E; e++) o[e][t] *= f;
            }
        };
        unsigned pw[NT][4];
        auto weights = [&](int t, float (&x)[8]) {
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                x[k] = exp2_(fmaf(x[k], a.c, nref[t]));
                sum += x[k];
            }
            l[t] += sum;
#pragma unroll
            for (int k = 0; k < 4; k++) pw[t][k] = pack2<T>(x[2 * k], x[2 * k + 1]);
        };
        u32x4 vf[E];
        auto turn_values = [&]() {
#pragma unroll
            for (int e = 0; e < E; e++) {  // dimension m16 * E + e of eight keys
                const unsigned sel = (e & 1) ? 0x07060302u : 0x05040100u;
#pragma unroll
                for (int k = 0; k < 4; k++) vf[e][k] = __builtin_amdgcn_perm(vw[2 * k + 1][e >> 1], vw[2 * k][e >> 1], sel);
            }
        };
        auto add_values = [&](int t) {
#pragma unroll
            for (int e = 0; e < E; e++) o[e][t] = mat<T>::mul(vf[e], u32x4{pw[t][0], pw[t][1], pw[t][2], pw[t][3]}, o[e][t]);
        };
        // of a lane's eight keys those that its column sees
        // (the lane's number, unknown to the compiler: what follows from it is not kept in registers from block to block)
        auto lane_here = [&]() {
            int self = lane;
            asm volatile("" : "+v"(self));
            return self;
        };
        auto sees = [&](int t, int kt, bool known0, bool known1) {
            const bool in_shared = SHARED || kt < P;
            const int self = lane_here(), c = 16 * t + (self & 15), quad = self >> 4, from = s.lo[c], stop = min(s.hi[c], in_shared ? L0 : hi1);
            unsigned bits = 0;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int first = kt + 16 * h + quad * 4;
                unsigned four = (h ? known1 : known0) ? 0xFu : 0u;
                if (!SHARED && !in_shared) four &= tree_bits(s.mask[c], a.words, first - words_at);
                four &= from - first >= 4 ? 0u : 0xFu << max(from - first, 0);
                bits |= (four & (stop <= first ? 0u : 0xFu >> max(4 - (stop - first), 0))) << (4 * h);
            }
            return bits;
        };
        bool odd = false;                  // infinities or NaN among values that some columns see
        bool start = max(lo1, k0) + 128 <= min(hi0, k1) - 31;      // (each wave has a block that its columns see whole)
#pragma unroll 1
        for (int first = kt; first < k1; first += 63 * 128) {
            // page ids of the wave's next 63 blocks, one a lane, and which of these blocks all columns see whole (the bit behind the
            // last one's is not set)
            const int many = min((k1 - first + 127) / 128, 63), lanes = first + 128 * min(lane, many - 1);
            const int ids0 = id_of(lanes, 0), ids1 = id_of(lanes, 1);
            const unsigned long long whole = __ballot(lane < many && is_full(lanes, ids0, ids1));
            const unsigned long long known0 = __ballot(known(ids0)), known1 = __ballot(known(ids1));
            const unsigned halves0 = half_of(lanes, 0, ids0), halves1 = half_of(lanes, 1, ids1);
            // (behind the last block it is asked for again)
            auto ask_keys = [&](int n) { load_keys(__builtin_amdgcn_readlane(halves0, min(n, many - 1)), __builtin_amdgcn_readlane(halves1, min(n, many - 1))); };
            auto ask_values = [&](int n) { load_values(__builtin_amdgcn_readlane(halves0, min(n, many - 1)), __builtin_amdgcn_readlane(halves1, min(n, many - 1))); };
            // (the order in which they are asked for is the one in which they are waited for)
            ask_keys(0);
            turn_keys();
            ask_keys(1);
            __builtin_amdgcn_sched_barrier(0);
            ask_values(0);
            __builtin_amdgcn_sched_barrier(0);
            if (start) {
                // The first reference is the largest of all four waves' first blocks: far fewer scores pass it by the slack later on
                start = false;
                const int self = lane_here(), m16 = self & 15, quad = self >> 4;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    float x[8];
                    scores(t, x);
                    const float y = over_quads(largest(x));
                    if (quad == 0) s.top[wv][16 * t + m16] = whole & 1 ? y : -INFINITY;
                }
                __syncthreads();
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const int c = 16 * t + m16;
                    const float y = fmaxf(fmaxf(s.top[0][c], s.top[1][c]), fmaxf(s.top[2][c], s.top[3][c]));
                    if (y > -INFINITY) refer_to(t, y);
                }
            }
            int n = 0;
#pragma unroll 1
            for (;;) {
                // ---- blocks that all columns see whole ----
#pragma unroll 1
                while (whole >> n & 1) {
                    float x[NT][8], top[NT];
#pragma unroll
                    for (int t = 0; t < NT; t++) scores(t, x[t]);
                    turn_keys();
                    ask_keys(n + 2);
                    bool over = false;
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        top[t] = largest(x[t]);
                        over |= top[t] > thr[t];
                    }
                    if (__any(over)) {
#pragma unroll
                        for (int t = 0; t < NT; t++) move_to(t, top[t]);
                    }
                    // products of a column group with the values beside the next group's weights
                    weights(0, x[0]);
                    turn_values();
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        add_values(t);
                        if (t + 1 < NT) weights(t + 1, x[t + 1]);
                    }
                    ask_values(++n);
                }
                if (n >= many) break;
                // ---- others: at a window's edges, the shared positions' end, pages that are not there, and the tree ----
                unsigned any_sees = 0, bits[NT];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    bits[t] = sees(t, first + 128 * n, known0 >> n & 1, known1 >> n & 1);
                    any_sees |= bits[t];
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    float x[8];
                    scores(t, x);
#pragma unroll
                    for (int k = 0; k < 8; k++) x[k] = bits[t] >> k & 1 ? x[k] : -INFINITY;
                    const float top = largest(x);
                    if (__any(top > thr[t])) move_to(t, top);
                    weights(t, x);
                    __builtin_amdgcn_sched_barrier(0);
                }
                any_sees = any_of_16(any_sees);
                unsigned full = 0;             // (a value whose exponent bits are all set carries into its sign)
#pragma unroll
                for (int k = 0; k < 8; k++)
#pragma unroll
                    for (int w = 0; w < VW; w++) {
                        vw[k][w] &= 0u - (any_sees >> k & 1);
                        full |= (vw[k][w] & mat<T>::EXP * 0x10001u) + (mat<T>::EXP & -mat<T>::EXP) * 0x10001u;
                    }
                if (__any(full & 0x80008000u)) {
                    // A weight of 0 times an infinity would reach columns that do not see the key: such values are left out (below)
                    odd = true;
#pragma unroll
                    for (int k = 0; k < 8; k++)
#pragma unroll
                        for (int w = 0; w < VW; w++) {
                            if ((vw[k][w] & mat<T>::EXP) == mat<T>::EXP) vw[k][w] &= 0xFFFF0000u;
                            if ((vw[k][w] >> 16 & mat<T>::EXP) == mat<T>::EXP) vw[k][w] &= 0x0000FFFFu;
                        }
                }
                __builtin_amdgcn_sched_barrier(0);
                turn_values();
#pragma unroll
                for (int t = 0; t < NT; t++) add_values(t);
                __builtin_amdgcn_sched_barrier(0);
                turn_keys();
                ask_keys(n + 2);
                ask_values(++n);
                if (n >= many) break;
                }
        }
        // ---- the wave's sums to LDS, behind the last of its keys ----
        const int self = lane_here(), m16 = self & 15, quad = self >> 4;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int c = 16 * t + m16;
            l[t] += __shfl_xor(l[t], 16);
            l[t] += __shfl_xor(l[t], 32);
            if (quad == 0) {
                ((float*)&s.m[c])[wv] = thr[t] == -INFINITY ? -INFINITY : -nref[t];
                ((float*)&s.l[c])[wv] = l[t];
            }
#pragma unroll
            for (int k = 0; k < E; k++) {
                f32x4 x;
#pragma unroll
                for (int r = 0; r < 4; r++) x[r] = o[(4 * k + r) % E][t][(4 * k + r) / E];
                *(f32x4*)(s.wave[wv].o + c * PITCH + quad * 4 * E + 4 * k) = x;
            }
        }
        if (odd) {
            // Infinities and NaN that some columns of a block see: how many a column sees of either sign (NaN: of both, and so an
            // infinity whose weight is 0) is counted by products of ones
#pragma unroll 1
            for (kt = k0 + 32 * wv; kt < k1; kt += 128) {
                const int id0 = id_of(kt, 0), id1 = id_of(kt, 1);
                if (is_full(kt, id0, id1)) continue;
                const unsigned half0 = half_of(kt, 0, id0), half1 = half_of(kt, 1, id1);
                load_values(half0, half1);
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int c = 0; c < CH; c++) kf[h][c] = *(const u32x4*)((const T*)a.keys + (size_t)(h ? half1 : half0) * (16 * D) + m16 * D + c * 32 + quad * 8);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const unsigned bits = sees(t, kt, known(id0), known(id1));
                    float x[8];
                    load_queries(t);
                    scores(t, x);
                    u32x4 st, nt;              // ones for the keys that the column sees, and for those of them without weight
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const unsigned w = pack2<T>(exp2_(fmaf(x[2 * k], a.c, nref[t])), exp2_(fmaf(x[2 * k + 1], a.c, nref[t])));
                        st[k] = (bits >> 2 * k & 1 ? mat<T>::ONE : 0u) | (bits >> 2 * k & 2 ? mat<T>::ONE << 16 : 0u);
                        nt[k] = st[k] & ((w & 0x7FFFu ? 0u : 0xFFFFu) | (w & 0x7FFF0000u ? 0u : 0xFFFF0000u));
                    }
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        u32x4 up, down;
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            up[k] = down[k] = 0;
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const unsigned v = vw[2 * k + h][e >> 1] >> (16 * (e & 1)) & 0xFFFFu, one = mat<T>::ONE << (16 * h);
                                const bool bad = (v & mat<T>::EXP) == mat<T>::EXP, nan = bad && (v & (0x7FFFu ^ mat<T>::EXP));
                                up[k] |= nan || (bad && !(v & 0x8000u)) ? one : 0u;
                                down[k] |= nan || (bad && (v & 0x8000u)) ? one : 0u;
                            }
                        }
                        const f32x4 plus = mat<T>::mul(down, nt, mat<T>::mul(up, st, f32x4{0, 0, 0, 0}));
                        const f32x4 less = mat<T>::mul(up, nt, mat<T>::mul(down, st, f32x4{0, 0, 0, 0}));
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            float& at = s.wave[wv].o[(16 * t + m16) * PITCH + quad * 4 * E + r * E + e];
                            if (plus[r] > 0.0f) at += INFINITY;
                            if (less[r] > 0.0f) at -= INFINITY;
                        }
                    }
                }
            }
        }
    }
    // ---- the four waves joined: their sums through LDS, then each thread adds up four neighbouring dimensions of a column ----
    constexpr int LD = D / 4, STEP = 256 / LD, TURNS = (NC + STEP - 1) / STEP;   // threads a column, columns at once
    const bool alone = a.sp + a.so == 1;
    const int d = threadIdx.x % LD * 4, with = any ? min((k1 - k0 + 31) / 32, 4) : 0;   // (waves from `with` on had no block)
    float gate[TURNS];
    if (alone && a.gate) {
#pragma unroll
        for (int n = 0; n < TURNS; n++) {
            const int c = n * STEP + threadIdx.x / LD;
            gate[n] = a.gate[(size_t)row_of(c) * a.n_head + head_of(c)];
        }
    }
    __syncthreads();
    float top[TURNS], sum[TURNS];
    f32x4 x[TURNS], f[TURNS];
#pragma unroll
    for (int n = 0; n < TURNS; n++) {
        const int c = min(n * STEP + (int)threadIdx.x / LD, NC - 1);
        const f32x4 m4 = s.m[c], l4 = s.l[c];
        top[n] = -INFINITY;
        sum[n] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++)
            if (w < with) top[n] = fmaxf(top[n], m4[w]);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            f[n][w] = rescale(m4[w], top[n]);
            if (w < with) sum[n] += l4[w] * f[n][w];
        }
        x[n] = f32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (w >= with) break;
#pragma unroll
        for (int n = 0; n < TURNS; n++) x[n] += *(const f32x4*)(s.wave[w].o + min(n * STEP + (int)threadIdx.x / LD, NC - 1) * PITCH + d) * f[n][w];
    }
#pragma unroll
    for (int n = 0; n < TURNS; n++) {
        const int c = n * STEP + threadIdx.x / LD;
        if (c >= NC || c0 + c >= ncol) continue;
        const size_t rh = (size_t)row_of(c) * a.n_head + head_of(c);
        if (alone) {
            float per = 1.0f / sum[n];
            if (a.gate) per *= 1.0f / (1.0f + expf(-gate[n]));
            uint2 y = {0u, 0u};
            if (sum[n] != 0.0f) y = {pack2<T>(x[n][0] * per, x[n][1] * per), pack2<T>(x[n][2] * per, x[n][3] * per)};
            *(uint2*)((T*)a.out + rh * D + d) = y;
            if (a.lse && d == 0) a.lse[rh] = sum[n] == 0.0f ? -INFINITY : (top[n] + log2f(sum[n])) * 0.69314718055994531f;
        } else {
            const size_t at = (size_t)(SHARED ? part : a.sp + part) * a.rows * a.n_head + rh;
            if (d == 0) a.part_ml[at] = make_float2(top[n], sum[n]);
            if (any) *(f32x4*)(a.part_o + at * D + d) = x[n];
        }
    }
}

// Waves per SIMD that the registers are to allow: the most without spills in the loops (heads of 128, one column group, at three
// waves 64 requests x 4 words over 2048 positions 50 us, at two 30)
constexpr int waves_of(int D, int nts, int nto) {
    const int nt = nts > nto ? nts : nto;
    return nt == 4 || D > 64 ? 2 : nt == 2 ? 3 : 4;
}

template <class T, int D, int NTS, int NTO>
__global__ __launch_bounds__(256, waves_of(D, NTS, NTO)) void k_tree_attn(pattn_args a) {
    __shared__ __align__(16) union { tree_space<D, NTO> own; tree_space<D, NTS ? NTS : 1> shared; } s;
    int b = blockIdx.x;
    if constexpr (NTS > 0) {
        const long long grp = b >> 3, gs = (a.shared_blocks + 7) >> 3, all = gridDim.x >> 3;
        const long long before = grp * gs / all, next = (grp + 1) * gs / all;   // shared groups before this one, with it
        if (next > before) {
            b = (int)(before * 8) + (b & 7);
            if (b < a.shared_blocks) attend<T, D, NTS ? NTS : 1, true>(a, b, s.shared);
            return;
        }
        b = (int)((grp - before) * 8) + (b & 7);
        if (b >= a.own_blocks) return;
    }
    attend<T, D, NTO, false>(a, b, s.own);
}

template <class T, int D, int NTS, int NTO> hipError_t run_attn(const pattn_args& a, hipStream_t s) {
    const long long blocks = NTS ? ((a.shared_blocks + 7ll) / 8 + (a.own_blocks + 7ll) / 8) * 8 : a.own_blocks;
    k_tree_attn<T, D, NTS, NTO><<<dim3((unsigned)blocks), 256, 0, s>>>(a);
    return hipGetLastError();
}
template <class T, int D> hipError_t run_all(const pattn_args& a, hipStream_t s) {
    if (a.sp) return a.nts == 1 ? run_attn<T, D, 1, 1>(a, s) : a.nto == 1 ? run_attn<T, D, 2, 1>(a, s) : run_attn<T, D, 2, 2>(a, s);
    if constexpr (D <= 64)
        if (a.nto == 4) return run_attn<T, D, 0, 4>(a, s);
    return a.nto == 1 ? run_attn<T, D, 0, 1>(a, s) : run_attn<T, D, 0, 2>(a, s);
}
template <class T> hipError_t run_dim(int D, const pattn_args& a, hipStream_t s) {
    return D == 32 ? run_all<T, 32>(a, s) : D == 64 ? run_all<T, 64>(a, s) : run_all<T, 128>(a, s);
}

}  // namespace

// Which workgroups take the shared positions, and into how many parts the keys go.
bool tree_attn_split(int D, pattn_args& a) {
    const long long cols = (long long)a.rows * a.grp, most = (long long)a.max_rows * a.grp;
    // Column groups of 16 a workgroup takes. Wide tiles read a block of keys fewer times, narrow ones make more workgroups that run
    // at once, so the work of all columns decides (columns times positions times kv heads, w; heads of 128 twice), where one group does
    // not hold a request's columns. us by 1, 2 and 4 groups of heads of 64, 8 kv heads: 64 requests x 8 words over 500 positions (w 4
    // million) 13.0, 14.5 and 22.4, 64 x 16 over 500 (8) 18.0, 18.7 and 23.8, one of 64 words over 4096 (8) 14.6, 14.1 and 17.3, one of 32
    // over 16000 (16) 19.4, 17.6 and 20.3, 8 x 64 over 2500 (23) 21.5, 20.4 and 24.6, one of 256 over 4096 (34) 23.8, 20.3 and 28.7, 64 x
    // 32 over 4096 (136) 120, 94.8 and 89.0, 64 x 64 over 4096 (273) 176, 127 and 113. Four groups of heads of 128 do not fit the
    // registers; by 1 and 2, 4 kv heads: one of 64 words over 4096 (8) 14.6 and 18.5, 64 x 16 over 500 (8) 21.7 and 20.2, one of 32 over
    // 16000 (16) 19.5 and 21.1, 8 x 64 over 2500 (23) 24.4 and 23.0, one of 256 over 4096 (34) 21.3 and 24.8, one of 33 over 32749 (35)
    // 30.6 and 27.2, 64 x 64 over 4096 (273) 180 and 143. Work alone does not tell a long request from a batch: the rule takes the slower
    // side for 64 x 32 over 4096 (by 7 %) and, in heads of 128, for 64 x 16 over 500 (7), one of 32 over 16000 (8) and one of 256 over
    // 4096 (16)
    a.nts = cols <= 16 ? 1 : 2;
    auto groups = [&](long long range) {
        if (a.window) range = std::min(range, a.window + 63ll + a.max_rows);
        const double w = (double)cols * range * a.n_kv * (D > 64 ? 2 : 1);
        return most <= 16 || w <= 12e6 ? 1 : D > 64 || most <= 32 || w < 200e6 ? 2 : 4;
    };
    a.nto = groups(a.prefix_len + a.max_len);
    long long own = cols / (16 * a.nto) + a.n;
    const long long all = (cols + 16 * a.nts - 1) / (16 * a.nts);
    auto split = [&](long long tiles, long long range, long long want, int* parts, int* chunk) {
        const long long p = std::max(std::min(want / std::max(tiles * a.n_kv, 1ll), (range + 511) / 512), 1ll);
        *chunk = (int)std::max(((range + p - 1) / p + 127) / 128 * 128, 128ll);
        *parts = (int)std::max((range + *chunk - 1) / *chunk, 1ll);
    };
    a.own_at = (a.prefix_len + 31) / 32 * 32;
    // Requests read the shared positions themselves where their columns fill their workgroups (sharing would save no reads, and
    // nothing has to be joined), and where they are few or the shared positions are: sharing costs a launch and the parts' sums.
    // us apart and fused, by requests x words behind shared positions, 1000 own ones, 8 kv heads of 64, then 4 of 128: 64 x 64 behind
    // 1024 142 and 85, 114 and 76; 64 x 24 behind 4096 104 and 87, 95 and 89; with more than twice as many tiles of requests as of all
    // columns 32 x 2 behind 1024 (tiles times positions 40960) 17 and 14, 21 and 19, 64 x 4 behind 1024 (98304) 27 and 23, 27 and 26,
    // 32 x 2 behind 4096 (163840) 21 and 31, 24 and 30, 64 x 4 behind 4096 (393216) 34 and 48, 40 and 48
    a.fused = a.prefix_len == 0 || own <= all * 2 || own * a.prefix_len <= 100000;
    a.sp = a.pchunk = 0;
    if (!a.fused) {
        a.nto = std::min(groups(a.max_len), 2);
        own = cols / (16 * a.nto) + a.n;
    }
    if (!a.fused) split(all, a.window && a.window + 31ll < a.prefix_len ? a.window + 31ll : a.prefix_len, 512, &a.sp, &a.pchunk);
    long long range = (a.fused ? a.own_at : 0ll) + a.max_len;
    if (a.window) range = std::min(range, a.window + 63ll + a.max_rows);
    // One workgroup per compute unit, of 512 keys or more: one request of 64 words over 33000 positions (8 kv heads of 64) 32 us, with
    // three quarters as many parts 37, with one and a half times as many 35 (the join reads all of them); 4 kv heads of 128 31, 34 and 36.
    // 64 requests x 4 words behind 2048 shared positions, 4 kv heads of 128, by 256, 512 and 1024 keys a part 44.8, 39.7 and 38.5,
    // 8 of 64 35.4, 35.1 and 38.6 (one input again and again)
    split(std::max((cols + 16 * a.nto - 1) / (16 * a.nto), (long long)a.n), range, 256, &a.so, &a.ochunk);
    const long long shared_blocks = all * a.n_kv * a.sp, own_blocks = own * a.n_kv * a.so;
    const long long rh = (long long)a.rows * a.n_head, join = a.sp + a.so == 1 ? 0 : a.sp + a.so > 16 ? rh : (rh + 3) / 4;
    // (columns of one kv head are counted in 32 bits in the kernel)
    if (shared_blocks + own_blocks + 16 > most_blocks(256) || join > most_blocks(256) || cols > INT_MAX / 2) return false;
    a.shared_blocks = (int)shared_blocks;
    a.own_blocks = (int)own_blocks;
    return true;
}

hipError_t launch_tree_attn(int D, int type, const pattn_args& a, hipStream_t s) {
    const hipError_t e = type == TY_F16 ? run_dim<_Float16>(D, a, s) : run_dim<__bf16>(D, a, s);
    return e == hipSuccess ? launch_page_join(D, type, a, s) : e;
}

}  // namespace sh
