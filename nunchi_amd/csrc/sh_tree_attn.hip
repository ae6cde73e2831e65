// Attention of a batch whose requests try a tree of drafted words each (sh_tree_attn): the workgroups of sh_attend.h, in which
// a row sees of its request's last positions those whose bits its mask has. The parts are joined by sh_page_attn.hip's kernel.
#include <hip/hip_runtime.h>

#include "sh_attend.h"

namespace sh {
namespace {

constexpr int waves_of(int D, int nts, int nto) { return nts > 1 || nto > 1 ? 2 : D > 64 ? 3 : 4; }

template <class T, int D, int NTS, int NTO>
__global__ __launch_bounds__(256, waves_of(D, NTS, NTO)) void k_tree_attn(pattn_args a) {
    __shared__ __align__(16) union { join_space<D, NTO> own; join_space<D, NTS ? NTS : 1> shared; } js;
    int b = blockIdx.x;
    if constexpr (NTS > 0) {
        const long long grp = b >> 3, gs = (a.shared_blocks + 7) >> 3, all = gridDim.x >> 3;
        const long long before = grp * gs / all, next = (grp + 1) * gs / all;   // shared groups before this one, with it
        if (next > before) {
            b = (int)(before * 8) + (b & 7);
            if (b < a.shared_blocks) attend<T, D, NTS ? NTS : 1, true, true>(a, b, js.shared);
            return;
        }
        b = (int)((grp - before) * 8) + (b & 7);
        if (b >= a.own_blocks) return;
    }
    attend<T, D, NTO, false, true>(a, b, js.own);
}

template <class T, int D, int NTS, int NTO> hipError_t run_attn(const pattn_args& a, hipStream_t s) {
    const long long blocks = NTS ? ((a.shared_blocks + 7ll) / 8 + (a.own_blocks + 7ll) / 8) * 8 : a.own_blocks;
    k_tree_attn<T, D, NTS, NTO><<<dim3((unsigned)blocks), 256, 0, s>>>(a);
    return hipGetLastError();
}
template <class T, int D> hipError_t run_all(const pattn_args& a, hipStream_t s) {
    constexpr int M = attn_many(D);
    const int nts = a.sp ? attn_col_groups(D, (long long)a.rows * a.grp) : 0, nto = attn_col_groups(D, (long long)a.max_rows * a.grp);
    if (nts == 0) return nto == 1 ? run_attn<T, D, 0, 1>(a, s) : run_attn<T, D, 0, M>(a, s);
    if (nts == 1) return run_attn<T, D, 1, 1>(a, s);   // (a request has no more columns than all of them)
    return nto == 1 ? run_attn<T, D, M, 1>(a, s) : run_attn<T, D, M, M>(a, s);
}
template <class T> hipError_t run_dim(int D, const pattn_args& a, hipStream_t s) {
    return D == 32 ? run_all<T, 32>(a, s) : D == 64 ? run_all<T, 64>(a, s) : run_all<T, 128>(a, s);
}

}  // namespace

hipError_t launch_tree_attn(int D, int type, const pattn_args& a, hipStream_t s) {
    const hipError_t e = type == TY_F16 ? run_dim<_Float16>(D, a, s) : run_dim<__bf16>(D, a, s);
    return e == hipSuccess ? launch_page_join(D, type, a, s) : e;
}

}  // namespace sh
