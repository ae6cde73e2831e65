// Which kernel sh_tree_attn takes for given sizes, and into how many parts it cuts the shared positions and the own ones: the library's own rule, for
// tests that are to reach every kernel. Arguments, any number of times: n rows n_head n_kv head_dim prefix_len max_len max_rows window.
#include <cstdio>
#include <cstdlib>

#include "../../nunchi_amd/csrc/sh_serve.h"

int main(int argc, char** argv) {
    for (int k = 1; k + 8 < argc; k += 9) {
        int v[9];
        for (int i = 0; i < 9; i++) v[i] = std::atoi(argv[k + i]);
        sh::pattn_args a{};
        a.n = v[0], a.rows = v[1], a.n_head = v[2], a.n_kv = v[3], a.grp = v[2] / v[3], a.prefix_len = v[5], a.max_len = v[6];
        a.max_rows = v[7] < v[1] ? v[7] : v[1];
        a.window = v[8] < v[5] + v[6] ? v[8] : 0;
        if (!sh::tree_attn_split(v[4], a)) return 1;
        std::printf("%d %d %d %d\n", a.sp ? a.nts : 0, a.nto, a.sp, a.so);
    }
}
