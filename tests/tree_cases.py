"""Cases of tree_attn that reach each of its kernels: k_tree_attn<type, head_dim, column groups of the shared positions' workgroups (0: none of their
own), of the requests'>. tests/test_tree_split.py asks the library's rule which kernel each case takes, tests/test_gpu_tree_wide.py runs them."""
import numpy as np

DIMS = (32, 64, 128)


def _lens(base, sizes):
    return [b + m for b, m in zip(base, sizes)]


def _short(n, most, seed):
    """Own positions before the words: none, one, and numbers around blocks and pages."""
    return [0, 1, 31, 32, 33, 63, 64, 65][:n] + np.random.default_rng(seed).integers(0, most, max(n - 8, 0)).tolist()


def cases():
    out = []
    for D in DIMS:
        wide = 2 if D > 64 else 1
        # 16 columns in all behind a long shared beginning
        sizes = [1] * 13 + [0, 2, 1]
        add = dict(D=D, H=2, K=2, page=16, sizes=sizes, lens=_lens(_short(16, 300, D), sizes))
        out += [dict(add, kernel=(1, 1), prefix=6101, window=0), dict(add, kernel=(1, 1), prefix=6101, window=3000), dict(add, kernel=(1, 1), prefix=9003, window=40)]
        # a few words of many requests
        sizes = [1, 2, 3, 4, 0, 4, 1, 2] * 5
        add = dict(D=D, H=8, K=2, page=32, sizes=sizes, lens=_lens(_short(40, 150, D + 1), sizes))
        out += [dict(add, kernel=(2, 1), prefix=1777, window=0), dict(add, kernel=(2, 1), prefix=1777, window=700), dict(add, kernel=(2, 1), prefix=1777, window=3)]
        # more words than one column group holds, and one request that is long
        sizes = ([5] * 9 + [1, 12, 0]) * 5
        base = _short(60, 90, D + 2)
        base[30] = 2700 // wide
        add = dict(D=D, H=16, K=4, page=64, sizes=sizes, lens=_lens(base, sizes))
        out += [dict(add, kernel=(2, 2), prefix=1403, window=0), dict(add, kernel=(2, 2), prefix=1403, window=2650 // wide)]
        # two column groups, no shared workgroups
        sizes = [40, 9, 0, 33]
        add = dict(D=D, H=16, K=4, page=32, sizes=sizes, lens=_lens([70, 9700 // wide, 8, 200], sizes))
        out += [dict(add, kernel=(0, 2), prefix=0, window=0), dict(add, kernel=(0, 2), prefix=99, window=0), dict(add, kernel=(0, 2), prefix=99, window=9600 // wide)]
        # four
        if D <= 64:
            sizes = [64, 60, 33, 0, 100]
            add = dict(D=D, H=64, K=8, page=128, sizes=sizes, lens=_lens([0, 12500, 63, 40, 1000], sizes))
            out += [dict(add, kernel=(0, 4), prefix=0, window=0), dict(add, kernel=(0, 4), prefix=301, window=0), dict(add, kernel=(0, 4), prefix=301, window=12400)]
        # one column group: the usual sizes, whole and in parts
        sizes = [3, 40, 0, 1, 12]
        add = dict(D=D, H=8, K=2, page=16, sizes=sizes, lens=_lens([9, 1700, 4, 31, 64], sizes))
        out += [dict(add, kernel=(0, 1), prefix=77, window=0), dict(add, kernel=(0, 1), prefix=77, window=50)]
    return out


def name(c):
    return f"{c['kernel'][0]}-{c['kernel'][1]}-D{c['D']}-prefix{c['prefix']}-window{c['window']}"


def sizes_of(c):
    """What the rule goes by: n rows n_head n_kv head_dim prefix_len max_len max_rows window."""
    return [len(c["sizes"]), sum(c["sizes"]), c["H"], c["K"], c["D"], c["prefix"], max(c["lens"]), max(c["sizes"]), c["window"]]
