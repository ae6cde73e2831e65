"""The operators for drafted words where plans, masks, pages and lengths are not the ordinary ones: what one of them refuses, the others do not
take for whole. References and tolerances are tests/test_gpu_tree.py's."""
import numpy as np
import pytest

import nunchi_amd

torch = pytest.importorskip("torch")
import test_gpu_tree as tt  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return nunchi_amd.Context(0, stream=torch.cuda.current_stream().cuda_stream)


def test_take_first_rows_with_a_parent(ctx):
    """A first row whose parent is not before it has no bits in the plan, nor has what follows it: nothing of the request is kept, the
    positions of its rows and their pages go back. The requests beside it do not notice."""
    sizes, held = [3, 20, 4, 2, 3], [40, 30, 15, 16, 9]
    for first in (0, 2, -2, 2 ** 31 - 1, -2 ** 31):
        parent, words, picks, _ = tt.take_case(8, sizes, 2)
        for at in (3, 23):
            parent[at] = first
        length = [h + m for h, m in zip(held, sizes)]
        table, free = np.arange(5 * 6).reshape(5, 6) + 400, np.arange(900, 960)
        want = tt.take_reference(sizes, parent, words, picks, held, length, table, 16, free, 40)
        _, pos = tt.run_plan(ctx, tt.starts(sizes), parent, held, length, 32)
        assert (pos[3:27] == -1).all() and (pos[:3] >= 0).all() and (pos[27:] >= 0).all()
        got = tt.run_take(ctx, tt.starts(sizes), parent, words, picks, held, length, table, 16, free, 40)
        assert got["count"][1] == got["count"][2] == 0 and got["next"][1] == got["next"][2] == -1 and (got["path"][3:27] == -1).all()
        assert got["length"][1:3].tolist() == held[1:3]
        other = [0, 3, 4]
        assert got["count"][other].tolist() == want["count"][other].tolist() and got["length"][other].tolist() == want["length"][other].tolist()
        # pages of positions 30 .. 49 (16 a page: two behind the first two) and 15 .. 18 (one behind the first)
        back = sum((table[i, -(-int(got["length"][i]) // 16):-(-length[i] // 16)].tolist() for i in range(5)), [])
        assert [int(x) for x in table[1, 2:4]] == [x for x in back if x in table[1]] and [int(table[2, 1])] == [x for x in back if x in table[2]]
        assert got["taken"].tolist() == [40 - len(back)] and got["free"][40 - len(back):40].tolist() == back
