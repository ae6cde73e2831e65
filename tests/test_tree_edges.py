"""Checks of the operators for drafted words that need no GPU: refusals before the context or any buffer is touched (the context and the buffers
are addresses only)."""
from types import SimpleNamespace

import pytest

import nunchi_amd
from test_batch_args import ARG, BASE, _lib, at
from test_tree_args import TAKE


def planned(**bad):
    """sh_tree_take_planned's arguments: sh_tree_take's with the positions behind the parents."""
    v = {}
    for k, x in TAKE.items():
        v[k] = x
        if k == "parent":
            v["pos"] = at(14)
    return {**v, **bad}.values()


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(n=0), dict(n=4097), dict(rows=-1), *[{k: None} for k in ("cu", "parent", "words", "picks", "held", "len",
                                 "path", "count", "next", "len_out", "free", "taken", "taken_out")], dict(page=24), dict(cols=-1), dict(n_free=-1),
                                 # an output over an input, or over another output
                                 dict(path=at(14)), dict(count=at(14) + 32), dict(taken_out=at(14) + 4), dict(free=at(14) - 76), dict(path=at(1)), dict(len_out=at(5)),
                                 dict(taken_out=at(11) + 76)], ids=str)
def test_take_planned_refused(bad):
    assert _lib().sh_tree_take_planned(*planned(**bad)) == ARG
    assert b"sh_tree_take_planned" in _lib().sh_last_error()


def test_take_positions_are_checked():
    torch = pytest.importorskip("torch")
    ctx = SimpleNamespace(h=SimpleNamespace(value=BASE), device=-1)

    def i(*size):
        return torch.zeros(size, dtype=torch.int32)

    take = dict(cu=i(5), parent=i(2), words=i(2), picks=i(2), held=i(4), length=i(4), path=i(2), count=i(4), next=i(4), length_out=i(4))
    for bad, error in [(dict(pos=i(3)), ValueError), (dict(pos=torch.zeros(2)), TypeError), (dict(pos=i(2, 1)), ValueError), (dict(pos=i(4)[::2]), ValueError)]:
        with pytest.raises(error):
            nunchi_amd.tree_take(ctx, **{**take, **bad})
