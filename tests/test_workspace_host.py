"""How much memory attention over the cache asks for, which is a matter of sizes alone."""
import ctypes

import pytest
from test_operators_host import P, _pool, _status


def _bytes(call, pool, *sizes):
    need = ctypes.c_uint64(0)
    status, text = _status(call, ctypes.addressof(pool), *sizes, ctypes.byref(need))
    assert status == 0, text
    return need.value


def _plain(pool, batch, tokens, rows, heads):
    return _bytes("msim_kv4_attend_workspace", pool, batch, tokens // pool.page_size, rows, heads)


def _tree(pool, batch, tokens, rows, heads, parents=1):
    return _bytes("msim_kv4_attend_ex_workspace", pool, batch, tokens // pool.page_size, rows, heads, parents)


@pytest.mark.parametrize("batch,rows", [(4, 256), (1, 64), (2, 128), (8, 512)])
def test_calls_without_parents_need_nothing_of_trees(batch, rows):
    """Some trees of these sizes go in tiles of 256 rows over wide tables. Other calls do not."""
    pool = _pool(kv_heads=8, dim=128)
    narrow = _plain(pool, batch, 1024, rows, 32)
    for tokens in (6144, 131072, 2**30):
        assert _plain(pool, batch, tokens, rows, 32) == narrow
        assert _tree(pool, batch, tokens, rows, 32, parents=0) == narrow
    assert narrow < 20e6
    assert _tree(pool, batch, 131072, rows, 32) > 3 * narrow
    assert _tree(pool, batch, 1024, rows, 32) == narrow
    assert _tree(pool, batch, 512, rows, 32) == _plain(pool, batch, 512, rows, 32) == 0


@pytest.mark.parametrize("tokens", [1024, 131072])
@pytest.mark.parametrize("batch,rows,heads", [(4, 256, 8), (5, 5 * 1024, 8), (3, 9, 2)])
def test_less_than_a_tree_needs(tokens, batch, rows, heads):
    """The lesser of what a tree and another call of its sizes use is what a tree must have."""
    pool = _pool()
    pages, least = tokens // 16, min(_plain(pool, batch, tokens, rows, heads), _tree(pool, batch, tokens, rows, heads))
    for bytes_ in (0, 16, least - 1):
        args = [P, P, P, batch, pages, rows, P, 256, 64, heads, 0, 0.125, 1, 0, None, 0, 0, 0, P, P, 256, 64, None, P,
                bytes_, None]
        got = _status("msim_kv4_attend_ex_async", ctypes.addressof(pool), *args)
        assert got[0] == 1 and "workspace" in got[1]
