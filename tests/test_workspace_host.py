"""How much memory attention over the cache asks for, which is a matter of sizes alone."""
import ctypes

import pytest
from test_operators_host import P, _pool, _status

from maxsim_amd import _native


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


class _Pool(ctypes.Structure):
    """csrc/kv4.hpp's Kv4Pool."""

    _fields_ = [("arrays", ctypes.c_void_p * 4), ("num_pages", ctypes.c_int32), ("page_shift", ctypes.c_int32),
                ("kv_heads", ctypes.c_int32), ("dim", ctypes.c_int32)]


class _Batch(ctypes.Structure):
    """Its Kv4Batch."""

    _fields_ = [("table", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("offsets", ctypes.c_void_p),
                ("batch", ctypes.c_int32), ("max_pages", ctypes.c_int32), ("rows", ctypes.c_int32)]


def _slots(cus, batch, pages, rows, parents):
    """Rows of partial results in the library's own answer for a device of `cus` CUs: 32 heads of 128 on
    8, pages of 16."""
    call = getattr(_native.load(), "_ZN4msim20kv4_attend_workspaceERKNS_7Kv4PoolERKNS_8Kv4BatchEibi")
    call.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_bool, ctypes.c_int]
    call.restype = ctypes.c_size_t
    pool = _Pool((ctypes.c_void_p * 4)(), 4, 4, 8, 128)
    sizes = _Batch(P, P, P, batch, pages, rows)
    return call(ctypes.addressof(pool), ctypes.addressof(sizes), 32, parents, cus) // (130 * 4)


@pytest.mark.parametrize("cus", [32, 64, 256, 304])
def test_tiles_of_256_rows_by_the_number_of_cus(cus):
    """A workgroup of them for each CU, in two slots; smaller tiles have less than half of that."""
    large = 2 * 256 * cus
    # Trees: 4 x 64 rows with six granules of 128 keys for each CU, and fewer.
    pages = 6 * 128 * cus // (4 * 8) // 16
    assert _slots(cus, 4, pages, 256, True) >= large
    assert _slots(cus, 4, pages - 1, 256, True) < large // 2
    # Other calls: one tile a sequence and head, for half the CUs, and for fewer.
    assert _slots(cus, cus // 16, 1000, cus // 16 * 64, False) >= large
    if cus > 32:
        assert _slots(cus, cus // 32, 1000, cus // 32 * 64, False) < large // 2
