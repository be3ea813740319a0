"""Argument checks of the cache's and the 4-bit products' C ABI, which run before any device call."""
import ctypes

import pytest

from maxsim_amd import _native

P = 4096  # stands for a device address: never read


def _pool(**kw):
    fields = {"k_codes": P, "k_scales": P, "v_codes": P, "v_scales": P, "num_pages": 4, "kv_heads": 2,
              "page_size": 16, "dim": 64, **kw}
    return _native.Kv4Pool(*(fields[name] for name, _ in _native.Kv4Pool._fields_))


def _status(call, *args):
    lib = _native.load()
    return getattr(lib, call)(*args), lib.msim_last_error().decode()


@pytest.mark.parametrize("kw,status,text", [
    ({"dim": 80}, 3, "head_dim"), ({"page_size": 24}, 1, "page_size"), ({"page_size": 8}, 1, "page_size"),
    ({"num_pages": 0}, 1, "num_pages"), ({"kv_heads": 0}, 1, "kv_heads"), ({"k_codes": None}, 1, "NULL"),
    ({"v_scales": P + 4}, 1, "aligned"),
])
def test_pool_checks(kw, status, text):
    pool = _pool(**kw)
    args = [P, P, None, 3, 2, 3, P, 128, 64, P, 128, 64, 0, None]
    got = _status("msim_kv4_append_async", ctypes.addressof(pool), *args)
    assert got[0] == status and text in got[1]
    got = _status("msim_kv4_read_async", ctypes.addressof(pool), *args)
    assert got[0] == status and text in got[1]


@pytest.mark.parametrize("change,status,text", [
    ({0: None}, 1, "page_table"), ({1: None}, 1, "lengths"), ({3: -1}, 1, "negative"), ({5: 4}, 1, "one row per"),
    ({4: 1 << 28}, 3, "2^31"), ({3: 1 << 27, 5: 1 << 27}, 3, "2^26"), ({6: None}, 1, "k must"), ({9: P + 1}, 1, "v must"),
    ({12: 3}, 1, "type"),
])
def test_batch_checks(change, status, text):
    pool = _pool()
    args = [P, P, None, 3, 2, 3, P, 128, 64, P, 128, 64, 0, None]
    for i, v in change.items():
        args[i] = v
    got = _status("msim_kv4_append_async", ctypes.addressof(pool), *args)
    assert got[0] == status and text in got[1]


@pytest.mark.parametrize("change,status,text", [
    ({9: 3}, 1, "multiple of kv_heads"), ({9: 0}, 1, "multiple of kv_heads"), ({11: float("nan")}, 1, "scale"),
    ({13: -1}, 1, "window"), ({14: P, 16: -1}, 1, "mask"), ({17: None}, 1, "out"), ({21: None}, 1, "workspace"),
    ({22: 16}, 1, "workspace"), ({6: None}, 1, "q must"),
])
def test_attend_checks(change, status, text):
    pool = _pool()
    args = [P, P, None, 3, 40, 3, P, 256, 64, 4, 0, 0.125, 1, 0, None, 0, 0, P, 256, 64, None, P, 1 << 40, None]
    for i, v in change.items():
        args[i] = v
    got = _status("msim_kv4_attend_async", ctypes.addressof(pool), *args)
    assert got[0] == status and text in got[1]


def test_key_positions_stay_within_32_bits():
    """Kernels look past a sequence's end: a table whose last keys' successors pass 2^31 is refused."""
    for page_size, most in ((16, (2**31 - 4097) // 16), (4096, 2**19 - 2), (65536, 2**15 - 1)):
        pool = _pool(page_size=page_size)
        need = ctypes.c_uint64(0)
        for pages, status in ((most, 0), (most + 1, 3)):
            got = _status("msim_kv4_attend_workspace", ctypes.addressof(pool), 1, pages, 1, 4, ctypes.byref(need))
            assert got[0] == status and (status == 0 or "2^31" in got[1])
            args = [P, P, None, 0, pages, 0, P, 128, 64, P, 128, 64, 0, None]
            assert _status("msim_kv4_append_async", ctypes.addressof(pool), *args)[0] == status


@pytest.mark.parametrize("scale,status", [(1e300, 1), (2.5e38, 1), (-1e39, 1), (float("inf"), 1), (2.3e38, 0), (0.0, 0)])
def test_scales_that_single_precision_has_not(scale, status):
    args = [None, None, None, 0, 0, 0, None, 0, 0, 4, 0, scale, 1, 0, None, 0, 0, None, 0, 0, None, None, 0, None]
    pool = _pool()
    got = _status("msim_kv4_attend_async", ctypes.addressof(pool), *args)
    assert got[0] == status and (status == 0 or "scale" in got[1])


def test_calls_of_no_rows_do_nothing():
    pool = _pool()
    assert _status("msim_kv4_append_async", ctypes.addressof(pool), None, None, None, 0, 0, 0, None, 0, 0, None, 0, 0, 0,
                   None)[0] == 0
    assert _status("msim_kv4_attend_async", ctypes.addressof(pool), None, None, None, 0, 0, 0, None, 0, 0, 4, 0, 1.0, 1,
                   0, None, 0, 0, None, 0, 0, None, None, 0, None)[0] == 0
    assert _status("msim_linear4_async", P, P, 16, 128, 32, None, None, 0, 128, 0, None, 16, None)[0] == 0


def test_layout_sizes_and_checks():
    codes, scales = ctypes.c_uint64(0), ctypes.c_uint64(0)
    out = ctypes.byref(codes), ctypes.byref(scales)
    assert _status("msim_linear4_layout_bytes", 17, 160, 32, *out)[0] == 0
    assert codes.value == 2 * 2 * 1024 and scales.value == 2 * 2 * 16 * 4 * 2
    for n, k, group, text in ((0, 128, 32, "rows"), (4, 100, 32, "multiple"), (4, 128, 48, "group_size"),
                              (4, 0, 32, "rows")):
        got = _status("msim_linear4_layout_bytes", n, k, group, *out)
        assert got[0] == 1 and text in got[1]
    assert _status("msim_linear4_layout_bytes", 1 << 25, 128, 32, *out)[0] == 3
    assert _status("msim_linear4_layout_async", P + 2, P, 4, 128, 32, P, P, None)[0] == 1
    base = [P, P, 16, 128, 32, None, P, 2, 128, 0, P, 16, None]
    for i, v, status in ((9, 5, 1), (7, -1, 1), (7, 1 << 21, 3), (0, P + 8, 1), (6, None, 1), (10, P + 2, 1)):
        args = list(base)
        args[i] = v
        assert _status("msim_linear4_async", *args)[0] == status
