"""Argument checks of pages, rotary positions, kept rows and trees in the C ABI, which run before any device call."""
import ctypes

import pytest
from test_operators_host import P, _pool, _status


# The pool comes first.
ATTEND = [None, P, P, None, 3, 40, 3, P, 256, 64, 4, 0, 0.125, 1, 0, None, 0, 0, 0, None, P, 256, 64, None, P, 1 << 40,
          None]
KEEP = [None, P, P, None, 3, 2, 3, P, 4, P, None]


def _cache_status(call, defaults, change):
    pool = _pool()
    args = [ctypes.addressof(pool), *defaults[1:]]
    for i, v in change.items():
        args[i] = v
    return _status(call, *args)


@pytest.mark.parametrize("change,status,text", [
    ({18: -1}, 1, "sinks"), ({13: 0, 19: P}, 1, "causal"), ({10: 3}, 1, "multiple of kv_heads"),
    ({14: -1}, 1, "window"), ({20: None}, 1, "out"), ({24: None}, 1, "workspace"), ({25: 16}, 1, "workspace"),
])
def test_attend_checks(change, status, text):
    got = _cache_status("msim_kv4_attend_ex_async", ATTEND, change)
    assert got[0] == status and text in got[1]


@pytest.mark.parametrize("change,status,text", [
    ({4: -1}, 1, "negative"), ({1: None}, 1, "page_table"), ({8: -1}, 1, "width"), ({8: (1 << 26) + 1}, 3, "2^20"),
    ({4: (1 << 20) + 1, 6: (1 << 20) + 1}, 3, "2^20"), ({7: None}, 1, "kept"), ({9: None}, 1, "kept"),
    ({6: 4}, 1, "one row per"), ({5: 1 << 28}, 3, "2^31"),
])
def test_keep_checks(change, status, text):
    got = _cache_status("msim_kv4_keep_async", KEEP, change)
    assert got[0] == status and text in got[1]


@pytest.mark.parametrize("change,status,text", [
    ({7: 24}, 1, "page_size"), ({7: 8}, 1, "page_size"), ({7: 1 << 17}, 1, "page_size"), ({6: 0}, 1, "num_pages"),
    ({6: 1 << 31}, 1, "num_pages"), ({4: -1}, 1, "negative"), ({10: -1}, 1, "negative"), ({10: 1 << 27}, 3, "2^26"),
    ({5: 1 << 27}, 3, "2^31"), ({4: 1 << 20, 5: 1 << 12}, 3, "2^31"), ({0: None}, 1, "NULL"), ({1: None}, 1, "NULL"),
    ({2: None}, 1, "NULL"), ({3: None}, 1, "NULL"), ({11: None}, 1, "NULL"), ({12: None}, 1, "NULL"),
    ({13: None}, 1, "NULL"),
])
def test_pages_checks(change, status, text):
    args = [P, P, P, P, 3, 5, 100, 16, None, None, 7, P, P, P, None]
    for i, v in change.items():
        args[i] = v
    got = _status("msim_pages_update_async", *args)
    assert got[0] == status and text in got[1]


ROTARY = [P, P, 32, 64, 1, 0, P, 0, 3, 0, P, 256, 64, 4, P, 256, 64, P, 128, 64, 2, P, 128, 64, None]


@pytest.mark.parametrize("change,status,text", [
    ({9: 3}, 1, "type"), ({2: 0}, 1, "rotary dims"), ({2: 33}, 1, "rotary dims"), ({3: 258}, 3, "256"),
    ({4: 0}, 1, "axes"), ({4: 33}, 1, "axes"), ({8: -1}, 1, "negative"), ({13: -1}, 1, "negative"),
    ({20: -1}, 1, "negative"), ({8: (1 << 25) + 1}, 3, "2^25"), ({13: 1 << 17}, 3, "2^16"), ({0: None}, 1, "NULL"),
    ({1: None}, 1, "NULL"), ({6: None}, 1, "NULL"), ({10: None}, 1, "NULL"), ({14: None}, 1, "NULL"),
    ({17: None}, 1, "NULL"), ({21: None}, 1, "NULL"), ({10: P + 2}, 1, "aligned"), ({21: P + 1}, 1, "aligned"),
])
def test_rotary_checks(change, status, text):
    args = list(ROTARY)
    for i, v in change.items():
        args[i] = v
    got = _status("msim_rotary_async", *args)
    assert got[0] == status and text in got[1]


def test_calls_of_no_rows_do_nothing():
    pool = _pool()
    args = [ctypes.addressof(pool), None, None, None, 0, 0, 0, None, 4, None, None]
    assert _status("msim_kv4_keep_async", *args)[0] == 0
    args = list(ROTARY)
    args[8] = 0
    assert _status("msim_rotary_async", *args)[0] == 0
    args[8], args[13], args[20] = 3, 0, 0
    assert _status("msim_rotary_async", *args)[0] == 0
