"""What calls on tensors take as arguments."""
import numpy as np
import pytest
import torch
from test_gpu_pages import Lists

from maxsim_amd import CachePages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("number", [9, np.int64(9), np.int32(9), np.uint8(9), np.array([4, 9]).max()])
def test_numbers_of_tokens(gpu, number):
    pages, lists = CachePages(50, 6, 5, page_size=16), Lists(50, 6, 5, 16)
    for rows in (None, 54, np.int64(60)):
        got = pages.update(number, rows=rows)
        want = lists.update([9] * 6, None, 54 if rows is None else int(rows))
        assert all(g.tolist() == w for g, w in zip(got, want))
    lists.check(pages)
    with pytest.raises(ValueError):
        pages.update(-number if not isinstance(number, np.unsignedinteger) else np.int64(-9))
    lists.check(pages)
