"""Allocations of calls on tensors, as dispatch modes and the profiler see them."""
import pytest
import torch
from test_gpu_kvcache import BF16, Batch, _fill, _queries
from torch.utils._python_dispatch import TorchDispatchMode

from maxsim_amd import CachePages, Int4KVCache, Int4Linear, Rotary

pytestmark = pytest.mark.gpu


class _Allocations(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.shapes = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if func is torch.ops.aten.empty.memory_format:
            self.shapes.append(tuple(out.shape))
        return out


def _calls():
    """Each call that allocates its outputs, and their shapes."""
    cache = Int4KVCache(40, 2, 64, page_size=16)
    _fill(cache, 3)
    batch = Batch(cache, [100, 20], [3, 2], seed=1)
    pages, rotary = CachePages(40, 2, 12, page_size=16), Rotary(64)
    linear = Int4Linear.from_float(torch.ones((32, 64), device="cuda"), 32)
    q, at = _queries(5, 4, 64, BF16, 2), torch.arange(5, dtype=torch.int32, device="cuda")
    kept, new = torch.zeros((2, 1), dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    return [(lambda: cache.attend(q, *batch.args, return_lse=True), [(5, 4, 64), (5, 4)]),
            (lambda: cache.read(*batch.args, rows=5), [(5, 2, 64)] * 2),
            (lambda: cache.keep(*batch.args, kept), [(2,)]),
            (lambda: pages.update(new, rows=7), [(3,), (7,), (7,)]),
            (lambda: rotary(q, q[:, :2], at), [(5, 4, 64), (5, 2, 64)]),
            (lambda: linear(q[:, 0]), [(5, 32)])]


def test_modes_see_the_outputs(gpu):
    for call, shapes in _calls():
        call()
        with _Allocations() as seen:
            call()
        assert [s for s in seen.shapes if s in shapes] == shapes


def test_the_profiler_sees_the_outputs(gpu):
    for call, shapes in _calls():
        call()
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
            call()
        assert sum(e.count for e in prof.key_averages() if e.key == "aten::empty") >= len(shapes)
