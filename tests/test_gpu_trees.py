"""Trees of drafted tokens whose positions lie far from their keys', and the bounds that
windows with sinks and trees share with the other calls over the cache."""
import ctypes

import pytest
import torch
from test_gpu_drafts import _check, _tree
from test_gpu_kvcache import BF16, F16, Batch, _fill, _queries

from maxsim_amd import Int4KVCache, _native

pytestmark = pytest.mark.gpu


# ------------------------------------- drafts that only the sinks leave visible
#
# Under a window a row sees those it comes after by their depth. Where the context is
# shorter than the sinks, some of the rows themselves are first tokens: a chain behind many
# siblings has them at keys far past the sinks, and below every key of the window.


def _late_chain(siblings, rows):
    """Siblings after the context, then a chain from the last of them."""
    return [-1] * siblings + list(range(siblings - 1, rows - 1))


def _late_branch(early, siblings, rows):
    """A chain, siblings after its fourth row, and a chain from the last of those."""
    return [*range(-1, early - 1), *[3] * siblings, *range(early + siblings - 1, rows - 1)]


# A wide table sends these trees through the kernel for prompts, a narrow one through the other.
@pytest.mark.parametrize("spare", [0, 600])
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("start,window,sinks", [(0, 4, 10), (5, 4, 12), (0, 1, 300), (100, 30, 140), (300, 40, 310),
                                                (300, 40, 299)])
def test_first_tokens_among_the_drafts(gpu, spare, kind, start, window, sinks):
    cache = Int4KVCache(200, 2, 64, page_size=16)
    _fill(cache, start)
    parents = [_late_chain(201, 1024), _late_branch(100, 300, 640)]
    new = [len(p) for p in parents]
    batch = Batch(cache, [start + n for n in new], new, seed=1, spare=spare)
    parents = torch.tensor(sum(parents, []), dtype=torch.int32)
    q = _queries(batch.rows, 8, 64, kind, 3)
    got, lse = cache.attend(q, *batch.args, parents=parents.cuda(), window=window, sinks=sinks, return_lse=True)
    _check(cache, batch, q, got, lse, parents=parents, window=window, sinks=sinks)


# ------------------------------------------------------------------ workspaces


def test_memory_of_a_causal_call(gpu):
    """A call without parents allocates nothing of what trees of its sizes would use."""
    cache = Int4KVCache(64, 8, 128, page_size=64)
    batch = Batch(cache, [1000, 500, 700, 300], [64] * 4, seed=1, spare=2000)
    q = _queries(batch.rows, 32, 128, BF16, 3)
    out = torch.empty_like(q)
    cache.attend(q, *batch.args, out=out)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    cache.attend(q, *batch.args, out=out)
    assert torch.cuda.max_memory_allocated() - before < 20e6


@pytest.mark.parametrize("sinks", [0, 20])
def test_trees_in_the_workspace_of_other_calls(gpu, sinks):
    """The C call takes a workspace that holds no tiles of 256 rows, and one that does."""
    cache = Int4KVCache(160, 2, 64, page_size=16)
    _fill(cache, 5)
    new = [64] * 4
    batch = Batch(cache, [900, 64, 300, 131], new, seed=1, spare=2000)
    parents = _tree(new, 3)
    q, out = _queries(batch.rows, 8, 64, BF16, 3), torch.empty((batch.rows, 8, 64), dtype=BF16, device="cuda")
    lse, device_parents = torch.empty((batch.rows, 8), device="cuda"), parents.cuda()
    pool = _native.Kv4Pool(cache.k_codes.data_ptr(), cache.k_scales.data_ptr(), cache.v_codes.data_ptr(),
                           cache.v_scales.data_ptr(), 160, 2, 16, 64)
    sizes, need = (4, batch.table.shape[1], batch.rows), []
    for call, more in (("msim_kv4_attend_workspace", ()), ("msim_kv4_attend_ex_workspace", (1,))):
        size = ctypes.c_uint64(0)
        assert getattr(gpu, call)(ctypes.addressof(pool), *sizes, 8, *more, ctypes.byref(size)) == 0
        need.append(size.value)
    assert 0 < need[0] < need[1]
    window = 50 if sinks else 0
    for bytes_ in (*need, need[1] - 1, need[0] + 1):
        work = torch.full((bytes_ + 4096,), 77, dtype=torch.uint8, device="cuda")
        assert gpu.msim_kv4_attend_ex_async(
            ctypes.addressof(pool), batch.table.data_ptr(), batch.lengths.data_ptr(), batch.offsets.data_ptr(), *sizes,
            q.data_ptr(), 512, 64, 8, 2, 0.125, 1, window, None, 0, 0, sinks, device_parents.data_ptr(), out.data_ptr(),
            512, 64, lse.data_ptr(), work.data_ptr(), bytes_, torch.cuda.current_stream().cuda_stream) == 0
        _check(cache, batch, q, out, lse, parents=parents, window=window or None, sinks=sinks)
        assert bool((work[bytes_:] == 77).all())
