"""Trees of drafted tokens whose positions lie far from their keys', and the bounds that
windows with sinks and trees share with the other calls over the cache."""
import ctypes
import math

import pytest
import torch
from test_gpu_drafts import _check, _seen, _tree
from test_gpu_kvcache import BF16, F16, Batch, _fill, _pool, _queries, _rng

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


# --------------------------------------------------- product by product


def _check_by_products(cache, batch, q, got, got_lse, parents=None, **kw):
    """16-bit queries are taken whole, so a score is exact products added in single precision
    (a quarter of the dims, and four roundings of factors); a probability times its value
    scale keeps 2^-16.  Every result is the rounding of one within that of the expected."""
    dim, share = cache.head_dim, q.shape[1] // cache.kv_heads
    pool = _pool(cache)
    got, got_lse = got.cpu(), got_lse.cpu().double()
    for b, (n, m) in enumerate(zip(batch.host_lengths, batch.new)):
        rows, key = slice(int(batch.host_offsets[b]), int(batch.host_offsets[b]) + m), torch.arange(n)
        k, v = (x[batch.host_table[b].long()[key // cache.page_size], :, key % cache.page_size].transpose(0, 1)
                .repeat_interleave(share, 0) for x in pool)
        see = _seen(n, m, parents=None if parents is None else parents[rows].tolist(), **kw)
        qs = q[rows].cpu().double().transpose(0, 1)
        s = (qs @ k.transpose(1, 2) * dim**-0.5).masked_fill(~see, -math.inf)
        p = torch.softmax(s, -1)
        out, mass = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
        most = (qs.abs() @ k.abs().transpose(1, 2) * dim**-0.5).masked_fill(~see, 0).amax(-1).t()
        delta, sums = 2.0**-24 * (dim / 4 + 4) * most + 2.0**-23, 2.0**-24 * (n / 8 + 16)
        tol = (2.0**-16 + 2 * delta[..., None] + 2 * sums) * mass + 1e-30
        off = ~(((out - tol).to(q.dtype) <= got[rows]) & (got[rows] <= (out + tol).to(q.dtype)))
        assert not bool(off.any()), (b, int(off.sum()), float(((got[rows].double() - out).abs() / tol)[off].max()))
        lse = torch.logsumexp(s, -1).t()
        assert bool(((got_lse[rows] - lse).abs() <= delta + sums + 2.0**-22 * (1 + lse.abs())).all())


def _peaked(rows, heads, dim, kind, seed):
    """Queries whose rows have few large probabilities, or many small ones."""
    return _queries(rows, heads, dim, kind, seed, size=2.0) * (0.25 + torch.arange(heads, device="cuda") % 3)[:, None].to(kind)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (96, 64), (128, 16), (192, 32), (256, 64)])
@pytest.mark.parametrize("batch,lo,hi,new,kv_heads,share,window,sinks", [
    (32, 700, 1500, 1, 4, 4, 700, 40),    # whole items, all the waves of a CU, tiles of 16 rows
    (12, 700, 1500, 16, 8, 4, 1000, 8),   # the same, of 32 rows
    (70, 300, 800, 2, 2, 3, 330, 20),     # whole items, four waves
    (2, 2500, 4000, 3, 2, 4, 1500, 300),  # split items of 16 rows
    (3, 2500, 4000, 12, 1, 4, 1500, 5),   # and of 32
    (2, 600, 900, 270, 1, 4, 400, 33)])   # tiles of 256
def test_sinks_by_products(gpu, kind, dim, page, batch, lo, hi, new, kv_heads, share, window, sinks):
    lengths = torch.randint(lo, hi, (batch,), generator=_rng(dim)).tolist()
    cache = Int4KVCache(sum(-(-n // page) for n in lengths), kv_heads, dim, page_size=page)
    _fill(cache, 8)
    rows = Batch(cache, lengths, [new] * batch, seed=3)
    q = _peaked(rows.rows, kv_heads * share, dim, kind, 3)
    got, lse = cache.attend(q, *rows.args, window=window, sinks=sinks, return_lse=True)
    _check_by_products(cache, rows, q, got, lse, window=window, sinks=sinks)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (96, 64), (128, 16), (192, 32), (256, 64)])
@pytest.mark.parametrize("batch,lo,hi,new,kv_heads,share,spare", [
    (8, 700, 1000, 8, 8, 4, 0),       # whole items, all the waves of a CU, tiles of 16 rows
    (12, 700, 1000, 16, 8, 4, 0),     # the same, of 32 rows
    (70, 300, 500, 5, 2, 3, 0),       # whole items, four waves
    (2, 700, 900, 8, 2, 4, 0),        # split items of 16 rows
    (3, 2500, 4000, 24, 2, 4, 0),     # and of 32
    (4, 200, 900, 64, 2, 4, 30000)])  # tiles of 256, where the table is wide
@pytest.mark.parametrize("window,sinks", [(None, None), (150, 70)])
def test_trees_by_products(gpu, kind, dim, page, batch, lo, hi, new, kv_heads, share, spare, window, sinks):
    lengths = torch.randint(lo, hi, (batch,), generator=_rng(dim)).tolist()
    cache = Int4KVCache(sum(-(-n // page) for n in lengths), kv_heads, dim, page_size=page)
    _fill(cache, 8)
    rows = Batch(cache, lengths, [new] * batch, seed=3, spare=spare // page)
    parents = _tree(rows.new, 5, lean=0.6)
    q = _peaked(rows.rows, kv_heads * share, dim, kind, 3)
    got, lse = cache.attend(q, *rows.args, parents=parents.cuda(), window=window, sinks=sinks, return_lse=True)
    _check_by_products(cache, rows, q, got, lse, parents=parents, window=window, sinks=sinks)
