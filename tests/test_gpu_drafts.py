"""Windows with first tokens that stay visible, trees of drafted tokens, and the rows
of a tree that are kept, against plain float64 computations from the stored codes."""
import math

import pytest
import torch
from test_gpu_kvcache import BF16, F16, F32, ROUND, Batch, _fill, _pool, _queries, _rng

from maxsim_amd import CachePages, Int4KVCache, Int4Linear, Rotary

pytestmark = pytest.mark.gpu


def _seen(n, m, causal=True, window=None, sinks=None, parents=None, mask=None):
    """Which of a sequence's n keys its m rows see: bool [m, n], by the definition."""
    see = torch.zeros((m, n), dtype=torch.bool)
    start = n - m
    for i in range(m):
        if parents is None:
            at, own = start + i, None
            keys = {j: j for j in range(n) if not causal or j <= at}
        else:
            line = [i]
            while 0 <= int(parents[line[-1]]) < line[-1]:
                line.append(int(parents[line[-1]]))
            at = start + len(line) - 1
            keys = {j: j for j in range(start)}
            keys.update({start + row: at - back for back, row in enumerate(line)})
            if m > 1024:
                keys = {}
        for j, position in keys.items():
            if j < 0 or (window is not None and position <= at - window and not position < (sinks or 0)):
                continue
            see[i, j] = mask is None or (j < mask.shape[1] and bool(mask[i, j]))
    return see


def _check(cache, batch, q, got, got_lse=None, scale=None, parents=None, mask=None, **kw):
    """Against float64, with the bounds that the cache's other calls have: a score is dim
    products summed in single precision and two more roundings (queries in single
    precision keep 22 bits of their largest entry), a probability times its value scale
    keeps 16 bits (24 in single precision calls), sums are single precision."""
    kind, dim = q.dtype, cache.head_dim
    heads = q.shape[1]
    share = heads // cache.kv_heads
    scale = dim**-0.5 if scale is None else scale
    pool = _pool(cache)
    q, got = q.cpu().double(), got.cpu()
    done = torch.zeros(q.shape[0], dtype=torch.bool)
    for b, (n, m) in enumerate(zip(batch.host_lengths, batch.new)):
        if m == 0:
            continue
        rows = slice(int(batch.host_offsets[b]), int(batch.host_offsets[b]) + m)
        done[rows] = True
        key = torch.arange(n)
        page = batch.host_table[b].long()[key // cache.page_size]
        hole = (page < 0) | (page >= cache.num_pages)
        k, v = (x[page.clamp(0, cache.num_pages - 1), :, key % cache.page_size].transpose(0, 1) for x in pool)
        see = _seen(n, m, parents=None if parents is None else parents[rows].tolist(),
                    mask=None if mask is None else mask[rows].cpu(), **kw) & ~hole
        some = see.any(1)
        k, v = k.repeat_interleave(share, 0), v.repeat_interleave(share, 0)  # [heads, n, dim]
        qs = q[rows].transpose(0, 1)
        s = (qs @ k.transpose(1, 2)) * scale
        s = s.masked_fill(~see, -math.inf)
        top = s.amax(-1, keepdim=True).clamp(min=-1e300)
        p = torch.exp(s - top)
        total = p.sum(-1, keepdim=True)
        p = p / total.clamp(min=1e-300)
        out, mass = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
        sums = (qs.abs() @ k.abs().transpose(1, 2)).masked_fill(~see, 0).amax(-1) * abs(scale)
        part = qs.abs().amax(-1) * k.abs().sum(-1).masked_fill(hole, 0).amax(-1, keepdim=True) * abs(scale) * 2.0**-23
        delta = (2.0**-24 * (dim / 4 + 4) * sums + part + 2.0**-23).transpose(0, 1)
        many = 2.0**-24 * (n / 8 + 16)
        probs = 2.0**-21 if kind == F32 else 2.0**-11
        tol = ROUND[kind] * out.abs() + (probs + 2 * delta[..., None] + 2 * many) * mass + 1e-30
        if kind == F16:
            tol = tol + 2.0**-25
        diff = (got[rows].double() - out).abs()
        assert bool((diff <= tol).all()), float((diff / tol).max())
        assert not bool(got[rows][~some].any())
        if got_lse is not None:
            lse = (top + torch.log(total)).squeeze(-1).transpose(0, 1)
            seen_lse = got_lse.cpu()[rows]
            assert bool((seen_lse[~some] == -math.inf).all())
            diff = (seen_lse.double() - lse).abs()[some]
            assert bool((diff <= (delta + many + 2.0**-22 * (1 + lse.abs()))[some]).all())
    assert not bool(got[~done].any())


def _tree(sizes, seed, lean=1.5):
    """Parents: rows lean towards the first ones."""
    g = _rng(seed)
    return torch.cat([torch.empty(0), *((torch.arange(n) * torch.rand(n, generator=g) ** lean).floor() - 1
                                        for n in sizes)]).to(torch.int32)


# ------------------------------------------------------------------ sinks


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (96, 64), (128, 16), (192, 32), (256, 128)])
@pytest.mark.parametrize("window,sinks", [(1, 1), (40, 4), (33, 32), (16, 70), (500, 3), (64, 2**40)])
def test_windows_with_sinks(gpu, kind, dim, page, window, sinks):
    cache = Int4KVCache(90, 2, dim, page_size=page)
    _fill(cache, page)
    batch = Batch(cache, [275, 64, 0, 230, 5, 33, 1], [20, 1, 0, 37, 5, 2, 1], seed=1)
    q = _queries(batch.rows, 6, dim, kind, 3)
    got, lse = cache.attend(q, *batch.args, window=window, sinks=sinks, return_lse=True)
    _check(cache, batch, q, got, lse, window=window, sinks=sinks)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("window,sinks", [(1, 1), (100, 5), (257, 96), (31, 300), (1000, 4)])
def test_windows_with_sinks_at_prompts(gpu, kind, dim, window, sinks):
    cache = Int4KVCache(140, 2, dim, page_size=16)
    _fill(cache, dim)
    batch = Batch(cache, [700, 301, 0, 640], [300, 301, 0, 290], seed=1)
    q = _queries(batch.rows, 8, dim, kind, 3)
    got, lse = cache.attend(q, *batch.args, window=window, sinks=sinks, return_lse=True)
    _check(cache, batch, q, got, lse, window=window, sinks=sinks)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_long_contexts_with_sinks(gpu, kind, new):
    """Split items, and what lies between the sinks and the window in holes."""
    cache = Int4KVCache(700, 2, 64, page_size=16)
    _fill(cache, 3)
    batch = Batch(cache, [5003, 4000, 1700], [new] * 3, seed=2)
    for b, (n, first) in enumerate(((5003, 80), (4000, 80), (1700, 80))):
        batch.host_table[b, first // 16:(n - new - 700) // 16] = -1
    batch.table = batch.host_table.cuda()
    q = _queries(batch.rows, 8, 64, kind, 3)
    for window, sinks in ((700, 77), (33, 1), (640, 80)):
        got, lse = cache.attend(q, *batch.args, window=window, sinks=sinks, return_lse=True)
        _check(cache, batch, q, got, lse, window=window, sinks=sinks)


@pytest.mark.parametrize("new", [1, 6, 300])
def test_windows_and_sinks_as_masks(gpu, new):
    """A window, sinks, a mask and calls without causality together; sinks without a window say nothing."""
    cache = Int4KVCache(80, 2, 128, page_size=16)
    _fill(cache, 3)
    batch = Batch(cache, [400, 390, 310], [new] * 3, seed=2)
    q = _queries(batch.rows, 8, 128, BF16, 3)
    mask = (torch.rand((batch.rows, 395), generator=_rng(4)) < 0.6).cuda()
    mask[::7] = False
    for causal in (True, False):
        got, lse = cache.attend(q, *batch.args, causal=causal, window=50, sinks=9, mask=mask, return_lse=True)
        _check(cache, batch, q, got, lse, causal=causal, window=50, sinks=9, mask=mask)
    assert torch.equal(cache.attend(q, *batch.args, sinks=5), cache.attend(q, *batch.args))
    assert torch.equal(cache.attend(q, *batch.args, window=60, sinks=0), cache.attend(q, *batch.args, window=60))


@pytest.mark.parametrize("new", [2, 300])
def test_keys_between_sinks_and_window_have_no_effect(gpu, new):
    cache = Int4KVCache(80, 2, 128, page_size=16)
    _fill(cache, 3)
    batch = Batch(cache, [600, 490], [new] * 2, seed=2)
    q = _queries(batch.rows, 8, 128, BF16, 3)
    clean = cache.attend(q, *batch.args, window=90, sinks=37)
    for b, n in enumerate(batch.host_lengths):
        for j in range(37, n - new - 89):
            for scales in (cache.k_scales, cache.v_scales):
                scales[int(batch.host_table[b, j // 16]), :, j % 16] = math.nan
    assert torch.equal(cache.attend(q, *batch.args, window=90, sinks=37), clean)


# ------------------------------------------------------------------ trees


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (96, 64), (128, 16), (192, 32), (256, 128)])
@pytest.mark.parametrize("kv_heads,share", [(1, 1), (2, 4), (3, 5)])
def test_trees(gpu, kind, dim, page, kv_heads, share):
    cache = Int4KVCache(60, kv_heads, dim, page_size=page)
    _fill(cache, page)
    lengths, new = [275, 64, 0, 130, 5, 33, 1, 31], [20, 1, 0, 70, 5, 2, 1, 31]
    batch = Batch(cache, lengths, new, seed=1)
    parents = _tree(new, dim)
    q = _queries(batch.rows, kv_heads * share, dim, kind, 3)
    got, lse = cache.attend(q, *batch.args, parents=parents.cuda(), return_lse=True)
    _check(cache, batch, q, got, lse, parents=parents)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("window,sinks", [(1, None), (3, 2), (40, 4), (5, 130), (200, 129)])
def test_trees_under_windows_and_masks(gpu, kind, window, sinks):
    cache = Int4KVCache(60, 2, 64, page_size=16)
    _fill(cache, 5)
    new = [30, 12, 9, 40]
    batch = Batch(cache, [128 + 30, 100, 9, 41], new, seed=1)
    parents = _tree(new, 3, lean=0.3)  # deep ones
    q = _queries(batch.rows, 6, 64, kind, 3)
    mask = (torch.rand((batch.rows, 150), generator=_rng(4)) < 0.7).cuda()
    for m in (None, mask):
        got, lse = cache.attend(q, *batch.args, parents=parents.cuda(), window=window, sinks=sinks, mask=m,
                                return_lse=True)
        _check(cache, batch, q, got, lse, parents=parents, window=window, sinks=sinks, mask=m)


def test_a_chain_is_the_causal_call(gpu):
    cache = Int4KVCache(150, 2, 128, page_size=16)
    _fill(cache, 5)
    for new in ([7, 1, 30], [200, 3, 120], [1024, 5, 64]):
        batch = Batch(cache, [1100, 50, 700], new, seed=1)
        q = _queries(batch.rows, 8, 128, F32, 3)
        chain = torch.cat([torch.arange(n) - 1 for n in new]).to(torch.int32).cuda()
        for window in (None, 90):
            got = cache.attend(q, *batch.args, parents=chain, window=window)
            plain = cache.attend(q, *batch.args, window=window)
            assert bool(((got - plain).abs() <= 1e-5 * plain.abs().amax()).all())


def test_numbers_that_are_no_earlier_row(gpu):
    """Such rows come after the context, as -1 says."""
    cache = Int4KVCache(30, 2, 64, page_size=16)
    _fill(cache, 5)
    new = [9, 40]
    batch = Batch(cache, [100, 41], new, seed=1)
    parents = _tree(new, 3)
    parents[3], parents[5], parents[6], parents[12], parents[20] = 3, 8, 2**31 - 1, -2**31, 11
    q = _queries(batch.rows, 4, 64, BF16, 3)
    got, lse = cache.attend(q, *batch.args, parents=parents.cuda(), return_lse=True)
    _check(cache, batch, q, got, lse, parents=parents)


def test_more_rows_than_a_tree_has(gpu):
    cache = Int4KVCache(150, 1, 64, page_size=16)
    _fill(cache, 5)
    new = [3, 1025, 1]
    batch = Batch(cache, [40, 1100, 300], new, seed=1)
    parents = _tree(new, 3)
    q = _queries(batch.rows, 2, 64, BF16, 3)
    got, lse = cache.attend(q, *batch.args, parents=parents.cuda(), return_lse=True)
    _check(cache, batch, q, got, lse, parents=parents)
    assert not bool(got[3:1028].any()) and bool((lse[3:1028] == -math.inf).all())


def test_trees_of_padded_batches_and_bad_indices(gpu):
    """More rows than a sequence holds, holes, rows of no sequence, an output in place."""
    cache = Int4KVCache(12, 2, 128, page_size=16)
    _fill(cache, 5)
    new = [4, 2, 5]
    batch = Batch(cache, [40, 20, 3], new, seed=2)
    batch.host_table[0, 1], batch.host_table[1, 1] = 12, -7
    batch.table = batch.host_table.cuda()
    parents = _tree(new, 1)
    q = _queries(batch.rows, 4, 128, BF16, 3)
    got, lse = cache.attend(q, *batch.args, parents=parents.cuda(), return_lse=True)
    _check(cache, batch, q, got, lse, parents=parents)
    wide = torch.cat((q[:2], q, q[:3]))
    loose = torch.cat((parents[:2], parents, parents[:3])).cuda()
    out = cache.attend(wide, batch.table, batch.lengths, batch.offsets + 2, parents=loose, out=wide)
    assert out is wide and torch.equal(out[2:13], got) and not bool(out[:2].any()) and not bool(out[13:].any())
    one = Batch(cache, [40, 20, 3], [1, 1, 1], seed=2, offsets=False)
    q = _queries(3, 4, 128, BF16, 4)
    alone = torch.tensor([-1, 0, 5], dtype=torch.int32, device="cuda")
    assert torch.equal(cache.attend(q, *one.args, parents=alone), cache.attend(q, *one.args))


def test_long_contexts_and_trees(gpu):
    cache = Int4KVCache(1500, 2, 64, page_size=16)
    _fill(cache, 3)
    new = [64, 33, 200]
    batch = Batch(cache, [12003, 4000, 1700], new, seed=2)
    parents = _tree(new, 8)
    for kind in (F32, BF16):
        q = _queries(batch.rows, 8, 64, kind, 3)
        got, lse = cache.attend(q, *batch.args, parents=parents.cuda(), return_lse=True)
        _check(cache, batch, q, got, lse, parents=parents)


def test_drafts_that_a_row_does_not_come_after_have_no_effect(gpu):
    cache = Int4KVCache(20, 2, 128, page_size=16)
    _fill(cache, 3)
    batch = Batch(cache, [77], [8], seed=2)
    parents = torch.tensor([-1, 0, 0, 1, 2, 2, 4, 6], dtype=torch.int32)
    q = _queries(8, 8, 128, BF16, 3)
    clean = cache.attend(q, *batch.args, parents=parents.cuda())
    for row, line in ((7, {0, 2, 4, 6, 7}), (3, {0, 1, 3}), (5, {0, 2, 5})):
        spoilt = Int4KVCache(20, 2, 128, page_size=16)
        _fill(spoilt, 3)
        for other in set(range(8)) - line:
            j = 69 + other
            for scales in (spoilt.k_scales, spoilt.v_scales):
                scales[int(batch.host_table[0, j // 16]), :, j % 16] = math.nan
        got = spoilt.attend(q, *batch.args, parents=parents.cuda())
        assert torch.equal(got[row], clean[row])


# A table as wide as for long contexts sends trees that fill tiles of 256 query rows
# through the kernel for prompts.


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (96, 64), (128, 32)])
@pytest.mark.parametrize("window,sinks", [(None, None), (3, 2), (40, 130), (300, 5)])
@pytest.mark.parametrize("masked", [False, True])
def test_large_trees(gpu, kind, dim, page, window, sinks, masked):
    cache = Int4KVCache(2400 // page, 2, dim, page_size=page)
    _fill(cache, page)
    new = [60, 64, 58, 63]
    batch = Batch(cache, [275, 64, 900, 131], new, seed=1, spare=40000 // page)
    parents = _tree(new, dim, lean=0.4)
    q = _queries(batch.rows, 8, dim, kind, 3)
    mask = (torch.rand((batch.rows, 880), generator=_rng(4)) < 0.7).cuda() if masked else None
    got, lse = cache.attend(q, *batch.args, parents=parents.cuda(), window=window, sinks=sinks, mask=mask,
                            return_lse=True)
    _check(cache, batch, q, got, lse, parents=parents, window=window, sinks=sinks, mask=mask)


@pytest.mark.parametrize("chain", [False, True])
@pytest.mark.parametrize("lengths", [[1300, 1024], [1057, 2000], [1025, 900]])
def test_trees_of_many_words(gpu, chain, lengths):
    """A thousand rows of a sequence, more of them than it holds too, and of one too many."""
    cache = Int4KVCache(300, 2, 64, page_size=16)
    _fill(cache, 6)
    for new in ([1024, 1000], [1025, 1020]):
        batch = Batch(cache, lengths, new, seed=1, spare=3000)
        parents = torch.cat([torch.arange(n) - 1 for n in new]).to(torch.int32) if chain else _tree(new, 5, lean=0.7)
        q = _queries(batch.rows, 2, 64, BF16, 3)
        for kw in ({}, {"window": 200, "sinks": 1100}):
            got, lse = cache.attend(q, *batch.args, parents=parents.cuda(), return_lse=True, **kw)
            _check(cache, batch, q, got, lse, parents=parents, **kw)


# Many sequences, whose items stay whole in one launch.


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("share,new", [(1, 1), (4, 1), (4, 7), (1, 40), (40, 2)])
@pytest.mark.parametrize("window,sinks", [(700, 40), (1500, 3), (95, 260)])
def test_many_sequences_with_sinks(gpu, kind, share, new, window, sinks):
    g = _rng(new)
    lengths = torch.randint(1, 1900, (40,), generator=g).tolist()
    lengths[:3] = [1900, 2, 0]
    cache = Int4KVCache(sum(-(-n // 32) for n in lengths), 4, 64, page_size=32)
    _fill(cache, 8)
    rows = [min(n, new) for n in lengths]
    batch = Batch(cache, lengths, rows, seed=3, spare=200)
    q = _queries(batch.rows, 4 * share, 64, kind, 3)
    got, lse = cache.attend(q, *batch.args, window=window, sinks=sinks, return_lse=True)
    _check(cache, batch, q, got, lse, window=window, sinks=sinks)


@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("share,new", [(1, 3), (4, 12)])
def test_many_sequences_with_trees(gpu, kind, share, new):
    g = _rng(new)
    lengths = torch.randint(1, 1000, (70,), generator=g).tolist()
    lengths[:3] = [1000, 2, 0]
    cache = Int4KVCache(sum(-(-n // 32) for n in lengths), 4, 64, page_size=32)
    _fill(cache, 8)
    rows = [min(n, new) for n in lengths]
    batch = Batch(cache, lengths, rows, seed=3)
    parents = _tree(rows, 5)
    q = _queries(batch.rows, 4 * share, 64, kind, 3)
    for kw in ({}, {"window": 100, "sinks": 20}):
        got, lse = cache.attend(q, *batch.args, parents=parents.cuda(), return_lse=True, **kw)
        _check(cache, batch, q, got, lse, parents=parents, **kw)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("lengths,new", [([700], 64), ([0, 1, 900, 513, 130, 31, 800, 24], 24), ([1040, 1023], 39)])
def test_few_sequences_in_small_tiles(gpu, kind, dim, lengths, new):
    """Whole items of 16 rows, several for a sequence, some of them ragged or empty."""
    cache = Int4KVCache(sum(-(-n // 16) for n in lengths), 4, dim, page_size=16)
    _fill(cache, 8)
    rows = [min(n, new) for n in lengths]
    batch = Batch(cache, lengths, rows, seed=3, spare=150)
    parents = _tree(rows, 5)
    q = _queries(batch.rows, 16, dim, kind, 3)
    for kw in ({}, {"window": 60, "sinks": 33}):
        got, lse = cache.attend(q, *batch.args, parents=parents.cuda(), return_lse=True, **kw)
        _check(cache, batch, q, got, lse, parents=parents, **kw)
    for window, sinks in ((600, 4), (513, 100)):
        got, lse = cache.attend(q, *batch.args, window=window, sinks=sinks, return_lse=True)
        _check(cache, batch, q, got, lse, window=window, sinks=sinks)


@pytest.mark.parametrize("lo,hi,new", [(1, 2500, 9), (1, 700, 33), (2000, 6000, 2)])
def test_ragged_split_items(gpu, lo, hi, new):
    """Short and long sequences dealt out together."""
    lengths = torch.randint(lo, hi, (24,), generator=_rng(hi)).tolist()
    cache = Int4KVCache(sum(-(-n // 16) for n in lengths), 2, 64, page_size=16)
    _fill(cache, 8)
    rows = [min(n, new) for n in lengths]
    batch = Batch(cache, lengths, rows, seed=3, spare=200)
    parents = _tree(rows, 5)
    q = _queries(batch.rows, 4, 64, BF16, 3)
    got, lse = cache.attend(q, *batch.args, parents=parents.cuda(), return_lse=True)
    _check(cache, batch, q, got, lse, parents=parents)
    got, lse = cache.attend(q, *batch.args, window=4000, sinks=9, return_lse=True)
    _check(cache, batch, q, got, lse, window=4000, sinks=9)


def test_another_stream(gpu):
    cache = Int4KVCache(300, 2, 128, page_size=16)
    _fill(cache, 3)
    new = [20, 9]
    batch = Batch(cache, [3001, 1500], new, seed=2)
    parents = _tree(new, 8).cuda()
    kept = torch.tensor([[1, 4, 9], [0, 2, -1]], dtype=torch.int32, device="cuda")
    q = _queries(batch.rows, 8, 128, BF16, 3)
    want = cache.attend(q, *batch.args, parents=parents, window=900, sinks=7)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            assert torch.equal(cache.attend(q, *batch.args, parents=parents, window=900, sinks=7), want)
        assert cache.keep(*batch.args, kept).tolist() == [2984, 1493]


# ------------------------------------------------------------------ kept rows


@pytest.mark.parametrize("dim,page,heads", [(64, 16, 3), (96, 32, 2), (128, 64, 8), (192, 16, 1), (256, 128, 2)])
@pytest.mark.parametrize("width", [1, 5, 70, 300])
def test_kept_rows(gpu, dim, page, heads, width):
    cache = Int4KVCache(2200 // page, heads, dim, page_size=page)
    _fill(cache, dim)
    new = [1, 20, 0, 290, 7, 3, 16, 129]
    batch = Batch(cache, [page + 5, 75, 9, 3 * page + 301, 7, 2, 3 * page, 140], new, seed=4)
    g = _rng(width)
    kept = torch.full((len(new), width), -1, dtype=torch.int32)
    counts = []
    for b, n in enumerate(new):
        count = int(torch.randint(0, min(n, width) + 1, (1,), generator=g))
        kept[b, :count] = torch.randperm(n, generator=g)[:count].sort().values.to(torch.int32)
        counts.append(count)
    if width >= 20:  # ends that are no numbers of rows, or do not ascend
        kept[1, :6] = torch.tensor([0, 4, 4, 9, -1, 3])
        kept[4, :4] = torch.tensor([2, 6, 7, 8])
        kept[6, :5] = torch.tensor([3, 5, 2, 9, 11])
        counts[1], counts[4], counts[6] = 2, 2, 2
    before = [x.clone() for x in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    after = cache.keep(*batch.args, kept.cuda())
    assert after.tolist() == [max(0, n - m + c) for n, m, c in zip(batch.host_lengths, new, counts)]
    exp = [x.clone() for x in before]
    for b, (n, m, count) in enumerate(zip(batch.host_lengths, new, counts)):
        for i in range(count):
            to, source = n - m + i, n - m + int(kept[b, i])
            if source < 0 or to < 0:
                continue
            for x, y in zip(exp, before):
                x[int(batch.host_table[b, to // page]), :, to % page] = \
                    y[int(batch.host_table[b, source // page]), :, source % page]
    for x, y in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), exp):
        assert torch.equal(x, y)


def test_kept_rows_and_bad_indices(gpu):
    """More rows than a sequence holds, holes on either side, lengths past the table."""
    cache = Int4KVCache(12, 2, 64, page_size=16)
    _fill(cache, 5)
    batch = Batch(cache, [40, 45, 3, 33], [20, 30, 5, 10], seed=2)
    batch.host_table[0, 1] = 12   # rows 20 .. 31 of 40: targets
    batch.host_table[1, 2] = -3   # rows 32 .. 44 of 45: sources
    table, lengths = batch.host_table.cuda(), batch.lengths.clone()
    lengths[3] = 2**30
    kept = torch.tensor([[1, 13, 18], [16, 17, 20], [0, 3, 4], [2, 3, 9]], dtype=torch.int32, device="cuda")
    codes, scales = cache.k_codes.clone(), cache.k_scales.clone()
    after = cache.keep(table, lengths, batch.offsets, kept)
    long = batch.host_table.shape[1] * 16
    assert after.tolist() == [23, 18, 1, long - 7]
    t = batch.host_table.long()
    assert torch.equal(cache.k_codes[t[0, 0]], codes[t[0, 0]]) and torch.equal(cache.k_codes[t[0, 2]], codes[t[0, 2]])
    # Sequence 1: row 16 stands at 31, rows 17 and 20 in the hole; they go to 15, 16 and 17.
    assert torch.equal(cache.k_codes[t[1, 0], :, 15], codes[t[1, 1], :, 15])
    assert not bool(cache.k_codes[t[1, 1], :, :2].any()) and bool((cache.k_scales[t[1, 1], :, :2] == 1).all())
    assert torch.equal(cache.k_codes[t[1, 1], :, 2:], codes[t[1, 1], :, 2:])
    # Sequence 2: rows 0 and 1 stand before its first token; row 4 at 2 goes to 0.
    assert torch.equal(cache.k_codes[t[2, 0], :, 0], codes[t[2, 0], :, 2])
    assert torch.equal(cache.k_scales[t[2, 0], :, 1:], scales[t[2, 0], :, 1:])


def test_kept_rows_past_32_bits(gpu):
    """Pages whose codes begin past 2^32 bytes."""
    cache = Int4KVCache(132000, 8, 128, page_size=64)
    table = torch.tensor([[131999, 131072], [3, 131998]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([70, 100], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
    x = [torch.randn((50, 8, 128), generator=_rng(i)).cuda() for i in (1, 2)]
    cache.append(*x, table, lengths, offsets)
    before = cache.read(table, lengths, offsets, rows=50, dtype=F32)
    kept = torch.tensor([[3, 13, 19], [2, 28, -1]], dtype=torch.int32, device="cuda")
    after = cache.keep(table, lengths, offsets, kept)
    ends = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda")
    index = torch.tensor([3, 13, 19, 22, 48], device="cuda")
    for a, b in zip(cache.read(table, after, ends, rows=5, dtype=F32), before):
        assert torch.equal(a, b[index])


def test_kept_rows_of_single_tokens_and_empty_calls(gpu):
    cache = Int4KVCache(12, 2, 64, page_size=16)
    _fill(cache, 5)
    batch = Batch(cache, [40, 20, 3], [1, 1, 1], seed=2, offsets=False)
    codes = cache.k_codes.clone()
    kept = torch.tensor([[0], [-1], [1]], dtype=torch.int32, device="cuda")
    assert cache.keep(*batch.args, kept).tolist() == [40, 19, 2]
    assert cache.keep(*batch.args, kept[:, :0]).tolist() == [39, 19, 2]
    assert torch.equal(cache.k_codes, codes)
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert cache.keep(empty.view(0, 2), empty, None, empty.view(0, 3)).shape == (0,)


# ------------------------------------------------------------------ all of it


def test_a_drafting_loop(gpu):
    """Pages, positions, rows, trees, kept branches: the cache holds what a plain loop over
    the accepted tokens would, and attention over it is the same."""
    batch, heads, kv_heads, dim, page, drafts = 3, 4, 2, 64, 16, 6
    cache = Int4KVCache(60, kv_heads, dim, page_size=page)
    pages = CachePages(60, batch, 12, page_size=page)
    plain, plain_pages = Int4KVCache(60, kv_heads, dim, page_size=page), CachePages(60, batch, 12, page_size=page)
    rotary = Rotary(dim)
    width = 96
    weight = torch.randn(((heads + 2 * kv_heads) * dim, width), generator=_rng(0)).cuda() / 10
    linear = Int4Linear.from_float(weight, 32)

    def rows_of(x, positions):
        y = linear(x).view(-1, heads + 2 * kv_heads, dim)
        q, k = rotary(y[:, :heads], y[:, heads:heads + kv_heads], positions)
        return q, k, y[:, heads + kv_heads:]

    g = _rng(9)
    kept_lengths = None
    for step in range(7):
        if step == 0:  # prompts
            new = torch.tensor([37, 5, 60], dtype=torch.int32)
            parents = torch.cat([torch.arange(n) - 1 for n in new.tolist()]).to(torch.int32)
            kept = torch.arange(60, dtype=torch.int32).expand(batch, 60)
        else:
            new = torch.full((batch,), drafts, dtype=torch.int32)
            parents = _tree([drafts] * batch, step)
            lines = []
            for b in range(batch):
                row, line = int(torch.randint(0, drafts, (1,), generator=g)), []
                while row >= 0:
                    line.append(row)
                    row = int(parents[b * drafts + row])
                lines.append(line[::-1] + [-1] * (drafts - len(line)))
            kept = torch.tensor(lines, dtype=torch.int32)
        rows = int(new.sum())
        x = torch.randn((rows, width), generator=g).to(BF16).cuda()
        offsets, positions, _ = pages.update(new.cuda(), lengths=kept_lengths, rows=rows)
        # A row's position counts the rows that it comes after.
        first = torch.cat((torch.zeros(1, dtype=torch.int64), new.cumsum(0)[:-1])).repeat_interleave(new.long())
        depth = torch.zeros(rows, dtype=torch.int32)
        for i, p in enumerate(parents.tolist()):
            depth[i] = depth[int(first[i]) + p] + 1 if p >= 0 else 0
        start = (pages.lengths - new.cuda()).cpu().repeat_interleave(new.long())
        at = (start + depth).to(torch.int32).cuda()
        if step == 0:
            assert torch.equal(at, positions)
        q, k, v = rows_of(x, at)
        cache.append(k, v, pages.table, pages.lengths, offsets)
        out = cache.attend(q, pages.table, pages.lengths, offsets, parents=parents.cuda(), window=50, sinks=3)
        kept_lengths = cache.keep(pages.table, pages.lengths, offsets, kept.contiguous().cuda())
        # The plain loop takes in the accepted rows alone.
        index = torch.cat([first[offsets[b]] + kept[b][:int((kept[b] >= 0).sum())].long()
                           if step else torch.arange(int(offsets[b]), int(offsets[b + 1])) for b in range(batch)])
        counts = [int((kept[b] >= 0).sum()) if step else int(new[b]) for b in range(batch)]
        plain_offsets, plain_at, _ = plain_pages.update(torch.tensor(counts, dtype=torch.int32).cuda(), rows=len(index))
        assert torch.equal(plain_at, at[index.cuda()])
        args = plain_pages.table, plain_pages.lengths, plain_offsets
        plain.append(k[index.cuda()], v[index.cuda()], *args)
        assert torch.equal(kept_lengths, plain_pages.lengths)
        expected = plain.attend(q[index.cuda()], *args, window=50, sinks=3).float()
        diff = (out[index.cuda()].float() - expected).abs()
        assert bool((diff <= 2.0**-6 * expected.abs() + 2.0**-7 * expected.abs().amax()).all())
        whole = plain_pages.lengths.cumsum(0).to(torch.int32)
        ends = torch.cat((torch.zeros(1, dtype=torch.int32, device="cuda"), whole))
        for a, b in zip(cache.read(pages.table, kept_lengths, ends, dtype=F32),
                        plain.read(plain_pages.table, plain_pages.lengths, ends, dtype=F32)):
            assert torch.equal(a, b)


def test_graph_replays(gpu):
    """A drafting step in one graph: rows in, attention of the tree, kept rows, pages."""
    def make():
        cache, pages = Int4KVCache(60, 2, 64, page_size=16), CachePages(60, 3, 12, page_size=16)
        _fill(cache, 2)
        pages.update(torch.tensor([70, 33, 5], dtype=torch.int32).cuda())
        return cache, pages

    new = torch.full((3,), 8, dtype=torch.int32, device="cuda")
    x = torch.zeros((24, 8, 64), dtype=BF16, device="cuda")
    parents, kept = _tree([8] * 3, 0).cuda(), torch.zeros((3, 4), dtype=torch.int32, device="cuda")

    def step(cache, pages, lengths):
        offsets, positions, slots = pages.update(new, lengths=lengths, rows=24)
        cache.append(x[:, 4:6], x[:, 6:8], pages.table, pages.lengths, offsets)
        out = cache.attend(x[:, :4], pages.table, pages.lengths, offsets, parents=parents, window=40, sinks=5)
        lengths.copy_(cache.keep(pages.table, pages.lengths, offsets, kept))
        return out, positions, slots

    (cache, pages), (other, other_pages) = make(), make()
    lengths, other_lengths = pages.lengths.clone(), pages.lengths.clone()
    warm_cache, warm_pages = make()
    step(warm_cache, warm_pages, warm_pages.lengths.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache, pages, lengths)
    for i in range(5):
        x.copy_(torch.randn(x.shape, generator=_rng(i)))
        parents.copy_(_tree([8] * 3, i))
        kept.copy_(torch.tensor([[0, 3, 5, -1], [i, -1, -1, -1], [1, 2, 6, 7]]))
        graph.replay()
        torch.cuda.synchronize()
        want = step(other, other_pages, other_lengths)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(lengths, other_lengths)
        assert torch.equal(pages.table, other_pages.table) and torch.equal(cache.k_codes, other.k_codes)


def test_refusals(gpu):
    cache = Int4KVCache(6, 2, 64, page_size=16)
    table = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    lengths = torch.ones(2, dtype=torch.int32, device="cuda")
    q = torch.zeros((2, 4, 64), device="cuda")
    parents = torch.full((2,), -1, dtype=torch.int32, device="cuda")
    for kw in ({"sinks": -1, "window": 3}, {"parents": parents.long()}, {"parents": parents[:1]},
               {"parents": parents.cpu()}, {"parents": parents, "causal": False}, {"parents": [0, 1]},
               {"parents": parents.repeat(2)[::2]}):
        with pytest.raises(ValueError):
            cache.attend(q, table, lengths, **kw)
    kept = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    for args in ((table, lengths, None, kept.long()), (table, lengths, None, kept[:1]), (table, lengths, None, kept[0]),
                 (table, lengths, lengths, kept), (table, lengths, None, kept.cpu()), (table[:1], lengths, None, kept),
                 (table, lengths.long(), None, kept), (table, lengths, None, kept.repeat(1, 2)[:, ::2])):
        with pytest.raises(ValueError):
            cache.keep(*args)
    assert cache.attend(q[:0], table[:0], lengths[:0], parents=parents[:0]).shape == (0, 4, 64)
