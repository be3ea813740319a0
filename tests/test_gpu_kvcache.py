"""The 4-bit key/value cache: rows in, rows back and attention over them,
against plain float64 computations from the stored codes."""
import math

import numpy as np
import pytest
import torch

from maxsim_amd import Int4KVCache, pack_int4_symmetric

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ROUND = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}  # of a result, relative (the spacing, for bfloat16)


def _rng(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


class Batch:
    """Sequences in shuffled pages, and the rows of a call."""

    def __init__(self, cache, lengths, new, seed=0, spare=0, offsets=True):
        page = cache.page_size
        used = [-(-n // page) for n in lengths]
        pages = torch.randperm(cache.num_pages, generator=_rng(seed)).to(torch.int32)
        assert sum(used) <= cache.num_pages
        table = torch.full((len(lengths), max(used, default=0) + spare), -1, dtype=torch.int32)
        first = 0
        for b, n in enumerate(used):
            table[b, :n] = pages[first:first + n]
            first += n
        self.host_table, self.host_lengths, self.new = table, list(lengths), list(new)
        self.table = table.cuda()
        self.lengths = torch.tensor(lengths, dtype=torch.int32).cuda()
        off = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.host_offsets = off
        self.offsets = torch.from_numpy(off).cuda() if offsets else None
        self.rows = int(off[-1])

    @property
    def args(self):
        return self.table, self.lengths, self.offsets

    def slots(self, cache):
        """(row, page, slot) of the rows that have one."""
        out = []
        for b, (n, m) in enumerate(zip(self.host_lengths, self.new)):
            for i in range(m):
                pos = n - m + i
                if pos < 0:
                    continue
                page = int(self.host_table[b, pos // cache.page_size])
                if 0 <= page < cache.num_pages:
                    out.append((int(self.host_offsets[b]) + i, page, pos % cache.page_size))
        return out


def _fill(cache, seed, spread=0.5):
    """Every slot of the pool holds a random row."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        # Codes -7 .. 7 in both nibbles.
        c = torch.randint(-7, 8, (*codes.shape, 2), generator=g, device="cuda").to(torch.int8).view(torch.uint8)
        codes.copy_((c[..., 0] & 15) | ((c[..., 1] & 15) << 4))
        scales.copy_(0.15 * torch.exp(spread * torch.randn(scales.shape, generator=g, device="cuda")))


def _values(codes):
    c = codes.cpu().numpy()
    out = np.empty((*c.shape[:-1], c.shape[-1] * 2), np.float64)
    out[..., 0::2] = ((c & 15).astype(np.int16) ^ 8) - 8
    out[..., 1::2] = ((c >> 4).astype(np.int16) ^ 8) - 8
    return torch.from_numpy(out)


def _pool(cache):
    """Keys and values [pages, heads, page, dim] in float64."""
    return [_values(c) * s.cpu().double()[..., None]
            for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales))]


def _expected(cache, batch, q, scale=None, causal=True, window=None, mask=None):
    """(out, lse, tolerance's weight) in float64.  The weight bounds, per output,
    sum p |v| and the error of the scores."""
    heads, dim = q.shape[1], cache.head_dim
    share = heads // cache.kv_heads
    scale = dim**-0.5 if scale is None else scale
    pool_k, pool_v = _pool(cache)
    q = q.cpu().double()
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    mass = torch.zeros(q.shape, dtype=torch.float64)
    delta = torch.zeros(q.shape[:2], dtype=torch.float64)
    for b, (n, m) in enumerate(zip(batch.host_lengths, batch.new)):
        pages = batch.host_table[b].long()
        keep = torch.arange(n)
        page = pages[keep // cache.page_size]
        hole = (page < 0) | (page >= cache.num_pages)
        page = page.clamp(0, cache.num_pages - 1)
        for i in range(m):
            row, pos = int(batch.host_offsets[b]) + i, n - m + i
            see = ~hole
            if causal:
                see = see & (keep <= pos)
            if window is not None:
                see = see & (keep > pos - window)
            if mask is not None:
                hidden = torch.ones(n, dtype=torch.bool)
                width = min(n, mask.shape[1])
                hidden[:width] = ~mask[row, :width].cpu()
                see = see & ~hidden
            if not bool(see.any()):
                continue
            at, slot = page[see], keep[see] % cache.page_size
            for h in range(heads):
                k, v = pool_k[at, h // share, slot], pool_v[at, h // share, slot]
                s = (k @ q[row, h]) * scale
                top = s.max()
                p = torch.exp(s - top)
                out[row, h] = p @ v / p.sum()
                mass[row, h] = p @ v.abs() / p.sum()
                lse[row, h] = top + torch.log(p.sum())
                # A score is dim products summed in single precision and two more
                # roundings; single precision queries keep 22 bits of their largest.
                sums = float((k.abs() @ q[row, h].abs()).max()) * abs(scale)
                part = float(k.abs().sum(1).max() * q[row, h].abs().max()) * abs(scale) * 2.0**-23
                delta[row, h] = 2.0**-24 * (dim / 4 + 4) * sums + part + 2.0**-23
    return out, lse, mass, delta


def _check(cache, batch, q, got, got_lse=None, **kw):
    out, lse, mass, delta = _expected(cache, batch, q, **kw)
    kind = q.dtype
    probs = 2.0**-21 if kind == F32 else 2.0**-11  # rounding of probability times scale
    longest = max(batch.host_lengths, default=1)
    sums = 2.0**-24 * (longest / 8 + 16)  # a lane's keys, then the joins
    tol = ROUND[kind] * out.abs() + (probs + 2 * delta[..., None] + 2 * sums) * mass + 1e-30
    if kind == F16:
        tol = tol + 2.0**-25  # subnormal results
    diff = (got.cpu().double() - out).abs()
    assert bool((diff <= tol).all()), float((diff / tol).max())
    if got_lse is not None:
        empty = torch.isinf(lse)
        assert bool((torch.isinf(got_lse.cpu()) & (got_lse.cpu() < 0) == empty).all())
        diff = (got_lse.cpu().double() - lse).abs()[~empty]
        assert bool((diff <= (delta + sums + 2.0**-22 * (1 + lse.abs()))[~empty]).all())


def _queries(rows, heads, dim, kind, seed, size=1.0):
    return (size * torch.randn((rows, heads, dim), generator=_rng(seed))).to(kind).cuda()


# ------------------------------------------------------------------ rows


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page,heads", [(64, 16, 3), (96, 32, 2), (128, 64, 8), (192, 16, 1), (256, 128, 2)])
def test_rows_in_and_back(gpu, kind, dim, page, heads):
    cache = Int4KVCache(40, heads, dim, page_size=page)
    batch = Batch(cache, [1, page + 5, 0, 3 * page - 1, 17, 2 * page], [1, 9, 0, 3 * page - 1, 2, 40 if page > 16 else 30])
    x = [torch.randn((batch.rows, heads, dim), generator=_rng(i)) * 3 for i in (1, 2)]
    x[0][0] = 0.0  # a row of zeros
    x[1][1, 0, :] = torch.where(torch.arange(dim) % 3 == 0, 0.5, 1.0)  # quotients of 3.5
    x[0][2] *= 2.0**-14
    x = [t.to(kind).cuda() for t in x]
    before = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    cache.append(x[0], x[1], *batch.args)
    got = cache.read(*batch.args, rows=batch.rows, dtype=kind)
    for side, (codes, scales) in enumerate(((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales))):
        packed = pack_int4_symmetric(x[side].float().cpu().numpy().reshape(-1, dim), scale_granularity="token")
        exp_codes, exp_scales = before[2 * side], before[2 * side + 1]
        for row, pg, slot in batch.slots(cache):
            rows = slice(row * heads, (row + 1) * heads)
            exp_codes[pg, :, slot] = torch.from_numpy(packed.data[rows]).cuda()
            exp_scales[pg, :, slot] = torch.from_numpy(packed.token_scale[rows]).cuda()
        assert torch.equal(codes, exp_codes) and torch.equal(scales, exp_scales)
        exp = torch.from_numpy(packed.values.astype(np.float32) * packed.token_scale[:, None]).to(kind)
        assert torch.equal(got[side].cpu(), exp.view(batch.rows, heads, dim))


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_rows_of_a_fused_projection(gpu, kind, shift):
    """Keys and values as views of one buffer, at any alignment."""
    heads, dim = 4, 96
    cache = Int4KVCache(8, heads, dim, page_size=16)
    batch = Batch(cache, [33, 20, 1], [33, 3, 1], seed=4)
    width = 5 * heads * dim + 24 + shift
    fused = torch.randn((batch.rows, width), generator=_rng(3)).to(kind).cuda()
    k = fused[:, shift:shift + heads * dim].view(batch.rows, heads, dim)
    v = fused[:, shift + 2 * heads * dim:shift + 4 * heads * dim].view(batch.rows, heads, 2 * dim)[..., :dim]
    cache.append(k, v, *batch.args)
    plain = Int4KVCache(8, heads, dim, page_size=16)
    plain.append(k.contiguous(), v.contiguous(), *batch.args)
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        assert torch.equal(getattr(cache, name), getattr(plain, name))
    out = torch.zeros((2, batch.rows, heads, dim + 4 + shift), dtype=kind, device="cuda")
    got = cache.read(*batch.args, out=(out[0, ..., :dim], out[1, ..., shift:shift + dim]))
    exp = cache.read(*batch.args, dtype=kind)
    assert torch.equal(got[0], exp[0]) and torch.equal(got[1], exp[1])
    assert not bool(out[0, ..., dim:].any())


def test_rows_with_infinities_and_nans(gpu):
    cache = Int4KVCache(4, 2, 64, page_size=16)
    for kind in (F32, F16, BF16):
        x = torch.randn((6, 2, 64), generator=_rng(1)).to(kind)
        x[0, 0, 5], x[1, 1, 63], x[2, 0, 0] = math.inf, math.nan, -math.inf
        batch = Batch(cache, [6], [6])
        cache.append(x.cuda(), (x * 2).cuda(), *batch.args)
        for t in cache.read(*batch.args, dtype=kind):
            bad = torch.isnan(t).cpu()
            exp = ~torch.isfinite(x.float()).all(-1, keepdim=True).expand_as(x)
            assert torch.equal(bad, exp)


@pytest.mark.parametrize("size", [2.0**-149, 2.0**-140, 2.0**-127, 1e30, 3.3e38])
def test_rows_of_extreme_sizes(gpu, size):
    """The packer's arithmetic holds from subnormal rows to the largest ones."""
    x = np.random.default_rng(0).uniform(-1, 1, (32, 1, 128))
    x = torch.from_numpy(x * size).float()
    packed = pack_int4_symmetric(x.numpy().reshape(32, 128), scale_granularity="token")
    cache = Int4KVCache(1, 1, 128, page_size=32)
    batch = Batch(cache, [32], [32])
    cache.append(x.cuda(), x.cuda(), *batch.args)
    np.testing.assert_array_equal(cache.k_scales[0, 0].cpu().numpy(), packed.token_scale)
    np.testing.assert_array_equal(cache.v_codes[0, 0].cpu().numpy(), packed.data)


def test_many_short_sequences(gpu):
    """More sequences than a search step covers, many of them without rows."""
    cache = Int4KVCache(9000, 1, 64, page_size=16)
    new = torch.randint(0, 4, (8500,), generator=_rng(5)).tolist()
    batch = Batch(cache, [max(1, n) for n in new], new, seed=6)
    x = torch.randn((batch.rows, 1, 64), generator=_rng(7)).cuda()
    cache.append(x, -x, *batch.args)
    k, v = cache.read(*batch.args, dtype=F32)
    s = x.abs().amax(-1, keepdim=True) / 7
    assert bool(((k - x).abs() <= 0.5001 * s).all()) and torch.equal(k, -v)
    q = _queries(batch.rows, 1, 64, F32, 8)
    got = cache.attend(q, *batch.args, window=1)  # each token sees itself
    assert bool(((got - v).abs() <= 1e-6 * v.abs().amax(-1, keepdim=True)).all())


def test_holes_and_bad_indices(gpu):
    """Page numbers outside the pool, lengths past the table, more rows than a
    sequence holds, rows of no sequence."""
    cache = Int4KVCache(6, 2, 128, page_size=16)
    _fill(cache, 1)
    batch = Batch(cache, [40, 20, 3], [4, 2, 5], seed=2)
    batch.host_table[0, 1] = 6
    batch.host_table[1, 1] = -7
    batch.table = batch.host_table.cuda()
    q = _queries(batch.rows, 4, 128, BF16, 3)
    got, lse = cache.attend(q, *batch.args, return_lse=True)
    _check(cache, batch, q, got, lse)
    assert not bool(got[6:8].any())  # sequence 2's first rows stand before its first token
    before = cache.k_codes.clone()
    x = torch.ones((batch.rows, 2, 128), dtype=BF16, device="cuda")
    cache.append(x, x, *batch.args)
    changed = (cache.k_codes != before).any(-1).any(1).sum()
    assert int(changed) == len(batch.slots(cache))
    k, _ = cache.read(*batch.args, rows=batch.rows)
    have = {row for row, _, _ in batch.slots(cache)}
    for row in range(batch.rows):
        assert bool(k[row].any()) == (row in have)
    # A length past the table ends with it; offsets may leave rows out.
    long = torch.tensor([10**9, 20, 3], dtype=torch.int32, device="cuda")
    cut = batch.host_table.shape[1] * 16
    other = Batch(cache, [cut, 20, 3], [2, 0, 3], seed=2)
    other.host_table, other.table = batch.host_table, batch.table
    q = _queries(9, 4, 128, BF16, 4)
    offsets = torch.tensor([2, 4, 4, 7], dtype=torch.int32, device="cuda")
    got, lse = cache.attend(q, batch.table, long, offsets, return_lse=True)
    _check(cache, other, q[2:7], got[2:7], lse[2:7])
    assert not bool(got[:2].any()) and not bool(got[7:].any())
    assert bool((lse[:2] == -math.inf).all()) and bool((lse[7:] == -math.inf).all())
    k, _ = cache.read(batch.table, long, offsets, rows=9)
    assert not bool(k[:2].any()) and not bool(k[7:].any())
    empty = torch.zeros((0, 2), dtype=torch.int32, device="cuda")
    got = cache.attend(q, empty, torch.zeros(0, dtype=torch.int32, device="cuda"),
                       torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert not bool(got.any())


def test_slots_given_to_two_rows(gpu):
    """Words and scales of either row in the shared slots, and nothing elsewhere."""
    caches = [Int4KVCache(4, 3, 128, page_size=16) for _ in range(3)]
    table = torch.tensor([[1], [1]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([9, 9], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 5, 10], dtype=torch.int32, device="cuda")
    x = (torch.randn((10, 3, 128), generator=_rng(1)) * torch.arange(1, 11)[:, None, None]).cuda()
    caches[0].append(x, -x, table, lengths, offsets)
    for cache, rows in zip(caches[1:], (x[:5], x[5:])):
        cache.append(rows, -rows, table[:1], lengths[:1], offsets[:2])
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        got, one, other = (getattr(cache, name) for cache in caches)
        if name.endswith("codes"):
            got, one, other = (t.view(torch.int32) for t in (got, one, other))
        assert bool(((got == one) | (got == other)).all())


# ------------------------------------------------------------- attention


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("kv_heads,share", [(1, 1), (2, 4), (3, 6), (1, 16), (2, 20)])
def test_single_tokens(gpu, kind, dim, kv_heads, share):
    cache = Int4KVCache(80, kv_heads, dim, page_size=32)
    _fill(cache, dim)
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 0, 127, 128, 129, 300, 701]
    batch = Batch(cache, lengths, [1] * len(lengths), offsets=False)
    q = _queries(batch.rows, kv_heads * share, dim, kind, 2, size=2.0)
    got, lse = cache.attend(q, *batch.args, return_lse=True)
    _check(cache, batch, q, got, lse)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (96, 64), (128, 16), (128, 128), (256, 32)])
@pytest.mark.parametrize("causal,window", [(True, None), (True, 40), (False, None), (False, 9)])
def test_many_tokens(gpu, kind, dim, page, causal, window):
    cache = Int4KVCache(64, 2, dim, page_size=page)
    _fill(cache, page)
    batch = Batch(cache, [75, 64, 0, 130, 5, 33], [75, 1, 0, 37, 5, 2], seed=1)
    q = _queries(batch.rows, 6, dim, kind, 3)
    got, lse = cache.attend(q, *batch.args, causal=causal, window=window, return_lse=True)
    _check(cache, batch, q, got, lse, causal=causal, window=window)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("width", [0, 1, 40, 131, 200])
@pytest.mark.parametrize("causal", [True, False])
def test_masks(gpu, kind, width, causal):
    """Random masks, rows that see nothing, masks narrower than the sequences."""
    cache = Int4KVCache(24, 2, 128, page_size=16)
    _fill(cache, 9)
    batch = Batch(cache, [131, 70, 16, 90], [7, 1, 16, 30], seed=3)
    mask = torch.rand((batch.rows, width + 5), generator=_rng(width)) < 0.4
    mask[::5] = False
    mask = mask.cuda()[:, :width]  # its rows are strided
    q = _queries(batch.rows, 4, 128, kind, 5)
    got, lse = cache.attend(q, *batch.args, mask=mask, causal=causal, return_lse=True)
    _check(cache, batch, q, got, lse, mask=mask, causal=causal)
    assert not bool(got[::5].any()) and bool((lse[::5] == -math.inf).all())


@pytest.mark.parametrize("junk", [math.nan, math.inf, 3e38, 1e30, 1e-38])
@pytest.mark.parametrize("hide", ["mask", "window", "causal"])
def test_hidden_keys_have_no_effect(gpu, junk, hide):
    """Slots that a row does not see may hold anything."""
    cache = Int4KVCache(16, 2, 128, page_size=16)
    _fill(cache, 4)
    batch = Batch(cache, [100, 47], [6, 1], seed=1)
    q = _queries(batch.rows, 8, 128, BF16, 6)
    seen = {"mask": 50, "window": 94, "causal": 95}[hide]
    kw = {}
    if hide == "mask":
        mask = torch.ones((batch.rows, 100), dtype=torch.bool)
        mask[:, 50:] = False
        mask[:, 3] = False
        kw["mask"] = mask.cuda()
    if hide == "window":
        kw["window"] = 1
    clean = cache.attend(q, *batch.args, **kw)
    spoil = torch.zeros((16, 16), dtype=torch.bool)
    held = torch.zeros((16, 16), dtype=torch.bool)
    for b, n in enumerate(batch.host_lengths):
        for pos in range(n):
            page, slot = int(batch.host_table[b, pos // 16]), pos % 16
            held[page, slot] = True
            hidden = {"mask": pos >= seen or pos == 3, "window": pos < n - (6 if b == 0 else 1),
                      "causal": b == 0 and pos > seen - 1}[hide]
            spoil[page, slot] = hidden
    spoil |= ~held
    for scales in (cache.k_scales, cache.v_scales):
        s = scales.transpose(1, 2)
        s[spoil.cuda()] = junk
    got = cache.attend(q, *batch.args, **kw)
    rows = slice(0, 1) if hide == "causal" else slice(0, batch.rows)
    assert bool(torch.isfinite(got[rows]).all())
    assert torch.equal(got[rows], clean[rows])


def test_a_key_that_is_nan_reaches_the_rows_that_see_it(gpu):
    cache = Int4KVCache(4, 1, 64, page_size=16)
    _fill(cache, 4)
    batch = Batch(cache, [20], [20], seed=1)
    page, slot = int(batch.host_table[0, 0]), 7
    for scales in (cache.k_scales, cache.v_scales):
        _fill(cache, 4)
        scales[page, 0, slot] = math.nan
        got = cache.attend(_queries(20, 1, 64, F16, 1), *batch.args)
        assert bool(torch.isfinite(got[:7]).all()) and bool(torch.isnan(got[7:]).all())


@pytest.mark.parametrize("kind", [F32, F16, BF16])
def test_large_and_small_scores(gpu, kind):
    """One key decides, or all weigh the same."""
    cache = Int4KVCache(16, 1, 128, page_size=32)
    batch = Batch(cache, [201], [2], seed=5)
    for size in (0.0, 1e-6, 30.0, 3000.0 if kind != F16 else 300.0):
        _fill(cache, 7, spread=2.0)
        q = _queries(2, 8, 128, kind, 8, size=size)
        got, lse = cache.attend(q, *batch.args, return_lse=True)
        _check(cache, batch, q, got, lse)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
def test_value_scales_far_apart(gpu, kind):
    """Rows of zeros under large scales, others 2^-24 of them."""
    cache = Int4KVCache(16, 1, 128, page_size=32)
    batch = Batch(cache, [201], [2], seed=5)
    _fill(cache, 7, spread=2.0)
    cache.v_scales.mul_(torch.exp2(torch.randint(-12, 13, cache.v_scales.shape, generator=_rng(1)).float()).cuda())
    cache.v_codes[::2, :, ::3] = 0
    q = _queries(2, 8, 128, kind, 8)
    _check(cache, batch, q, cache.attend(q, *batch.args))
    _check(cache, batch, q, cache.attend(q, *batch.args, scale=-0.3), scale=-0.3)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("lengths,new", [([5000], [1]), ([4097, 300, 2600], [1, 1, 1]), ([2500, 40], [9, 3]),
                                         ([3000] + [20] * 300, [1] * 301)])
def test_split_sequences(gpu, kind, lengths, new):
    """Long sequences whose keys are shared among workgroups and joined."""
    cache = Int4KVCache(sum(-(-n // 64) for n in lengths), 2, 128, page_size=64)
    _fill(cache, 2)
    batch = Batch(cache, lengths, new, seed=2)
    q = _queries(batch.rows, 4, 128, kind, 3)
    got, lse = cache.attend(q, *batch.args, return_lse=True)
    _check(cache, batch, q, got, lse)
    for _ in range(3):
        assert torch.equal(cache.attend(q, *batch.args), got)


def test_pool_past_32_bit_offsets(gpu):
    """Pages whose codes lie more than 2^32 bytes into the pool."""
    cache = Int4KVCache(2200, 8, 256, page_size=2048)  # 4.6 GB of key codes
    assert cache.k_codes.numel() > 2**32
    lengths = [2048 + 100, 77]
    table = torch.tensor([[2199, 2190], [2150, -1]], dtype=torch.int32)
    batch = Batch(cache, [1], [1])
    batch.host_table, batch.table = table, table.cuda()
    batch.host_lengths, batch.new = lengths, lengths
    batch.host_offsets = np.array([0, lengths[0], sum(lengths)], np.int32)
    batch.offsets = torch.from_numpy(batch.host_offsets).cuda()
    batch.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    x = torch.randn((sum(lengths), 8, 256), generator=_rng(1)).to(F16).cuda()
    cache.append(x, x, batch.table, batch.lengths, batch.offsets)
    k, v = cache.read(batch.table, batch.lengths, batch.offsets, dtype=F32)
    assert torch.equal(k, v)
    packed = pack_int4_symmetric(x.float().cpu().numpy().reshape(-1, 256), scale_granularity="token")
    exp = packed.values.astype(np.float32) * packed.token_scale[:, None]
    assert torch.equal(k.cpu(), torch.from_numpy(exp).view_as(k))
    q = _queries(2, 8, 256, F32, 2)
    got = cache.attend(q, batch.table, batch.lengths)
    for b, (first, n) in enumerate(((0, lengths[0]), (lengths[0], lengths[1]))):
        kk = k[first:first + n].cpu().double()
        s = torch.einsum("hd,nhd->hn", q[b].cpu().double(), kk) / 16
        exp = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), kk)
        assert float((got[b].cpu().double() - exp).abs().max()) < 2e-5


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_strided_queries_and_outputs(gpu, kind, shift):
    cache = Int4KVCache(16, 2, 96, page_size=16)
    _fill(cache, 1)
    batch = Batch(cache, [60, 33, 7], [20, 1, 3], seed=1)
    fused = torch.randn((batch.rows, 4 * 96 + 50 + shift), generator=_rng(2)).to(kind).cuda()
    q = fused[:, shift:shift + 4 * 96].view(batch.rows, 4, 96)
    out = torch.full((4, batch.rows, 96 + shift + 3), 5.0, dtype=kind, device="cuda")
    view = out.permute(1, 0, 2)[..., shift:shift + 96]
    assert cache.attend(q, *batch.args, out=view) is view
    assert torch.equal(view, cache.attend(q.contiguous(), *batch.args))
    assert bool((out[..., :shift] == 5).all()) and bool((out[..., shift + 96:] == 5).all())


def test_step_on_another_stream_and_in_a_graph(gpu):
    """append and attend captured once, replayed over changing inputs."""
    cache = Int4KVCache(64, 2, 128, page_size=16)
    _fill(cache, 3)
    batch = Batch(cache, [700, 20, 33], [1, 1, 1], seed=4, spare=2, offsets=False)
    q, k, v = (torch.zeros((3, h, 128), dtype=BF16, device="cuda") for h in (8, 2, 2))
    stream = torch.cuda.Stream()

    def step():
        cache.append(k, v, *batch.args)
        return cache.attend(q, *batch.args, return_lse=True)

    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for i in range(5):
        for t, h in ((q, 8), (k, 2), (v, 2)):
            t.copy_(_queries(3, h, 128, BF16, 10 * i + h))
        batch.lengths.copy_(torch.tensor([700 - i, 20 + i, 33 - 7 * i], dtype=torch.int32))
        eager = step()
        torch.cuda.synchronize()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])


# ---------------------------------------------------------------- prompts
#
# Many new tokens per sequence: rows times shared heads reach half a workgroup's
# 256 on average.


def _prompts(dim, page, seed, lengths=(301, 128, 700, 0, 150), new=(301, 128, 130, 0, 97), spare=0):
    cache = Int4KVCache(sum(-(-n // page) for n in lengths) + 2, 2, dim, page_size=page)
    _fill(cache, seed)
    return cache, Batch(cache, list(lengths), list(new), seed=seed, spare=spare)


@pytest.mark.parametrize("kind", [F16, BF16, F32])
@pytest.mark.parametrize("dim,page", [(64, 16), (96, 32), (128, 64), (256, 16)])
@pytest.mark.parametrize("causal,window", [(True, None), (False, None), (True, 70), (False, 200)])
def test_prompts(gpu, kind, dim, page, causal, window):
    cache, batch = _prompts(dim, page, dim)
    q = _queries(batch.rows, 8, dim, kind, 3)
    got, lse = cache.attend(q, *batch.args, causal=causal, window=window, return_lse=True)
    _check(cache, batch, q, got, lse, causal=causal, window=window)
    assert torch.equal(cache.attend(q, *batch.args, causal=causal, window=window), got)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("share", [1, 3, 5, 16])
def test_prompts_of_any_sharing(gpu, kind, share):
    """Tiles of rows that end inside a token's heads."""
    cache, batch = _prompts(128, 16, share, lengths=(400, 333), new=(260, 300))
    q = _queries(batch.rows, 2 * share, 128, kind, 3, size=2.0)
    got, lse = cache.attend(q, *batch.args, return_lse=True)
    _check(cache, batch, q, got, lse)
    _check(cache, batch, q, cache.attend(q, *batch.args, scale=-0.2), scale=-0.2)
    _check(cache, batch, q, cache.attend(q, *batch.args, scale=0.0), scale=0.0)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("width", [0, 3, 300, 700])
def test_prompts_under_masks(gpu, kind, width):
    cache, batch = _prompts(64, 32, 4)
    mask = torch.rand((batch.rows, width + 3), generator=_rng(width)) < 0.5
    mask[::7] = False
    mask[40:300, :128] = False  # whole buffers of keys that most rows do not see
    mask = mask.cuda()[:, 1:1 + width]
    q = _queries(batch.rows, 6, 64, kind, 5)
    got, lse = cache.attend(q, *batch.args, mask=mask, return_lse=True)
    _check(cache, batch, q, got, lse, mask=mask)
    assert not bool(got[::7].any()) and bool((lse[::7] == -math.inf).all())


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("width", [0, 3, 300, 700])
def test_longer_prompts_under_masks(gpu, kind, width):
    """The same where every sequence has two workgroups' rows or more, on average."""
    cache, batch = _prompts(64, 32, 4)
    mask = torch.rand((batch.rows, width + 3), generator=_rng(width)) < 0.5
    mask[::7] = False
    mask[40:300, :128] = False
    mask = mask.cuda()[:, 1:1 + width]
    q = _queries(batch.rows, 12, 64, kind, 5)
    got, lse = cache.attend(q, *batch.args, mask=mask, return_lse=True)
    _check(cache, batch, q, got, lse, mask=mask)
    assert not bool(got[::7].any()) and bool((lse[::7] == -math.inf).all())


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [255, 256, 257, 511, 512, 513, 700])
def test_rows_about_a_workgroup(gpu, kind, dim, rows):
    """Numbers of rows at which tiles are full and other kernels are chosen."""
    cache, batch = _prompts(dim, 64, rows, lengths=(rows + 44,), new=(rows,))
    q = _queries(rows, 2, dim, kind, 4)
    got, lse = cache.attend(q, *batch.args, return_lse=True)
    _check(cache, batch, q, got, lse)


@pytest.mark.parametrize("kind", [F16, BF16])
def test_prompts_over_holes_and_strides(gpu, kind):
    cache, batch = _prompts(96, 16, 6, lengths=(400, 300), new=(270, 300))
    batch.host_table[0, 3], batch.host_table[0, 11], batch.host_table[1, 0] = -1, cache.num_pages, -5
    batch.table = batch.host_table.cuda()
    fused = torch.randn((batch.rows, 4 * 96 + 31), generator=_rng(2)).to(kind).cuda()
    q = fused[:, 5:5 + 4 * 96].view(batch.rows, 4, 96)
    out = torch.full((4, batch.rows, 96 + 3), 5.0, dtype=kind, device="cuda")
    view = out.permute(1, 0, 2)[..., 1:97]
    cache.attend(q, *batch.args, out=view)
    _check(cache, batch, q, view)
    assert bool((out[..., :1] == 5).all()) and bool((out[..., 97:] == 5).all())
    # Rows outside the offsets come out as rows that see nothing.
    more = torch.cat((q[:2], q, q[:3]))
    got, lse = cache.attend(more, batch.table, batch.lengths, batch.offsets + 2, return_lse=True)
    assert torch.equal(got[2:-3], view)
    assert not bool(got[:2].any()) and not bool(got[-3:].any()) and bool((lse[-3:] == -math.inf).all())


@pytest.mark.parametrize("junk", [math.nan, math.inf, 3e38, 1e-38])
def test_prompts_do_not_see_what_is_hidden(gpu, junk):
    """Rows before a spoilt token, and tokens past the end."""
    cache, batch = _prompts(128, 16, 8, lengths=(500,), new=(400,))
    q = _queries(400, 8, 128, BF16, 6)
    clean = cache.attend(q, *batch.args)
    held = torch.zeros((cache.num_pages, 16), dtype=torch.bool)
    for pos in range(300):
        held[int(batch.host_table[0, pos // 16]), pos % 16] = True
    for scales in (cache.k_scales, cache.v_scales):
        scales.transpose(1, 2)[~held.cuda()] = junk
    got = cache.attend(q, *batch.args)
    assert bool(torch.isfinite(got[:200]).all())
    assert torch.equal(got[:200], clean[:200])
    if math.isnan(junk):
        assert bool(torch.isnan(got[200:]).all())


@pytest.mark.parametrize("kind", [F16, BF16])
def test_prompts_of_large_scores(gpu, kind):
    """References that move often, and scores of one key."""
    cache, batch = _prompts(128, 32, 9, lengths=(600, 290), new=(300, 290))
    for size in (0.0, 8.0, 300.0):
        q = _queries(batch.rows, 8, 128, kind, 8, size=size)
        got, lse = cache.attend(q, *batch.args, return_lse=True)
        _check(cache, batch, q, got, lse)


# -------------------------------------------------------------- refusals


def test_refusals(gpu):
    for args, error in (((0, 1, 64), ValueError), ((1, 0, 64), ValueError), ((1, 1, 80), NotImplementedError),
                        ((1, 1, 64, 24), ValueError), ((1, 1, 64, 8), ValueError)):
        with pytest.raises(error):
            Int4KVCache(*args)
    with pytest.raises(ValueError):
        Int4KVCache(1, 1, 64, device="cpu")
    cache = Int4KVCache(4, 2, 64, page_size=16)
    batch = Batch(cache, [5, 6], [1, 1], offsets=False)
    table, lengths, _ = batch.args
    x = torch.zeros((2, 2, 64), device="cuda")
    off = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    ok = (x, x, table, lengths)
    cache.append(*ok)
    for bad in ((x.cpu(), x, table, lengths), (x.double(), x.double(), table, lengths), (x, x.half(), table, lengths),
                (x[:1], x, table, lengths), (x[:, :1], x[:, :1], table, lengths), (x[..., :32], x[..., :32], table, lengths),
                (x, x, table.long(), lengths), (x, x, table, lengths.long()), (x, x, table[0], lengths),
                (x, x, table, lengths[:1]), (x, x, table.cpu(), lengths), (x, x, table, lengths, off[:2]),
                (x, x, table, lengths, off.long()), (x[:1], x[:1], table, lengths),
                (x.transpose(1, 2).contiguous().transpose(1, 2), x, table, lengths)):
        with pytest.raises(ValueError):
            cache.append(*bad)
    q = torch.zeros((2, 4, 64), device="cuda")
    mask = torch.ones((2, 6), dtype=torch.bool, device="cuda")
    for args, kw in (((q[:, :3], table, lengths), {}), ((q, table, lengths), {"window": 0}),
                     ((q, table, lengths), {"scale": math.inf}), ((q, table, lengths), {"mask": mask[:1]}),
                     ((q, table, lengths), {"mask": mask.to(torch.uint8)}), ((q, table, lengths), {"mask": mask.cpu()}),
                     ((q, table, lengths), {"mask": mask.t().contiguous().t()}),
                     ((q, table, lengths), {"out": q.half()}), ((q, table, lengths), {"out": q[:1]}),
                     ((q[:1], table, lengths), {})):
        with pytest.raises(ValueError):
            cache.attend(*args, **kw)
    for kw in ({"rows": 3}, {"dtype": torch.float64}, {"out": (x, x.half())}, {"out": (x, x), "rows": 1}):
        with pytest.raises(ValueError):
            cache.read(table, lengths, **kw)
    # No rows: nothing to do, nothing touched.
    none = (table[:0], lengths[:0])
    cache.append(x[:0], x[:0], *none)
    assert cache.attend(q[:0], *none).shape == (0, 4, 64)
    assert cache.read(*none)[0].shape == (0, 2, 64)


# --------------------------------------------------- product by product
#
# Queries are taken whole, and a probability times its value scale in 16 bits or whole.


def _check_by_products(cache, batch, q, got, got_lse=None, **kw):
    """As _check, by what the products themselves can lose: a score is exact products
    added in single precision (a quarter of the dims, and four roundings of factors), a
    probability times its scale keeps 2^-16 in 16-bit calls.  Every result is the
    rounding of one within that of the expected."""
    out, lse, mass, _ = _expected(cache, batch, q, **kw)
    share, dim = q.shape[1] // cache.kv_heads, cache.head_dim
    scale = abs(kw.get("scale") or dim**-0.5)
    delta = torch.zeros(q.shape[:2], dtype=torch.float64)
    pool_k = _pool(cache)[0].abs()
    for b, (n, m) in enumerate(zip(batch.host_lengths, batch.new)):
        keep = torch.arange(n)
        k = pool_k[batch.host_table[b].long()[keep // cache.page_size], :, keep % cache.page_size]  # [n, heads, dim]
        rows = slice(int(batch.host_offsets[b]), int(batch.host_offsets[b]) + m)
        for h in range(q.shape[1]) if n else ():
            sums = (q[rows, h].cpu().double().abs() @ k[:, h // share].t()).amax(-1) * scale
            delta[rows, h] = 2.0**-24 * (dim / 4 + 4) * sums + 2.0**-23
    sums = 2.0**-24 * (max(batch.host_lengths) / 8 + 16)
    tol = ((2.0**-21 if q.dtype == F32 else 2.0**-16) + 2 * delta[..., None] + 2 * sums) * mass + 1e-30
    got = got.cpu()
    off = ~(((out - tol).to(q.dtype) <= got) & (got <= (out + tol).to(q.dtype)))
    assert not bool(off.any()), (int(off.sum()), float(((got.double() - out).abs() / tol)[off].max()))
    if got_lse is not None:
        seen = ~torch.isinf(lse)
        assert bool(((got_lse.cpu().double() - lse).abs() <= delta + sums + 2.0**-22 * (1 + lse.abs()))[seen].all())


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim,rows", [(64, 1), (128, 1), (128, 9), (256, 3), (128, 300)])
def test_large_queries_over_zero_codes(gpu, kind, dim, rows):
    """A channel of the queries that is far larger than the others weighs nothing
    where the keys' codes are zero."""
    cache = Int4KVCache(12, 1, dim, page_size=32)
    _fill(cache, 3)
    cache.k_codes[..., 5] = 0  # channels 10 and 11
    batch = Batch(cache, [310], [rows], seed=1)
    q = _queries(rows, 8, dim, kind, 2, size=4.0)
    q[..., 10] = 6e4 if kind == F16 else 1e7
    q[..., 11] = 6e4 if kind == F16 else 3e6
    got, lse = cache.attend(q, *batch.args, return_lse=True)
    _check_by_products(cache, batch, q, got, lse)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("lengths,new", [([300], [1]), ([3000], [1]), ([400], [20]), ([700], [300])])
def test_largest_values(gpu, kind, lengths, new):
    """Values up to nearly the largest number of the type, over scores that rise along the keys."""
    cache = Int4KVCache(50, 1, 128, page_size=64)
    _fill(cache, 3)
    batch = Batch(cache, lengths, new, seed=1)
    for pos in range(lengths[0]):
        cache.k_scales[int(batch.host_table[0, pos // 64]), 0, pos % 64] = 0.1 + 0.4 * pos / lengths[0]
    cache.v_scales.fill_(4.5e37)
    q = _queries(batch.rows, 8, 128, kind, 2, size=0.5)
    got, lse = cache.attend(q, *batch.args, return_lse=True)
    _check(cache, batch, q, got, lse)


# ------------------------------------------------ outputs over inputs


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 300]])
def test_outputs_that_overlap(gpu, new):
    """In place of the queries and between them, but not across."""
    cache = Int4KVCache(90, 2, 64, page_size=16)
    _fill(cache, 1)
    batch = Batch(cache, [700, 20, 310], new, seed=1)
    rows = batch.rows
    fused = _queries(rows + 1, 8, 64, BF16, 2)
    exp = cache.attend(fused[:rows, :4], *batch.args)
    q, other = fused[:rows, :4], fused[:rows, 4:]
    assert torch.equal(cache.attend(q, *batch.args, out=other), exp)  # row by row beside q
    for out in (fused[1:, :4], fused[:rows, 1:5], fused[:rows, 3:7], fused.view(-1)[1:1 + rows * 256].view(rows, 4, 64),
                fused.view(-1)[8:].as_strided(q.shape, q.stride()), exp[:1].expand(rows, 4, 64) if rows > 1 else exp[:, :1],
                exp[:, :1].expand(rows, 4, 64)):
        with pytest.raises(ValueError, match="overlap"):
            cache.attend(q, *batch.args, out=out)
    assert torch.equal(cache.attend(q, *batch.args, out=q), exp) and torch.equal(q, exp)
    both = torch.zeros((rows, 2, 2, 64), dtype=BF16, device="cuda")
    k, v = cache.read(*batch.args, rows=rows)
    cache.read(*batch.args, out=(both[:, 0], both[:, 1]))
    assert torch.equal(both[:, 0], k) and torch.equal(both[:, 1], v)
    for out in ((k, k), (k[:1].expand(rows, 2, 64), v), (both[:, 0], both.view(-1)[2:].as_strided(k.shape, both[:, 0].stride()))):
        with pytest.raises(ValueError, match="overlap"):
            cache.read(*batch.args, out=out)


# --------------------------------------------------- rows of no sequence


@pytest.mark.parametrize("kind,new", [(BF16, [1, 2]), (BF16, [300, 700]), (F32, [300, 5]), (F16, [0, 0])])
@pytest.mark.parametrize("before,behind", [(0, 4000), (3000, 0), (129, 1000)])
def test_padded_batches(gpu, kind, new, before, behind):
    """Many rows before the first offset and behind the last, in strided outputs."""
    cache = Int4KVCache(80, 1, 64, page_size=16)
    _fill(cache, 1)
    batch = Batch(cache, [320, 700], new, seed=1)
    rows = before + batch.rows + behind
    q = _queries(rows, 6, 64, kind, 2)
    out = torch.full((rows, 6, 70), 3.0, dtype=kind, device="cuda")
    _, lse = cache.attend(q, batch.table, batch.lengths, batch.offsets + before, out=out[..., 1:65], return_lse=True)
    used = slice(before, before + batch.rows)
    if batch.rows:
        _check(cache, batch, q[used], out[used, :, 1:65], lse[used])
    for loose in (slice(0, before), slice(before + batch.rows, rows)):
        assert not bool(out[loose, :, 1:65].any()) and bool((lse[loose] == -math.inf).all())
    assert bool((out[..., 0] == 3).all()) and bool((out[..., 65:] == 3).all())


# ------------------------------------------ shapes that the others miss


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 192, 256])
@pytest.mark.parametrize("length,new", [(20011, 1), (9100, 3)])
def test_joins_of_many_parts(gpu, kind, dim, length, new):
    """One key/value head: more parts of an item than a wave joins at once."""
    cache = Int4KVCache(-(-length // 128), 1, dim, page_size=128)
    _fill(cache, 2)
    batch = Batch(cache, [length], [new], seed=2)
    q = _queries(new, 8, dim, kind, 3)
    got, lse = cache.attend(q, *batch.args, return_lse=True)
    _check(cache, batch, q, got, lse)
    if kind != F32:
        _check_by_products(cache, batch, q, got, lse)
    mask = torch.zeros((new, length), dtype=torch.bool, device="cuda")
    mask[:, 5000:5002] = True  # two keys of one part
    got, lse = cache.attend(q, *batch.args, mask=mask, return_lse=True)
    _check(cache, batch, q, got, lse, mask=mask)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("causal,window", [(True, None), (False, 50)])
def test_many_tokens_of_192_dims(gpu, kind, causal, window):
    cache = Int4KVCache(64, 2, 192, page_size=16)
    _fill(cache, 6)
    batch = Batch(cache, [75, 64, 0, 130, 5, 33], [75, 1, 0, 37, 5, 2], seed=1)
    q = _queries(batch.rows, 6, 192, kind, 3)
    got, lse = cache.attend(q, *batch.args, causal=causal, window=window, return_lse=True)
    _check(cache, batch, q, got, lse, causal=causal, window=window)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("lengths,new", [((201, 60), (2, 1)), ((700, 400), (600, 400))])
def test_all_bits_of_the_products(gpu, kind, dim, lengths, new):
    """Rows of zeros under large value scales, others 2^-24 of them: single tokens and
    prompts of two workgroups' rows."""
    cache, batch = _prompts(dim, 32, 5, lengths=lengths, new=new)
    q = _queries(batch.rows, 4, dim, kind, 3, size=2.0)
    got, lse = cache.attend(q, *batch.args, return_lse=True)
    _check_by_products(cache, batch, q, got, lse)
    cache.v_scales.mul_(torch.exp2(torch.randint(-12, 13, cache.v_scales.shape, generator=_rng(1)).float()).cuda())
    cache.v_codes[::2, :, ::3] = 0
    _check_by_products(cache, batch, q, cache.attend(q, *batch.args))
    _check_by_products(cache, batch, q, cache.attend(q, *batch.args, scale=-0.3), scale=-0.3)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("size", [2.0**-90, 2.0**-96, 2.0**-110, 2.0**90])
@pytest.mark.parametrize("rows", [1, 300])
def test_queries_of_any_size(gpu, kind, size, rows):
    """Very small queries over large keys, and the other way round."""
    cache = Int4KVCache(12, 1, 128, page_size=32)
    _fill(cache, 3)
    cache.k_scales.mul_(2.0**96 if size < 1 else 2.0**-90)
    batch = Batch(cache, [310], [rows], seed=1)
    q = _queries(rows, 8, 128, kind, 2, size=size)
    got, lse = cache.attend(q, *batch.args, return_lse=True)
    _check(cache, batch, q, got, lse)
    got, lse = cache.attend(q, *batch.args, scale=0.0, return_lse=True)
    _check(cache, batch, q, got, lse, scale=0.0)


@pytest.mark.parametrize("dim,share,rows", [(64, 8, 1), (96, 2, 5), (128, 8, 1), (128, 8, 9), (192, 4, 2), (256, 8, 3),
                                            (128, 8, 70)])
def test_single_precision_queries_are_whole(gpu, dim, share, rows):
    """All bits of a query count, beside a channel far larger than the others too."""
    cache = Int4KVCache(12, 1, dim, page_size=32)
    _fill(cache, 3)
    cache.k_codes[..., 5] = 0  # channels 10 and 11
    batch = Batch(cache, [310], [rows], seed=1)
    q = _queries(rows, share, dim, F32, 2, size=4.0)
    for size in (4.0, 3e7):
        q[..., 10] = size
        q[..., 11] = size / 7
        got, lse = cache.attend(q, *batch.args, return_lse=True)
        _check_by_products(cache, batch, q, got, lse)
