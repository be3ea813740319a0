"""CachePages against lists: whole state after every update."""
import random

import pytest
import torch

from maxsim_amd import CachePages

pytestmark = pytest.mark.gpu


class Lists:
    """The same with a list of pages per sequence and a list for the stack."""

    def __init__(self, num_pages, batch, max_pages, page):
        self.stack = list(range(num_pages - 1, -1, -1))
        self.owned = [[] for _ in range(batch)]
        self.lengths = [0] * batch
        self.num_pages, self.max_pages, self.page = num_pages, max_pages, page

    def update(self, new, cut, rows):
        page, back = self.page, []
        for b, pages in enumerate(self.owned):
            if cut is not None:
                self.lengths[b] = min(self.lengths[b], max(cut[b], 0))
            stay = -(-self.lengths[b] // page)
            back += pages[stay:]
            del pages[stay:]
        self.stack += back[::-1]
        offsets, positions, slots = [0], [], []
        asked_rows = asked_pages = 0
        had = len(self.stack)
        for b, pages in enumerate(self.owned):
            n = max(new[b], 0) if new is not None else 0
            if self.lengths[b] + n > self.max_pages * page:
                n = 0
            asked_rows += n
            if asked_rows > rows:
                n = 0
            need = -(-(self.lengths[b] + n) // page) - len(pages)
            asked_pages += need
            if need and asked_pages > had:
                n = need = 0
            pages += [self.stack.pop() for _ in range(need)]
            for p in range(self.lengths[b], self.lengths[b] + n):
                positions.append(p)
                slots.append(pages[p // page] * page + p % page)
            self.lengths[b] += n
            offsets.append(offsets[-1] + n)
        spare = [-1] * (rows - len(positions))
        return offsets, positions + spare, slots + spare

    def check(self, pages):
        table = torch.full((len(self.owned), self.max_pages), -1, dtype=torch.int32)
        for b, own in enumerate(self.owned):
            table[b, :len(own)] = torch.tensor(own, dtype=torch.int32)
        free = torch.tensor(self.stack + [-1] * (self.num_pages - len(self.stack)), dtype=torch.int32)
        assert torch.equal(pages.lengths.cpu(), torch.tensor(self.lengths, dtype=torch.int32))
        assert torch.equal(pages.table.cpu(), table)
        assert torch.equal(pages.free.cpu(), free)
        assert pages.free_count.cpu().tolist() == [len(self.stack)]


def _dev(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32).cuda()


def _step(pages, lists, new, cut, rows):
    got = pages.update(_dev(new), lengths=_dev(cut), rows=rows)
    want = lists.update(new, cut, rows)
    for g, w, kind in zip(got, want, (torch.int32, torch.int32, torch.int64)):
        assert torch.equal(g.cpu(), torch.tensor(w, dtype=kind))
    lists.check(pages)


@pytest.mark.parametrize("batch,max_pages,page,num_pages", [
    (1, 1, 16, 1), (1, 300, 16, 250), (5, 9, 16, 30), (63, 20, 32, 700), (64, 40, 64, 2000), (65, 11, 16, 300),
    (1023, 4, 16, 3000), (1024, 6, 128, 5000), (1025, 5, 16, 2600), (2500, 7, 16, 9000)])
def test_steps(gpu, batch, max_pages, page, num_pages):
    rng = random.Random(batch * 7 + page)
    pages = CachePages(num_pages, batch, max_pages, page_size=page)
    lists = Lists(num_pages, batch, max_pages, page)
    lists.check(pages)
    most = max_pages * page
    for step in range(8):
        kind = step % 4
        new = [rng.choice([0, 1, rng.randint(0, most)]) if kind == 0 else rng.randint(0, 9) if kind == 1
               else rng.choice([1, 1, -3, most + 1, 2**31 - 1]) if kind == 2 else 1 for _ in range(batch)]
        cut = None
        if step % 3:
            cut = [rng.choice([n, n - rng.randint(0, 20), 0, 2**31 - 1, -5]) if rng.random() < 0.5 else n
                   for n in lists.lengths]
        total = sum(min(max(n, 0), most) for n in new)
        rows = rng.choice([total, total + 7, total // 2, total])
        _step(pages, lists, new, cut, rows)
    _step(pages, lists, None, [0] * batch, 0)  # all of it comes back
    assert len(lists.stack) == num_pages


@pytest.mark.parametrize("rows", [4095, 4096, 4097, 9000])
def test_rows_of_either_launch(gpu, rows):
    pages, lists = CachePages(900, 7, 100, page_size=16), Lists(900, 7, 100, 16)
    _step(pages, lists, [3, 0, 17, 1, 0, 16, 1], None, rows)
    _step(pages, lists, [rows - 2000, 200, 0, 1000, 500, 0, 300], None, rows)


def test_a_pool_that_runs_out(gpu):
    pages, lists = CachePages(10, 4, 8, page_size=16), Lists(10, 4, 8, 16)
    _step(pages, lists, [64, 64, 32, 1], None, 161)  # ten pages go to the first three
    assert pages.lengths.tolist() == [64, 64, 32, 0]
    _step(pages, lists, [0, 1, 0, 1], None, 2)
    assert pages.lengths.tolist() == [64, 64, 32, 0]
    # One page back: the second takes it, the last waits; who needs none goes on.
    _step(pages, lists, [3, 16, 3, 16], [40, 64, 30, 0], 38)
    assert pages.lengths.tolist() == [43, 80, 30, 0]
    _step(pages, lists, [1, 1, 1, 1], [0, 0, 0, 0], 4)


def test_numbers_and_capacities(gpu):
    pages, lists = CachePages(50, 6, 5, page_size=16), Lists(50, 6, 5, 16)
    got = pages.update(9)
    want = lists.update([9] * 6, None, 54)
    assert all(g.tolist() == w for g, w in zip(got, want))
    got = pages.update(torch.tensor([1, -2, 0, 3, 0, 2], dtype=torch.int32).cuda())
    want = lists.update([1, 0, 0, 3, 0, 2], None, 6)
    assert all(g.tolist() == w for g, w in zip(got, want))
    got = pages.update(lengths=pages.lengths - 5)
    want = lists.update(None, [n - 5 for n in lists.lengths], 0)
    assert all(g.tolist() == w for g, w in zip(got, want))
    lists.check(pages)
    got = pages.update(lengths=pages.lengths)  # cuts nothing
    assert got[0].tolist() == [0] * 7 and got[1].shape == got[2].shape == (0,)
    lists.check(pages)


def test_states_that_hold_no_pages(gpu):
    """Numbers that a program wrote into the state stay numbers: nothing is read or written through them."""
    pages = CachePages(8, 3, 4, page_size=16)
    pages.lengths.copy_(torch.tensor([-7, 2**31 - 1, 20], dtype=torch.int32))
    pages.free_count.fill_(2**31 - 1)
    offsets, positions, slots = pages.update(1, lengths=_dev([5, 64, 20]))
    assert offsets.tolist() == [0, 1, 1, 2] and positions.tolist() == [0, 20, -1]
    assert slots.tolist()[1:] == [-1, -1]  # the third sequence's entry was none
    pages.free_count.fill_(-4)
    pages.update(1, lengths=_dev([0, 0, 0]))
    assert 0 <= int(pages.free_count) <= 8


def test_graph_replays(gpu):
    pages, lists = CachePages(300, 20, 16, page_size=16), Lists(300, 20, 16, 16)
    new, cut = _dev([0] * 20), _dev([0] * 20)
    pages.update(new, lengths=cut, rows=400)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pages.update(new, lengths=cut, rows=400)
    rng = random.Random(3)
    for _ in range(6):
        n = [rng.randint(0, 25) for _ in range(20)]
        c = [max(0, m - rng.randint(0, 12)) for m in lists.lengths]
        new.copy_(_dev(n))
        cut.copy_(_dev(c))
        graph.replay()
        torch.cuda.synchronize()
        want = lists.update(n, c, 400)
        assert all(g.tolist() == w for g, w in zip(out, want))
        lists.check(pages)


def test_another_stream(gpu):
    pages, lists = CachePages(300, 20, 16, page_size=16), Lists(300, 20, 16, 16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for n in (40, 3, 60):
            _step(pages, lists, [n] * 20, None, 20 * n)


def test_refusals(gpu):
    for args, kw in (((0, 1, 1), {}), ((1, 0, 1), {}), ((1, 1, 0), {}), ((4, 2, 2), {"page_size": 24}),
                     ((4, 2, 2), {"page_size": 8}), ((4, 2, 2), {"device": "cpu"})):
        with pytest.raises(ValueError):
            CachePages(*args, **kw)
    for args, kw in (((2**31, 1, 1), {}), ((4, 2**16, 2**15), {}), ((4, 1, 2**27 - 256), {"page_size": 16})):
        with pytest.raises(NotImplementedError):
            CachePages(*args, **kw)
    pages = CachePages(8, 3, 4, page_size=16)
    three = torch.ones(3, dtype=torch.int32, device="cuda")
    for new, kw in (([1, 1, 1], {}), ([1, 1, 1], {"rows": 3}), (three.long(), {"rows": 3}), (three[:2], {"rows": 2}), (three.cpu(), {"rows": 3}), (-1, {}),
                    (three, {"rows": -1}), (three, {"lengths": three.long(), "rows": 3}),
                    (three, {"lengths": three[:1], "rows": 3}), (three.repeat(2)[::2], {"rows": 3})):
        with pytest.raises(ValueError):
            pages.update(new, **kw)
    with pytest.raises(NotImplementedError):
        pages.update(three, rows=2**26 + 1)
    assert pages.lengths.tolist() == [0, 0, 0] and pages.free_count.tolist() == [8]
