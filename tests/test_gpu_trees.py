"""Trees of drafted tokens whose positions lie far from their keys', and the bounds that
windows with sinks and trees share with the other calls over the cache."""
import pytest
import torch
from test_gpu_drafts import _check
from test_gpu_kvcache import BF16, F16, Batch, _fill, _queries

from maxsim_amd import Int4KVCache

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
