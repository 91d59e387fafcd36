"""Groups of requests that hold the same first blocks: batches whose best groups take a run of lists apart."""
import random

import pytest

from kyro_amd import BlockManager
from tests.test_prefix_groups import _check, _most_saved, _prompts


def _saved(prompts, block_size=1):
    bm = BlockManager(block_size, 65536)
    ids = _prompts(bm, prompts)
    lists, saved = _check(bm, ids)
    return lists, saved


def test_a_deep_group_stays_and_a_list_beside_it_joins_the_outer_one():
    lists, saved = _saved([[int(x) for x in p] for p in ("1121111111", "12", "112111", "11111121122")])
    assert saved == _most_saved(lists) == 7


def test_two_deep_lists_and_three_that_share_less():
    deep = [1, 2, 3] + list(range(11, 18))
    lists, saved = _saved([deep + [101], deep + [102], [1, 2, 3, 201], [1, 2, 3, 202], [1, 2, 301]])
    assert saved == _most_saved(lists) == 14


def test_what_joins_depends_on_how_deep_the_outer_group_is():
    """A run inside two others: with the middle one as a group its lists join that, without it the outer one."""
    for middle in range(2, 12):
        for extra in range(4):
            front = [1] + [2] * middle
            prompts = [front + [3] * 6 + [100 + i] for i in range(2)] + [front + [200 + i] for i in range(extra)] + \
                [[1, 300 + i] for i in range(2)]
            lists, saved = _saved(prompts)
            assert saved == _most_saved(lists), (middle, extra)


@pytest.mark.parametrize("seed", range(150))
def test_random_batches_that_share_deeply(seed):
    rng = random.Random(seed)
    # Three of four tokens are the same, so that runs lie deep inside each other.
    prompts = [[rng.choice((1, 1, 1, 2)) for _ in range(rng.randint(1, 12))] for _ in range(rng.randint(4, 7))]
    lists, saved = _saved(prompts)
    assert saved == _most_saved(lists)


def _best(lists):
    """The most blocks left out, by the tree of common starts: a list counts for the deepest open start above it, and an
    open start costs its own length once."""
    def walk(members, depth, above):
        # members agree in their first `depth` blocks; `above`: length of the nearest open start
        rest, by = [], {}
        for x in members:
            by.setdefault(x[depth], []).append(x) if len(x) > depth else rest.append(x)
        if not rest and len(by) == 1:
            return walk(members, depth + 1, above)
        def parts(a):
            total = len(rest) * a
            for group in by.values():
                total += a if len(group) == 1 else walk(group, depth + 1, a)
            return total
        return max(parts(above), parts(depth) - depth) if depth else parts(above)
    return walk([tuple(x) for x in lists], 0, 0) if lists else 0


@pytest.mark.parametrize("seed", range(10))
def test_larger_batches(seed):
    rng = random.Random(1000 + seed)
    prompts = [[1] * rng.randint(1, 6)]
    while len(prompts) < 40:  # each goes on from a part of an earlier one
        base = rng.choice(prompts)
        prompts.append(base[: rng.randint(1, len(base))] + [len(prompts) * 100 + j for j in range(rng.randint(0, 6))])
    lists, saved = _saved(prompts)
    assert saved == _best(lists)


def test_a_long_chain_of_nested_starts():
    """800 requests, each of which shares one block more with those behind it than the one before."""
    n = 800
    bm = BlockManager(1, 8 * n)
    prompt = list(range(1, n + 1))
    assert bm.allocate_with_prefix(0, prompt) is not None
    bm.free(0)
    ids = []
    for i in range(n):
        assert bm.allocate_with_prefix(1 + i, prompt[: i + 1] + [100000 + i]) is not None
        ids.append(1 + i)
    bm.take_copies()
    _, saved = _check(bm, ids)
    # Request i counts for the longest open start of at most i + 1 blocks. best[d]: the most that the requests from
    # d - 1 on leave out with the start of d blocks open.
    best = [0] * n
    for d in range(n - 1, 0, -1):
        best[d] = max([(n - d + 1) * d - d] + [(e - d) * d - d + best[e] for e in range(d + 1, n)])
    assert saved == max(best)
