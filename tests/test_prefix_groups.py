"""Groups of requests that hold the same first blocks (BlockManager.prefix_groups): against every way to split."""
import itertools
import random

import numpy as np
import pytest

from kyro_amd import BlockManager, KyroError


def _common(lists):
    n = 0
    for column in zip(*lists):
        if len(set(column)) > 1:
            break
        n += 1
    return n


def _most_saved(lists):
    """The most blocks that any partition into sets with a common start leaves out."""
    if len(lists) < 2:
        return 0
    best = 0
    first, rest = lists[0], lists[1:]
    for k in range(len(rest) + 1):
        for chosen in itertools.combinations(range(len(rest)), k):
            group = [first] + [rest[i] for i in chosen]
            others = [rest[i] for i in range(len(rest)) if i not in chosen]
            saved = (len(group) - 1) * _common(group) if len(group) > 1 else 0
            best = max(best, saved + _most_saved(others))
    return best


def _check(bm, ids):
    order, starts, blocks = bm.prefix_groups(ids)
    assert order.dtype == starts.dtype == blocks.dtype == np.int32
    assert sorted(order.tolist()) == list(range(len(ids)))
    assert starts[0] == 0 and starts[-1] == len(ids) and len(starts) == len(blocks) + 1
    assert (np.diff(starts) > 0).all()
    lists = [bm.request(r)[0] for r in ids]
    saved = 0
    for g in range(len(blocks)):
        members = [lists[order[i]] for i in range(starts[g], starts[g + 1])]
        if len(members) == 1:
            assert blocks[g] == 0
        else:
            assert 0 < blocks[g] == _common(members) or blocks[g] == 0 == _common(members)
            saved += (len(members) - 1) * int(blocks[g])
    return lists, saved


def _prompts(bm, prompts):
    """Requests with these prompts, whose whole blocks the cache hands on."""
    ids = []
    for i, p in enumerate(prompts):
        assert bm.allocate_with_prefix(i, p) is not None
        bm.free(i)
    for i, p in enumerate(prompts):
        assert bm.allocate_with_prefix(100 + i, list(p) + [90000 + i]) is not None
        ids.append(100 + i)
    bm.take_copies()
    return ids


def test_a_common_prompt_is_one_group():
    bm = BlockManager(4, 256)
    system = list(range(1000, 1012))  # three blocks
    ids = _prompts(bm, [system + [i * 10 + j for j in range(5)] for i in range(4)] + [[7] * 9])
    order, starts, blocks = bm.prefix_groups(ids)
    lists, saved = _check(bm, ids)
    assert saved == 9
    big = int(np.argmax(np.diff(starts)))
    assert sorted(order[starts[big]:starts[big + 1]].tolist()) == [0, 1, 2, 3] and blocks[big] == 3


def test_the_longer_prefix_of_few_or_the_shorter_of_many():
    # Six requests share 2 blocks; two of them share 8. As one group they leave out 10 blocks, as 2 and 4 6 + 8.
    bm = BlockManager(2, 512)
    short = [1, 2, 3, 4]
    long_ = short + list(range(20, 32))
    ids = _prompts(bm, [long_ + [50 + i, 60] for i in range(2)] + [short + [70 + i, 80] for i in range(4)])
    _, saved = _check(bm, ids)
    assert saved == 8 + 3 * 2
    # With three blocks instead of eight the one group wins: 10 against 3 + 6.
    bm = BlockManager(2, 512)
    ids = _prompts(bm, [short + [9, 9, 50 + i, 60] for i in range(2)] + [short + [70 + i, 80] for i in range(4)])
    _, saved = _check(bm, ids)
    assert saved == 10


@pytest.mark.parametrize("seed", range(20))
def test_no_other_groups_leave_out_more(seed):
    rng = random.Random(seed)
    bm = BlockManager(2, 4096)
    prompts = [[rng.randint(1, 2) for _ in range(2 * rng.randint(1, 6))] for _ in range(rng.randint(1, 6))]
    ids = _prompts(bm, prompts)
    rng.shuffle(ids)
    lists, saved = _check(bm, ids)
    assert saved == _most_saved(lists)


def test_one_none_and_the_same_request_twice():
    bm = BlockManager(4, 64)
    order, starts, blocks = bm.prefix_groups([])
    assert order.size == 0 and starts.tolist() == [0] and blocks.size == 0
    assert bm.allocate(5, 9)
    order, starts, blocks = bm.prefix_groups([5])
    assert order.tolist() == [0] and starts.tolist() == [0, 1] and blocks.tolist() == [0]
    order, starts, blocks = bm.prefix_groups([5, 5])
    assert order.tolist() == [0, 1] and starts.tolist() == [0, 2] and blocks.tolist() == [3]


def test_a_request_that_is_not_there_is_an_error():
    bm = BlockManager(4, 64)
    with pytest.raises(KyroError):
        bm.prefix_groups([1])


def test_many_requests_nested_deeply():
    bm = BlockManager(1, 70000)
    prompt = list(range(1, 301))
    assert bm.allocate_with_prefix(0, prompt) is not None
    bm.free(0)
    ids = []
    for i in range(300):  # request i shares i + 1 blocks with those behind it
        assert bm.allocate_with_prefix(1 + i, prompt[: i + 1] + [100000 + i]) is not None
        ids.append(1 + i)
    bm.take_copies()
    lists, saved = _check(bm, ids)
    # n of the longest as one group of 301 - n blocks; the rest in groups of their own.
    assert saved >= max((n - 1) * (301 - n) for n in range(2, 301))
