"""Entries that extend leaves out, and what the rest of a step makes of them: keep leaves them alone, whether they bring
rows or not, and a pool that ran out is reported as such by the sync behind the whole step."""
import pytest
import torch

import kyro_amd
from kyro_amd import RequestTables, _lib

pytestmark = pytest.mark.gpu

BS = 16


def i32(x, gpu):
    return torch.tensor(list(x), dtype=torch.int32, device=gpu)


def snapshot(t):
    return [x.clone() for x in (t.requests, t.blocks, t.pool, t.pool_count)]


def same(t, before):
    return all(torch.equal(x, y) for x, y in zip((t.requests, t.blocks, t.pool, t.pool_count), before))


def state(gpu, rows):
    """Requests 0 to 5 of 50, 100, 20, 5, 60 and 0 tokens; 4 holds 2 shared blocks, 5 the two blocks of an extend that no
    keep followed. `rows` state rows: past 32768 of them extend is two launches."""
    t = RequestTables.new(BS, rows=rows, max_blocks=8, pool=range(30), num_blocks=40, device=gpu)
    t.admit(4, [35, 36], 20)
    who, new = i32([0, 1, 2, 3, 4], gpu), i32([50, 100, 20, 5, 40], gpu)
    step = t.extend(who, new, total_q=215)
    t.keep(who, step.context_lens, step.q_start_loc, new)
    t.extend(i32([5], gpu), i32([30], gpu), total_q=30)
    assert t.requests[:6, :3].tolist() == [[50, 4, 0], [100, 7, 0], [20, 2, 0], [5, 1, 0], [60, 4, 2], [0, 2, 0]]
    return t


@pytest.mark.parametrize("rows", [8, 40000])
@pytest.mark.parametrize("who, new, total, width, ctx, lens", [
    # a table narrower than the context of a request that brings nothing
    ([0, 1, 4], [1, 0, 2], 3, 4, [51, 0, 62], [51, 0, 61]),
    # rows below 0, which count as 0
    ([0, 1, 4], [1, -1, 2], 3, 8, [51, 0, 62], [51, 0, 61]),
    ([0, 5, 4], [1, -3, 2], 3, 8, [51, 0, 62], [51, 0, 61]),
    # rows past max_rows: all behind them are left out, those without rows too
    ([0, 1, 4, 2, 5], [1, 20, 0, 0, 0], 10, 8, [51, 0, 0, 0, 0], [51, 0, 0, 0, 0])])
def test_keep_leaves_refused_entries_without_rows_alone(gpu, rows, who, new, total, width, ctx, lens):
    t = state(gpu, rows)
    srows = i32(who, gpu)
    step = t.extend_async(srows, i32(new, gpu), total_q=total, max_blocks_per_seq=width)
    before = snapshot(t)
    kept = t.keep_async(srows, step.context_lens, step.q_start_loc, i32([0] * len(who), gpu), plus=1)
    with pytest.raises(kyro_amd.KyroError) as e:
        kyro_amd.sync()
    assert e.value.status == _lib.KYRO_EINVAL
    assert step.context_lens.tolist() == ctx and kept.tolist() == lens
    for r, n in zip(who, lens):  # served entries count their first row, and no block is free for it
        if n:
            before[0][r, 0] = n
    assert same(t, before)
    # The next step goes on from there.
    step = t.extend(i32([1, 4, 5], gpu), i32([1, 1, 30], gpu), total_q=32)
    assert step.context_lens.tolist() == [101, int(before[0][4, 0]) + 1, 30]
    assert step.positions[:2].tolist() == [100, int(before[0][4, 0])]


@pytest.mark.parametrize("rows", [8, 40000])
def test_keep_of_entries_without_rows(gpu, rows):
    """Served ones: the length stays, and blocks that an extend took for more rows go back; an empty request keeps what it
    holds until it brings rows or ends."""
    t = state(gpu, rows)
    t.extend(i32([2], gpu), i32([40], gpu), total_q=40)
    assert t.requests[2].tolist() == [20, 4, 0, 0]
    srows = i32([2, 5, 3, -1], gpu)
    step = t.extend(srows, i32([0, 0, 0, 0], gpu), total_q=0)
    before = snapshot(t)
    lens = t.keep(srows, step.context_lens, step.q_start_loc, i32([7, 7, 7, 7], gpu), plus=3)
    assert lens.tolist() == [20, 0, 5, 0]
    at = int(before[3])
    before[2][at:at + 2] = before[1][2, 2:4]
    before[3] += 2
    before[0][2, 1] = 2
    assert same(t, before)


def test_lengths_near_two_to_the_31(gpu):
    """A block of 1.5e9 tokens: length and block size together pass 31 bits."""
    bs, tokens = 1_500_000_000, 1_400_000_000
    t = RequestTables.new(bs, rows=1, max_blocks=1, pool=[0], num_blocks=1, device=gpu)
    t.requests[0] = i32([tokens, 1, 0, 0], gpu)
    t.pool_count.zero_()
    step = t.extend(None, i32([3], gpu), total_q=3)
    assert step.context_lens.tolist() == [tokens + 3] and step.slots.tolist() == [tokens, tokens + 1, tokens + 2]
    assert t.keep(None, step.context_lens, step.q_start_loc, i32([2], gpu)).tolist() == [tokens + 2]
    assert t.requests.tolist() == [[tokens + 2, 1, 0, 0]] and t.pool_count.item() == 0
