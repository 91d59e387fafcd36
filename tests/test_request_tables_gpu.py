"""Block tables on the GPU against a restatement with loops: whole numbers, so every comparison is for equality."""
import numpy as np
import pytest
import torch

import kyro_amd
from kyro_amd import RequestTables, StepTables, _lib

pytestmark = pytest.mark.gpu


class Model:
    """The state on the host, and the calls on it one entry after the other."""

    def __init__(self, bs, rows, max_blocks, pool):
        self.bs, self.max_blocks = bs, max_blocks
        self.requests = np.zeros((rows, 4), np.int64)
        self.blocks = np.zeros((rows, max_blocks), np.int64)
        self.pool = np.array(list(pool), np.int64)
        self.count = len(self.pool)

    def extend(self, state_rows, new, width, total_q):
        B = len(new)
        table, ctx = np.zeros((B, width), np.int64), np.zeros(B, np.int64)
        start = np.concatenate([[0], np.cumsum(np.maximum(new, 0))])
        positions, slots = np.full(total_q, -1), np.full(total_q, -1)
        asked, count = 0, self.count
        for b, (r, m) in enumerate(zip(state_rows, new)):
            good = 0 <= r < len(self.requests) and list(state_rows).count(r) == 1 and m >= 0 and start[b + 1] <= total_q
            if not good:
                continue
            n, held = int(self.requests[r, 0]), int(self.requests[r, 1])
            if n + m > min(width, self.max_blocks) * self.bs:
                continue
            need = max(0, -(-(n + m) // self.bs) - held)
            asked += need
            if need and asked > count:
                continue
            for _ in range(need):
                self.count -= 1
                self.blocks[r, held] = self.pool[self.count]
                held += 1
            self.requests[r, 1] = held
            ctx[b] = n + m
            table[b, : min(held, width)] = self.blocks[r, : min(held, width)]
            for j in range(m):
                p = n + j
                positions[start[b] + j] = p
                slots[start[b] + j] = self.blocks[r, p // self.bs] * self.bs + p % self.bs
        return table, ctx, start, positions, slots

    def shrink(self, r, tokens, stay):
        for i in range(stay, int(self.requests[r, 1])):
            self.pool[self.count] = self.blocks[r, i]
            self.count += 1
        self.requests[r, 0], self.requests[r, 1] = tokens, min(stay, int(self.requests[r, 1]))

    def keep(self, state_rows, ctx, start, kept, plus=0):
        out = np.zeros(len(ctx), np.int64)
        for b, r in enumerate(state_rows):
            m = start[b + 1] - start[b]
            k = kept[b] + plus if m else 0
            if r < 0 or ctx[b] < m or not 0 <= k <= m:
                continue
            out[b] = ctx[b] - m + k
            self.shrink(r, out[b], max(-(-int(out[b]) // self.bs), int(self.requests[r, 2])))
        return out

    def release(self, state_rows):
        for r in state_rows:
            if r >= 0:
                self.shrink(r, 0, int(self.requests[r, 2]))
                self.requests[r] = 0


def pair(gpu, bs, rows, max_blocks, pool, num_blocks=None):
    pool = list(pool)
    t = RequestTables.new(bs, rows=rows, max_blocks=max_blocks, pool=pool, num_blocks=num_blocks or max(pool, default=0) + 1, device=gpu)
    return t, Model(bs, rows, max_blocks, pool)


def i32(x, gpu):
    return torch.tensor(list(map(int, x)), dtype=torch.int32, device=gpu)


def same_state(t, m):
    assert np.array_equal(t.requests.cpu().numpy(), m.requests)
    assert np.array_equal(t.blocks.cpu().numpy(), m.blocks)
    assert np.array_equal(t.pool.cpu().numpy(), m.pool)
    assert t.pool_count.item() == m.count


def same_step(step, want):
    for name, x in zip(StepTables._fields, want):
        assert np.array_equal(getattr(step, name).cpu().numpy(), x), name


# (block size, batch, state rows, most tokens, most rows, table width beyond the longest): within the one-launch
# form's bounds and past each of them (1024 entries, 16384 table entries, 4096 rows, 32768 state rows)
SIZES = [(16, 1, 1, 40, 1, 0), (16, 7, 9, 300, 40, 3), (1, 30, 33, 90, 5, 0), (24, 64, 80, 4000, 9, 90), (16, 1024, 1030, 200, 2, 2),
         (16, 1025, 1025, 200, 2, 0), (32, 2500, 3000, 100, 3, 0), (64, 8, 8, 150000, 8, 0), (16, 3, 3, 100, 2500, 0),
         (16, 12, 40000, 300, 9, 0), (8, 5, 131072, 33000, 2, 0)]


@pytest.mark.parametrize("bs,B,R,most,rows,wide", SIZES, ids=lambda x: str(x))
def test_steps_of_a_serving_loop(gpu, bs, B, R, most, rows, wide):
    """Five steps: some of the batch extends, keeps some rows, requests end and new ones with shared blocks come."""
    rng = np.random.RandomState(bs * 1000 + B)
    width = -(-(most + 5 * rows) // bs) + 1
    t, m = pair(gpu, bs, R, width, rng.permutation(B * width * 2 + 7)[: B * width + 5], num_blocks=B * width * 2 + 7)
    live = rng.choice(R, B, replace=False)
    for r in live[: 200]:
        n = rng.randint(0, most + 1)
        ids = np.arange(-(-n // bs))
        t.admit(r, ids, n)
        m.requests[r, :3], m.blocks[r, : len(ids)] = (n, len(ids), len(ids)), ids
    for step_no in range(5):
        batch = rng.permutation(live)[: max(1, B - step_no)]
        batch[len(batch) // 2:] = np.where(rng.rand(len(batch) - len(batch) // 2) < 0.1, -1, batch[len(batch) // 2:])
        new = np.where(batch < 0, 0, rng.randint(0, rows + 1, len(batch)))
        total = int(new.sum()) + (step_no % 2) * 3
        step = t.extend(i32(batch, gpu), i32(new, gpu), total_q=total, max_blocks_per_seq=width + wide)
        want = m.extend(batch, new, width + wide, total)
        same_step(step, want)
        same_state(t, m)
        kept = rng.randint(0, np.maximum(new, 1))
        kept[new == 0] = 99  # not read
        plus = step_no % 2
        lens = t.keep(i32(batch, gpu), step.context_lens, step.q_start_loc, i32(kept, gpu), plus=plus)
        assert np.array_equal(lens.cpu().numpy(), m.keep(batch, want[1], want[2], kept, plus))
        same_state(t, m)
        ended = rng.permutation(live)[: B // 3]
        t.release(i32(list(ended) + [-1], gpu))
        m.release(ended)
        same_state(t, m)
    assert sorted(m.pool[: m.count].tolist() + [b for r in range(R) for b in m.blocks[r, m.requests[r, 2]:m.requests[r, 1]]]) == \
        sorted(set(m.pool[: m.count].tolist() + [b for r in range(R) for b in m.blocks[r, m.requests[r, 2]:m.requests[r, 1]]]))


@pytest.mark.parametrize("wide", [0, 40000])
def test_repeated_calls_change_nothing_more(gpu, wide):
    t, m = pair(gpu, 16, 4, 8, range(20))
    rows, new = [2, 0, 3], [17, 16, 0]
    kw = dict(total_q=33, max_blocks_per_seq=8 + wide)
    for _ in range(2):
        step = t.extend(i32(rows, gpu), i32(new, gpu), **kw)
    want = m.extend(rows, new, 8 + wide, 33)
    same_step(step, want)
    same_state(t, m)
    for _ in range(2):
        lens = t.keep(i32(rows, gpu), step.context_lens, step.q_start_loc, i32([3, 16, 0], gpu))
    assert lens.tolist() == m.keep(rows, want[1], want[2], [3, 16, 0]).tolist() == [3, 16, 0]
    same_state(t, m)


# Blocks needed: 1, 2, 2, 0, 1 of the pool's 5, so that the last one is one too many; or 1, 2, 3, 0, 1, where the third
# request gets none, and neither does the last, though a block would be left for it.
@pytest.mark.parametrize("third, served", [(40, 60), (50, 0)])
@pytest.mark.parametrize("wide", [0, 40000])
def test_a_pool_that_runs_out(gpu, wide, third, served):
    """In the order of the batch; a request that needs no block is served. The error is that of space, once."""
    t, m = pair(gpu, 16, 6, 8, range(5))
    for r in range(6):
        t.admit(r, [9, 8], 20)
        m.requests[r, :3], m.blocks[r, :2] = (20, 2, 2), (9, 8)
    t.num_blocks = 10
    rows, new, total = [0, 1, 2, 3, 4], [16, 30, third, 12, 13], 71 + third
    with pytest.raises(kyro_amd.KyroError) as e:
        t.extend(i32(rows, gpu), i32(new, gpu), total_q=total, max_blocks_per_seq=8 + wide)
    assert e.value.status == _lib.KYRO_ENOSPACE and "pool" in str(e.value)
    step = t.extend_async(i32(rows, gpu), i32(new, gpu), total_q=total, max_blocks_per_seq=8 + wide)
    with pytest.raises(kyro_amd.KyroError):
        kyro_amd.sync()
    m.extend(rows, new, 8 + wide, total)
    want = m.extend(rows, new, 8 + wide, total)  # the second call: those served hold theirs
    assert want[1].tolist() == [36, 50, served, 32, 0]
    same_step(step, want)
    same_state(t, m)
    kept = [16, 30, third, 0, 13]
    lens = t.keep(i32(rows, gpu), step.context_lens, step.q_start_loc, i32(kept, gpu))
    assert lens.tolist() == m.keep(rows, want[1], want[2], kept).tolist() == [36, 50, served, 20, 0]
    same_state(t, m)


@pytest.mark.parametrize("wide", [0, 40000])
def test_what_is_refused_on_the_device(gpu, wide):
    """A faulty entry is left out, reported, and changes nothing; the others are served."""
    width = 6
    for rows, new, total in (([0, 9, 2], [1, 1, 1], 3), ([0, 1, 1, 2], [5, 5, 5, 5], 20), ([0, 1, 2], [3, -4, 3], 6),
                             ([0, 1, 2], [3, 97, 3], 200), ([0, 1, 2], [3, 20, 30], 40)):
        t, m = pair(gpu, 16, 4, width, range(20))
        got = t.extend_async(i32(rows, gpu), i32(new, gpu), total_q=total, max_blocks_per_seq=width + wide)
        with pytest.raises(kyro_amd.KyroError) as e:
            kyro_amd.sync()
        assert e.value.status == _lib.KYRO_EINVAL
        same_step(got, m.extend(rows, new, width + wide, total))
        same_state(t, m)
    # records: negative, more shared than held, more held than the state has room for, tokens past the blocks
    for bad in ([-1, 0, 0], [0, -1, 0], [0, 0, -1], [5, 1, 2], [0, 7, 0], [17, 1, 0]):
        t, m = pair(gpu, 16, 3, width, range(20))
        t.requests[1, :3] = i32(bad, gpu)
        m.requests[1, :3] = bad
        got = t.extend_async(i32([0, 1, 2], gpu), i32([20, 1, 20], gpu), total_q=41, max_blocks_per_seq=width + wide)
        with pytest.raises(kyro_amd.KyroError, match="record"):
            kyro_amd.sync()
        assert got.context_lens.tolist() == [20, 0, 20] and got.q_start_loc.tolist() == [0, 20, 21, 41]
        assert got.block_table[:, :3].tolist() == [[19, 18, 0], [0, 0, 0], [17, 16, 0]] and t.pool_count.item() == 16
        assert t.requests[1, :3].tolist() == bad
    # a pool whose count is none, and ids outside the caches
    for count in (-1, 21):
        t, m = pair(gpu, 16, 3, width, range(20))
        t.pool_count.fill_(count)
        got = t.extend_async(i32([0, 1], gpu), i32([1, 0], gpu), total_q=1, max_blocks_per_seq=width + wide)
        with pytest.raises(kyro_amd.KyroError, match="pool"):
            kyro_amd.sync()
        assert got.context_lens.tolist() == [0, 0] and t.pool_count.item() == count
        with pytest.raises(kyro_amd.KyroError, match="pool"):
            t.release(i32([0], gpu))
        assert t.pool_count.item() == count
    t, m = pair(gpu, 16, 3, width, range(20), num_blocks=19)
    with pytest.raises(kyro_amd.KyroError, match="block_table"):
        t.extend(i32([0, 1], gpu), i32([1, 1], gpu), total_q=2, max_blocks_per_seq=width + wide)


def test_keep_refuses_on_the_device(gpu):
    def fresh():
        t, m = pair(gpu, 16, 4, 6, range(12))
        rows, new = [0, 1, 2], [20, 30, 40]
        step = t.extend(i32(rows, gpu), i32(new, gpu), total_q=90)
        return t, m, rows, step, m.extend(rows, new, 6, 90)

    for kept in ([1, 31, 5], [1, -1, 5]):
        t, m, rows, step, want = fresh()
        got = t.keep_async(i32(rows, gpu), step.context_lens, step.q_start_loc, i32(kept, gpu))
        with pytest.raises(kyro_amd.KyroError):
            kyro_amd.sync()
        assert got.tolist() == m.keep(rows, want[1], want[2], kept).tolist() == [1, 0, 5]
        same_state(t, m)
    for name, value in (("context_lens", 29), ("context_lens", 300), ("q_start_loc", 55)):
        t, m, rows, step, want = fresh()
        getattr(step, name)[1] = value
        got = t.keep_async(i32(rows, gpu), step.context_lens, step.q_start_loc, i32([1, 1, 1], gpu))
        with pytest.raises(kyro_amd.KyroError):
            kyro_amd.sync()
        assert got[1].item() == 0 and t.requests[1].tolist() == [0, 2, 0, 0]
    t, m, rows, step, want = fresh()  # a pool that would pass its capacity: nothing moves
    t.pool_count.fill_(12)
    before = [x.clone() for x in (t.requests, t.blocks, t.pool)]
    for f in (lambda: t.keep(i32(rows, gpu), step.context_lens, step.q_start_loc, i32([1, 1, 1], gpu)), lambda: t.release(i32(rows, gpu))):
        with pytest.raises(kyro_amd.KyroError, match="pool"):
            f()
        assert all(torch.equal(x, y) for x, y in zip(before, (t.requests, t.blocks, t.pool))) and t.pool_count.item() == 12
    t, m, rows, step, want = fresh()  # the same request twice: both are left alone
    got = t.keep_async(i32([0, 1, 1], gpu), step.context_lens, step.q_start_loc, i32([1, 1, 1], gpu))
    with pytest.raises(kyro_amd.KyroError, match="state row"):
        kyro_amd.sync()
    assert got.tolist() == [1, 0, 0] and t.requests[:, 0].tolist() == [1, 0, 0, 0]


def test_rows_by_default_and_outputs_that_are_given(gpu):
    t, m = pair(gpu, 16, 5, 6, range(30))
    new = [3, 0, 40]
    out = StepTables(torch.full((3, 6), -7, device=gpu), torch.full((3,), -7, device=gpu), torch.full((4,), -7, dtype=torch.int32, device=gpu),
                     torch.full((50,), -7, device=gpu), torch.full((50,), -7, device=gpu))
    got = t.extend(None, i32(new, gpu), total_q=50, max_blocks_per_seq=6, out=out)
    want = m.extend([0, 1, 2], new, 6, 50)
    same_step(got, want)
    assert all(x is y for x, y in zip(got, out))
    lens = t.keep(None, got.context_lens, got.q_start_loc, i32([1, 5, 17], gpu), out=got.context_lens)
    assert lens.tolist() == m.keep([0, 1, 2], want[1], want[2], [1, 5, 17]).tolist() == [1, 0, 17]
    same_state(t, m)


def test_without_positions_or_slots(gpu):
    """The C entry point takes NULL for either."""
    for positions, slots in ((True, False), (False, True), (False, False)):
        t, m = pair(gpu, 16, 3, 6, range(30))
        rows, new = i32([1, 2], gpu), i32([30, 5], gpu)
        table, ctx = torch.zeros((2, 6), dtype=torch.int64, device=gpu), torch.zeros(2, dtype=torch.int64, device=gpu)
        start, at = torch.zeros(3, dtype=torch.int32, device=gpu), torch.full((35,), -7, device=gpu)
        c = t._context()
        _lib.check(_lib.lib().kyro_tables_extend(
            c.handle, t._params(2, 6, 35), rows.data_ptr(), new.data_ptr(), t.requests.data_ptr(), t.blocks.data_ptr(), t.pool.data_ptr(),
            t.pool_count.data_ptr(), table.data_ptr(), ctx.data_ptr(), start.data_ptr(), at.data_ptr() if positions else None,
            at.data_ptr() if slots else None))
        kyro_amd.sync()
        want = m.extend([1, 2], [30, 5], 6, 35)
        assert np.array_equal(table.cpu(), want[0]) and ctx.tolist() == [30, 5] and start.tolist() == [0, 30, 35]
        assert np.array_equal(at.cpu(), want[3] if positions else want[4] if slots else np.full(35, -7))


@pytest.mark.parametrize("width", [40, 20000])
def test_a_captured_step_replays(gpu, width):
    """extend, then keep of what `kept` holds at the time: every replay goes on from the last one's lengths. Eager
    work runs between the replays."""
    t, m = pair(gpu, 16, 8, 40, range(300))
    rows, new, kept = [5, 1, -1, 3], i32([8, 8, 0, 8], gpu), i32([0, 0, 0, 0], gpu)
    srows = i32(rows, gpu)
    kyro_amd.context(0).reserve(4 * 32)
    torch.cuda.synchronize()
    out = StepTables(torch.zeros((4, width), dtype=torch.int64, device=gpu), torch.zeros(4, dtype=torch.int64, device=gpu),
                     torch.zeros(5, dtype=torch.int32, device=gpu), torch.zeros(24, dtype=torch.int64, device=gpu),
                     torch.zeros(24, dtype=torch.int64, device=gpu))
    lens = torch.zeros(4, dtype=torch.int64, device=gpu)
    s = torch.cuda.Stream(gpu)
    s.wait_stream(torch.cuda.current_stream(gpu))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        t.extend_async(srows, new, total_q=24, max_blocks_per_seq=width, out=out)
        t.keep_async(srows, out.context_lens, out.q_start_loc, kept, plus=1, out=lens)
    for i in range(6):
        k = [i % 8, 7, 0, (5 * i) % 8]
        kept.copy_(i32(k, gpu))
        g.replay()
        torch.cuda.synchronize()
        want = m.extend(rows, [8, 8, 0, 8], width, 24)
        same_step(out, want)
        assert lens.tolist() == m.keep(rows, want[1], want[2], k, 1).tolist()
        same_state(t, m)
        if i == 3:  # an eager call between two replays
            t.release(i32([1], gpu))
            m.release([1])
            same_state(t, m)


def test_on_another_stream(gpu):
    t, m = pair(gpu, 16, 4, 6, range(20))
    s = torch.cuda.Stream(gpu)
    rows, new = i32([3, 0], gpu), i32([33, 7], gpu)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        step = t.extend_async(rows, new, total_q=40)
        lens = t.keep_async(rows, step.context_lens, step.q_start_loc, new)
    s.synchronize()
    same_step(step, m.extend([3, 0], [33, 7], 6, 40))
    assert lens.tolist() == [33, 7]
