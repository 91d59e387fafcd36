"""A step whose pool runs out, with one sync behind all of it: the status is that of space, the requests that were served
are computed, and the others are as before."""
import pytest
import torch

import kyro_amd
from kyro_amd import PagedAttention, PagedKVCache, RequestTables, _lib
from tests import helpers as h

pytestmark = pytest.mark.gpu

BS, H, HKV, D = 16, 4, 2, 64


def i32(x, gpu):
    return torch.tensor(list(x), dtype=torch.int32, device=gpu)


def rows_of(gen, n, heads, gpu):
    return torch.randn((n, heads, D), generator=gen).to(gpu)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("append", ["kv", "qkv"])
def test_a_step_whose_pool_runs_out(gpu, append, shared):
    gen = torch.Generator().manual_seed(4)
    kv, attn = PagedKVCache(BS, HKV, D), PagedAttention(BS, H, D, HKV)
    kc, vc = (torch.zeros((8, HKV, BS, D), device=gpu) for _ in range(2))
    t = RequestTables.new(BS, rows=4, max_blocks=4, pool=range(4), num_blocks=8, device=gpu)
    srows, groups = i32([0, 1, 2, -1], gpu), (i32([0, 3], gpu), i32([0], gpu))
    keys, values = {}, {}

    def step(new, kept):
        total = sum(new)
        q, k, v = rows_of(gen, total, H, gpu), rows_of(gen, total, HKV, gpu), rows_of(gen, total, HKV, gpu)
        s = t.extend_async(srows, i32(new, gpu), total_q=total)
        if append == "kv":
            kv.append_kv_async(k, v, kc, vc, s.block_table, s.context_lens, q_start_loc=s.q_start_loc)
        else:
            q = kv.append_qkv_async(q, k, v, kc, vc, s.block_table, s.context_lens, q_start_loc=s.q_start_loc)
        args = q, kc, vc, s.block_table, s.context_lens
        kw = dict(q_start_loc=s.q_start_loc, max_q_len=max(new))
        out = attn.forward_shared_async(*args, *groups, **kw) if shared else attn.forward_async(*args, **kw)
        lens = t.keep_async(srows, s.context_lens, s.q_start_loc, i32(kept, gpu))
        return s, q, k, v, out, lens

    def check(served, new, got):
        s, q, k, v, out, lens = got
        at = 0
        for b, n in enumerate(new):
            rows = slice(at, at + n)
            at += n
            if b not in served:
                assert not out[rows].any()
                continue
            keys[b] = torch.cat([keys.get(b, k[:0]), k[rows]])
            values[b] = torch.cat([values.get(b, v[:0]), v[rows]])
            for j in range(n):
                seen = len(keys[b]) - n + j + 1
                qj = q[at - n + j].double().view(HKV, H // HKV, D)
                p = torch.softmax(qj @ keys[b][:seen].double().permute(1, 2, 0) / D ** 0.5, -1)
                exact = (p @ values[b][:seen].double().transpose(0, 1).contiguous()).view(H, D)
                # f32, as the other attention tests.
                assert (out[at - n + j].double() - exact).abs().max() <= h.ATOL_F32_SUMS

    new = [16, 20, 9, 0]
    got = step(new, new)
    kyro_amd.sync()
    check({0, 1, 2}, new, got)
    assert t.pool_count.item() == 0 and got[5].tolist() == new
    # One more row of request 0 needs a block that is not there; 1 and 2 have room.
    before = [x.clone() for x in (t.requests, t.blocks, t.pool, t.pool_count)]
    new = [1, 12, 7, 0]
    got = step(new, new)
    with pytest.raises(kyro_amd.KyroError) as e:
        kyro_amd.sync()
    assert e.value.status == _lib.KYRO_ENOSPACE and "not enough free blocks" in str(e.value)
    check({1, 2}, new, got)
    assert got[5].tolist() == [0, 32, 16, 0]
    before[0][1, 0], before[0][2, 0] = 32, 16
    assert all(torch.equal(x, y) for x, y in zip((t.requests, t.blocks, t.pool, t.pool_count), before))
    # With request 2 gone the same step is served.
    t.release(i32([2], gpu))
    del keys[2], values[2]
    srows[2] = -1
    new = [1, 0, 0, 0]
    got = step(new, new)
    kyro_amd.sync()
    check({0}, new, got)
    assert got[5].tolist() == [17, 32, 0, 0]


@pytest.mark.parametrize("append", ["kv", "qkv"])
def test_other_faults_beside_a_pool_that_runs_out(gpu, append):
    """A context that is wrong by itself stays an error of the caller, whatever the pool says; so does a length of 0 with
    rows where no pool ran out."""
    kv = PagedKVCache(BS, HKV, D)
    kc, vc = (torch.zeros((8, HKV, BS, D), device=gpu) for _ in range(2))
    gen = torch.Generator().manual_seed(5)

    def call(ctx, extend):
        if extend:
            t = RequestTables.new(BS, rows=1, max_blocks=4, pool=[], num_blocks=8, device=gpu)
            t.extend_async(None, i32([1], gpu), total_q=1)
        q, k, v = rows_of(gen, 3, H, gpu), rows_of(gen, 3, HKV, gpu), rows_of(gen, 3, HKV, gpu)
        args = kc, vc, torch.zeros((1, 4), dtype=torch.int64, device=gpu), torch.tensor([ctx], device=gpu)
        start = i32([0, 3], gpu)
        if append == "kv":
            kv.append_kv_async(k, v, *args, q_start_loc=start)
        else:
            kv.append_qkv_async(q, k, v, *args, q_start_loc=start)
        with pytest.raises(kyro_amd.KyroError) as e:
            kyro_amd.sync()
        assert not kc.any() and not vc.any()
        return e.value.status

    for ctx in (2, 65, -1):
        assert call(ctx, True) == call(ctx, False) == _lib.KYRO_EINVAL
    assert call(0, False) == _lib.KYRO_EINVAL
    assert call(0, True) == _lib.KYRO_ENOSPACE
