"""Block tables on the GPU, without a GPU: what the entry points refuse, their scratch, and the handle's checks."""
import ctypes

import numpy as np
import pytest
import torch

from kyro_amd import RequestTables, _lib
from tests.test_abi import struct_fields

GOOD = dict(block_size=16, batch_size=3, max_blocks_per_seq=8, num_state_rows=4, max_state_blocks=10, num_blocks=64,
            pool_capacity=20, max_rows=24, kept_plus=0)
EXTEND = dict(state_rows=1 << 20, new_rows=2 << 20, requests=3 << 20, blocks=4 << 20, pool=5 << 20, pool_count=6 << 20,
              block_table=7 << 20, context_lens=8 << 20, q_start_loc=9 << 20, positions=10 << 20, slots=11 << 20)
KEEP = dict(state_rows=1 << 20, context_lens=8 << 20, q_start_loc=9 << 20, kept=2 << 20, requests=3 << 20, blocks=4 << 20,
            pool=5 << 20, pool_count=6 << 20, out_context_lens=12 << 20)
RELEASE = dict(state_rows=1 << 20, requests=3 << 20, blocks=4 << 20, pool=5 << 20, pool_count=6 << 20)
CALLS = {"extend": EXTEND, "keep": KEEP, "release": RELEASE}


def call(name, **change):
    """No address is dereferenced: every check here is the host's, and a good call ends at its null context."""
    p = _lib.TablesParams(**{k: change.get(k, v) for k, v in GOOD.items()})
    rc = getattr(_lib.lib(), "kyro_tables_" + name)(None, ctypes.byref(p), *[change.get(k, v) for k, v in CALLS[name].items()])
    return rc, _lib.last_error()


@pytest.mark.parametrize("name, change", [
    ("extend", {}), ("extend", dict(state_rows=None)), ("extend", dict(positions=None, slots=None)),
    ("extend", dict(max_rows=0)), ("extend", dict(batch_size=0, state_rows=None)), ("extend", dict(pool=None, pool_capacity=0)),
    ("extend", dict(batch_size=9)), ("keep", {}), ("keep", dict(out_context_lens=8 << 20)), ("keep", dict(kept_plus=-1)),
    ("keep", dict(max_blocks_per_seq=0, max_rows=-5)), ("release", {}), ("release", dict(batch_size=0))])
def test_good_calls_only_lack_their_context(name, change):
    rc, msg = call(name, **change)
    assert rc == _lib.KYRO_EINVAL and "null kyro_ctx" in msg, msg


@pytest.mark.parametrize("name", sorted(CALLS))
@pytest.mark.parametrize("change, status, text", [
    (dict(block_size=0), "EINVAL", "sizes"), (dict(batch_size=-1), "EINVAL", "sizes"), (dict(num_state_rows=0), "EINVAL", "sizes"),
    (dict(max_state_blocks=0), "EINVAL", "sizes"), (dict(num_blocks=0), "EINVAL", "sizes"), (dict(pool_capacity=-1), "EINVAL", "sizes"),
    (dict(num_state_rows=131073), "EUNSUPPORTED", "num_state_rows"), (dict(max_state_blocks=2 ** 27), "EUNSUPPORTED", "2^31 tokens"),
    (dict(batch_size=5, state_rows=None), "EINVAL", "without state_rows"), (dict(requests=None), "EINVAL", "null device pointer"),
    (dict(pool=None), "EINVAL", "null device pointer"), (dict(requests=(3 << 20) + 8), "EINVAL", "16-byte"),
    (dict(pool=(4 << 20) + 312, num_blocks=65), "EINVAL", "overlaps"), (dict(pool_count=(3 << 20) + 60), "EINVAL", "overlaps"),
    (dict(state_rows=(3 << 20) + 4), "EINVAL", "overlaps")])
def test_refusals_of_every_call(name, change, status, text):
    rc, msg = call(name, **change)
    assert rc == getattr(_lib, "KYRO_" + status) and text in msg and "tables_" + name in msg, msg


@pytest.mark.parametrize("name, change, status, text", [
    ("extend", dict(max_blocks_per_seq=0), "EINVAL", "sizes"), ("extend", dict(max_rows=-1), "EINVAL", "sizes"),
    ("extend", dict(new_rows=None), "EINVAL", "null device pointer"), ("extend", dict(q_start_loc=None), "EINVAL", "null device pointer"),
    ("extend", dict(block_table=4 << 20), "EINVAL", "overlaps"), ("extend", dict(slots=(10 << 20) + 184), "EINVAL", "overlaps"),
    ("extend", dict(q_start_loc=(2 << 20) - 12), "EINVAL", "overlaps"),
    ("extend", dict(batch_size=2 ** 24, max_blocks_per_seq=2 ** 22), "EUNSUPPORTED", "one launch"),
    ("keep", dict(kept=None), "EINVAL", "null device pointer"), ("keep", dict(out_context_lens=(8 << 20) + 8), "EINVAL", "overlaps"),
    ("keep", dict(out_context_lens=2 << 20), "EINVAL", "overlaps"),
    ("release", dict(batch_size=2 ** 24, max_state_blocks=2 ** 26), "EUNSUPPORTED", "one launch")])
def test_refusals(name, change, status, text):
    if change.get("batch_size", 0) > 1000:  # arrays of so many entries, apart from each other
        change = dict({k: i << 50 for i, k in enumerate(CALLS[name], 1)}, **change)
    rc, msg = call(name, **change)
    assert rc == getattr(_lib, "KYRO_" + status) and text in msg, msg


def test_null_params_and_structs():
    lib = _lib.lib()
    for name, ptrs in CALLS.items():
        assert getattr(lib, "kyro_tables_" + name)(None, None, *([None] * len(ptrs))) == _lib.KYRO_EINVAL
    assert [f[0] for f in _lib.TablesParams._fields_] == struct_fields("kyro_tables_params")


def test_workspace():
    n = ctypes.c_size_t()
    p = _lib.TablesParams(**dict(GOOD, batch_size=1000))
    assert _lib.lib().kyro_tables_workspace(ctypes.byref(p), ctypes.byref(n)) == _lib.KYRO_OK and n.value == 32000
    assert _lib.lib().kyro_tables_workspace(None, ctypes.byref(n)) == _lib.KYRO_EINVAL
    assert _lib.lib().kyro_tables_workspace(ctypes.byref(p), None) == _lib.KYRO_EINVAL


def handle(rows=4, max_blocks=6, pool=range(10)):
    return RequestTables.new(16, rows=rows, max_blocks=max_blocks, pool=list(pool), num_blocks=64, device="cpu")


def test_handle_and_admission():
    t = handle()
    assert t.requests.shape == (4, 4) and t.pool.tolist() == list(range(10)) and t.pool_count.tolist() == [10]
    t.admit(2, [40, 41, 42], 33)
    assert t.requests[2].tolist() == [33, 3, 3, 0] and t.blocks[2].tolist() == [40, 41, 42, 0, 0, 0]
    t.admit(2)
    assert t.requests[2].tolist() == [0, 0, 0, 0]
    for bad in (dict(row=4), dict(row=-1), dict(row=0, blocks=[1] * 7), dict(row=0, blocks=[1], tokens=17), dict(row=0, tokens=1),
                dict(row=0, blocks=[1], tokens=-1)):
        with pytest.raises(ValueError):
            t.admit(**bad)
    assert RequestTables.new(16, rows=1, max_blocks=1, pool=[], num_blocks=1, device="cpu").pool_count.tolist() == [0]


@pytest.mark.parametrize("change, error", [
    (dict(requests=torch.zeros(4, 3, dtype=torch.int32)), ValueError), (dict(requests=torch.zeros(4, 4)), TypeError),
    (dict(requests=np.zeros((4, 4))), TypeError), (dict(blocks=torch.zeros(3, 6, dtype=torch.int64)), ValueError),
    (dict(blocks=torch.zeros(6, 4, dtype=torch.int64).t()), ValueError), (dict(pool=torch.zeros(5, dtype=torch.int32)), TypeError),
    (dict(pool_count=torch.zeros(2, dtype=torch.int32)), ValueError), (dict(pool_count=torch.zeros((), dtype=torch.int32)), ValueError)])
def test_handle_refuses(change, error):
    good = dict(requests=torch.zeros(4, 4, dtype=torch.int32), blocks=torch.zeros(4, 6, dtype=torch.int64),
                pool=torch.zeros(5, dtype=torch.int64), pool_count=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(error):
        RequestTables(16, **dict(good, **change), num_blocks=9)


def test_call_arguments():
    t, i32, i64 = handle(), torch.int32, torch.int64
    rows, new = torch.zeros(2, dtype=i32), torch.ones(2, dtype=i32)
    ctx, start = torch.zeros(2, dtype=i64), torch.zeros(3, dtype=i32)
    with pytest.raises(ValueError, match="GPU"):
        t.extend(rows, new, total_q=2)
    with pytest.raises(ValueError, match="GPU"):
        t.keep(rows, ctx, start, new)
    with pytest.raises(ValueError, match="GPU"):
        t.release(rows)
    for f in (lambda: t.extend(rows.long(), new, total_q=2), lambda: t.extend(rows, new.float(), total_q=2),
              lambda: t.extend(rows, [1, 1], total_q=2), lambda: t.keep(rows, ctx.int(), start, new),
              lambda: t.keep(rows, ctx, start.long(), new), lambda: t.release([0])):
        with pytest.raises(TypeError):
            f()
    out = (torch.zeros(2, 6, dtype=i64), ctx, start, torch.zeros(2, dtype=i64), torch.zeros(3, dtype=i64))
    for f in (lambda: t.extend(rows[:1], new, total_q=2), lambda: t.extend(None, torch.ones(5, dtype=i32), total_q=5),
              lambda: t.extend(rows, new, total_q=2, out=out), lambda: t.extend(rows, new[None], total_q=2),
              lambda: t.extend(rows, torch.ones(4, dtype=i32)[::2], total_q=2), lambda: t.keep(rows, ctx, start[:2], new),
              lambda: t.keep(rows, ctx, start, new[:1]), lambda: t.keep(rows, ctx, start, new, out=ctx[:1])):
        with pytest.raises(ValueError):
            f()


def test_an_empty_batch_needs_no_device():
    t, empty = handle(), torch.zeros(0, dtype=torch.int32)
    step = t.extend_async(empty, empty, total_q=3)
    assert step.q_start_loc.tolist() == [0] and step.slots.tolist() == [-1] * 3 and step.positions.tolist() == [-1] * 3
    assert t.keep_async(empty, step.context_lens, step.q_start_loc, empty).shape == (0,)
    t.release_async(empty)
