"""Accumulated weights and eviction without a GPU: what the entry points refuse, their scratch, and the block
manager's part."""
import ctypes
import math

import numpy as np
import pytest

from kyro_amd import BlockManager, KyroError, _lib
from tests.test_abi import struct_fields

W_GOOD = dict(block_size=16, num_heads=8, head_dim=64, num_kv_heads=2, batch_size=2, total_q=2, max_blocks_per_seq=4,
              num_blocks=9, dtype=_lib.KYRO_BF16, causal=1, scale=0.0, max_q_len=1, num_state_rows=2, max_tokens=64)
W_PTRS = dict(query=1 << 20, q_start_loc=None, row_positions=None, key_cache=2 << 20, block_table=3 << 20,
              context_lens=4 << 20, state_rows=None, weights=5 << 20, out_weights=5 << 20, positions=6 << 20)
E_GOOD = dict(block_size=16, num_kv_heads=2, head_dim=64, batch_size=2, max_blocks_per_seq=4, num_blocks=9,
              dtype=_lib.KYRO_BF16, budget=32, sink=4, recent=8, num_state_rows=2, max_tokens=64)
E_PTRS = dict(key_cache=1 << 20, value_cache=2 << 20, block_table=3 << 20, context_lens=4 << 20, state_rows=None,
              weights=5 << 20, positions=6 << 20, out_weights=5 << 20, out_positions=6 << 20, out_context_lens=7 << 20)


def weigh(**change):
    """No address is dereferenced: every check here is the host's, and a good call ends at its null context."""
    p = _lib.AttnWeightsParams(**{k: change.get(k, v) for k, v in W_GOOD.items()})
    rc = _lib.lib().kyro_attn_weights(None, ctypes.byref(p), *[change.get(k, v) for k, v in W_PTRS.items()])
    return rc, _lib.last_error()


def evict(**change):
    p = _lib.KvEvictParams(**{k: change.get(k, v) for k, v in E_GOOD.items()})
    rc = _lib.lib().kyro_kv_evict(None, ctypes.byref(p), *[change.get(k, v) for k, v in E_PTRS.items()])
    return rc, _lib.last_error()


def test_good_calls_only_lack_their_context():
    for f, changes in ((weigh, ({}, dict(out_weights=15 << 20), dict(total_q=9, q_start_loc=8 << 20, max_q_len=0),
                                dict(batch_size=0, total_q=0), dict(state_rows=9 << 20, num_state_rows=1))),
                       (evict, ({}, dict(out_weights=15 << 20, out_positions=16 << 20), dict(batch_size=0),
                                dict(budget=10 ** 9), dict(sink=0, recent=32)))):
        for change in changes:
            rc, msg = f(**change)
            assert rc == _lib.KYRO_EINVAL and "null kyro_ctx" in msg, (change, msg)


@pytest.mark.parametrize("change, status, text", [
    (dict(block_size=0), "EINVAL", "sizes"), (dict(max_tokens=0), "EINVAL", "sizes"), (dict(max_q_len=-1), "EINVAL", "sizes"),
    (dict(num_heads=7), "EINVAL", "num_kv_heads"), (dict(head_dim=68), "EUNSUPPORTED", "head_dim 68"),
    (dict(head_dim=264), "EUNSUPPORTED", "head_dim 264"), (dict(dtype=3), "EINVAL", "dtype"),
    (dict(scale=math.nan), "EINVAL", "scale"), (dict(scale=-0.5), "EINVAL", "scale"),
    (dict(scale=1e-44), "EINVAL", "scale"), (dict(scale=3e38), "EINVAL", "scale"), (dict(total_q=5), "EINVAL", "batch_size"),
    (dict(query=None), "EINVAL", "null device pointer"), (dict(positions=None), "EINVAL", "null device pointer"),
    (dict(key_cache=(2 << 20) + 8), "EINVAL", "16-byte"), (dict(num_state_rows=1), "EINVAL", "state row"),
    (dict(out_weights=(5 << 20) + 4), "EINVAL", "overlaps"),
    (dict(max_blocks_per_seq=2 ** 30, max_tokens=2 ** 31 - 1), "EUNSUPPORTED", "one launch")])
def test_weights_refusals(change, status, text):
    rc, msg = weigh(**change)
    assert rc == getattr(_lib, "KYRO_" + status) and text in msg, msg


@pytest.mark.parametrize("change, status, text", [
    (dict(num_kv_heads=0), "EINVAL", "sizes"), (dict(head_dim=12), "EUNSUPPORTED", "head_dim 12"), (dict(dtype=-1), "EINVAL", "dtype"),
    (dict(budget=0), "EINVAL", "budget"), (dict(sink=-1), "EINVAL", "sink"), (dict(recent=29), "EINVAL", "sink + recent"),
    (dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1), "EINVAL", "sink + recent"),
    (dict(value_cache=None), "EINVAL", "null device pointer"), (dict(out_context_lens=None), "EINVAL", "null device pointer"),
    (dict(value_cache=(2 << 20) + 2), "EINVAL", "16-byte"), (dict(num_state_rows=1), "EINVAL", "state row"),
    (dict(out_weights=(5 << 20) + 512), "EINVAL", "overlap"), (dict(out_positions=5 << 20), "EINVAL", "overlap"),
    (dict(out_weights=9 << 20, out_positions=9 << 20), "EINVAL", "overlap"),
    (dict(out_context_lens=4 << 20), "EINVAL", "out_context_lens"), (dict(out_context_lens=(4 << 20) + 8), "EINVAL", "out_context_lens"),
    (dict(max_blocks_per_seq=2 ** 30, max_tokens=2 ** 31 - 1), "EUNSUPPORTED", "one launch"),
    (dict(batch_size=2 ** 24, num_state_rows=2 ** 24), "EUNSUPPORTED", "one launch")])
def test_evict_refusals(change, status, text):
    rc, msg = evict(**change)
    assert rc == getattr(_lib, "KYRO_" + status) and text in msg, msg


def test_null_params_and_structs():
    lib = _lib.lib()
    assert lib.kyro_attn_weights(None, None, *([None] * 10)) == _lib.KYRO_EINVAL
    assert lib.kyro_kv_evict(None, None, *([None] * 10)) == _lib.KYRO_EINVAL
    n = ctypes.c_size_t()
    assert lib.kyro_kv_evict_workspace(None, ctypes.byref(n)) == _lib.KYRO_EINVAL
    assert lib.kyro_kv_evict_workspace(ctypes.byref(_lib.KvEvictParams(**E_GOOD)), None) == _lib.KYRO_EINVAL
    assert [f[0] for f in _lib.AttnWeightsParams._fields_] == struct_fields("kyro_attn_weights_params")
    assert [f[0] for f in _lib.KvEvictParams._fields_] == struct_fields("kyro_kv_evict_params")


def test_workspace():
    """Scratch is whole, and bounded where tables are far wider than the contexts in use."""
    lib, n = _lib.lib(), ctypes.c_size_t()
    for width in (4, 64, 8192, 2 ** 20):
        p = _lib.AttnWeightsParams(**dict(W_GOOD, batch_size=64, total_q=64 * 9, max_q_len=9, num_state_rows=64,
                                          max_blocks_per_seq=width, max_tokens=16 * width))
        assert lib.kyro_attn_weights_workspace(None, ctypes.byref(p), 1, ctypes.byref(n)) == _lib.KYRO_OK
        assert 0 < n.value <= 64 << 20
    p = _lib.KvEvictParams(**dict(E_GOOD, batch_size=64, budget=2048, max_blocks_per_seq=8192, max_tokens=131072))
    assert lib.kyro_kv_evict_workspace(ctypes.byref(p), ctypes.byref(n)) == _lib.KYRO_OK
    assert 64 * 2 * 2 * 2048 * 4 <= n.value <= 64 * 2 * 2 * 2048 * 4 + 4096


# ------------------------------------------------------------------------------------ block manager

def test_make_private_replaces_shared_blocks():
    bm = BlockManager(4, 24)
    prompt = list(range(10))
    bm.allocate_with_prefix(1, prompt)
    bm.free(1)  # three blocks go to the prefix cache
    blocks, cached = bm.allocate_with_prefix(2, prompt + [50, 51, 52])
    assert cached == 10
    old_copies = bm.take_copies()  # the partially matched third block
    assert len(old_copies) == 1
    bm.allocate_with_prefix(3, prompt[:8] + [99])
    assert bm.make_private(2)
    bm.check()
    copies = bm.take_copies()
    now = bm.block_table[2]
    assert [s for s, _ in copies] == blocks[:2] and [d for _, d in copies] == now[:2] and now[2:] == blocks[2:]
    assert not set(now) & set(bm.block_table[3])
    bm.check()
    assert bm.make_private(2) and bm.take_copies() == []  # nothing is shared any more


def test_make_private_forgets_the_prompt():
    bm = BlockManager(4, 24)
    bm.allocate_with_prefix(7, list(range(20)))
    bm.append_slots(7, 3)
    with pytest.raises(KyroError):
        bm.truncate(7, 8)  # the prompt's blocks may be shared
    assert bm.make_private(7)
    bm.truncate(7, 8)
    assert bm.request(7)[1] == 8 and len(bm.block_table[7]) == 2
    assert bm.append_slots(7, 5) and len(bm.block_table[7]) == 4
    bm.free(7)
    assert bm.num_cached_blocks == 0 and bm.num_free_blocks == 24
    bm.check()


def test_make_private_without_room():
    bm = BlockManager(4, 9)
    bm.allocate_with_prefix(1, list(range(12)))
    bm.free(1)
    bm.allocate_with_prefix(2, list(range(12)))
    bm.allocate_with_prefix(3, list(range(12)))  # both hold the three cached blocks
    assert bm.allocate(4, 16) is not None  # two of the nine are left
    before = bm.block_table[2]
    assert not bm.make_private(2)
    assert bm.block_table[2] == before and bm.take_copies() == []
    bm.check()
    bm.free(4, cache_prompt=False)
    assert bm.make_private(2) and len(bm.take_copies()) == 3
    bm.check()
    with pytest.raises(KyroError):
        bm.make_private(77)


def test_make_private_random_streams():
    """References stay whole through requests that share, part, shrink and end in any order."""
    rng = np.random.default_rng(5)
    bm, live = BlockManager(4, 60), {}
    for step in range(400):
        what = rng.integers(0, 5)
        if what <= 1 and len(live) < 8:
            got = bm.allocate_with_prefix(step, [int(x) for x in rng.integers(0, 2, rng.integers(1, 24))])
            if got:
                live[step] = True
        elif live:
            rid = int(rng.choice(list(live)))
            if what == 2:
                if bm.make_private(rid):
                    bm.truncate(rid, int(rng.integers(0, bm.request(rid)[1] + 1)))
            elif what == 3:
                bm.append_slots(rid, int(rng.integers(0, 6)))
            else:
                bm.free(rid, cache_prompt=bool(rng.integers(0, 2)))
                del live[rid]
        if rng.integers(0, 2):
            bm.take_copies()
        bm.check()


def test_no_rows_at_all_still_take_weights_elsewhere():
    """A call without rows is one to make where the weights go elsewhere, and needs its pointers then."""
    none = dict(total_q=0, q_start_loc=8 << 20, query=None)
    for change in (none, dict(none, out_weights=15 << 20), dict(none, weights=None, out_weights=None)):
        rc, msg = weigh(**change)
        assert rc == _lib.KYRO_EINVAL and "null kyro_ctx" in msg, (change, msg)
    rc, msg = weigh(**dict(none, out_weights=15 << 20, block_table=None))
    assert rc == _lib.KYRO_EINVAL and "null device pointer" in msg


# ------------------------------------------------------------------------------------ the front blocks alone

def shared_prompt(bm, tokens):
    """A request whose whole prompt is shared with the prefix cache."""
    bm.allocate_with_prefix(1, list(range(tokens)))
    bm.free(1)
    assert bm.allocate_with_prefix(2, list(range(tokens)))[1] == tokens


def test_make_private_of_the_front_fits_where_the_whole_does_not():
    """24 shared tokens cut to 6: two blocks are rewritten, and two are free. The four behind are only read, and
    their references go with the cut."""
    for front in (False, True):
        bm = BlockManager(4, 18)
        shared_prompt(bm, 24)
        assert bm.allocate(3, 40) is not None and bm.num_free_blocks == 2
        bm.allocate_with_prefix(4, list(range(24)))
        before = bm.block_table[2]
        if not front:
            assert not bm.make_private(2) and bm.block_table[2] == before
            continue
        assert bm.make_private(2, 6)
        copies, now = bm.take_copies(), bm.block_table[2]
        assert [s for s, _ in copies] == before[:2] and [d for _, d in copies] == now[:2] and now[2:] == before[2:]
        bm.check()
        bm.truncate(2, 6)
        assert bm.request(2)[1] == 6 and bm.block_table[2] == now[:2] and bm.block_table[4] == before
        bm.free(2)
        bm.check()
        assert bm.num_free_blocks == 2 and bm.num_cached_blocks == 6


def test_a_cut_inside_a_shared_block_is_refused():
    """Rows appended behind such a cut would be written into a block that others read."""
    bm = BlockManager(4, 30)
    shared_prompt(bm, 24)
    assert bm.make_private(2, 6)
    bm.take_copies()
    for bad in (9, 10, 23):
        with pytest.raises(KyroError):
            bm.truncate(2, bad)
    bm.truncate(2, 20)  # at a block's end: what follows goes to blocks of its own
    assert bm.append_slots(2, 3)
    assert bm.block_table[2][5] not in bm.request(2)[0][:5]
    bm.check()
    with pytest.raises(KyroError):
        bm.truncate(2, 11)
    bm.truncate(2, 8)
    bm.truncate(2, 7)
    bm.check()


@pytest.mark.parametrize("tokens", [0, 1, 4, 5, 24, 1000])
def test_make_private_of_so_many_tokens(tokens):
    bm = BlockManager(4, 30)
    shared_prompt(bm, 24)
    before = bm.block_table[2]
    n = min(6, -(-tokens // 4))
    assert bm.make_private(2, tokens)
    assert [s for s, _ in bm.take_copies()] == before[:n] and bm.block_table[2][n:] == before[n:]
    assert not set(bm.block_table[2][:n]) & set(before)
    bm.check()
    with pytest.raises(KyroError):
        bm.make_private(2, -1)
    with pytest.raises(KyroError):
        bm.make_private(77, 4)


def test_make_private_front_random_streams():
    """No block that a request may write, the front ones and the one its next row goes to, has another holder."""
    rng = np.random.default_rng(6)
    bm, live, front = BlockManager(4, 60), {}, {}
    for step in range(600):
        what = rng.integers(0, 6)
        if what <= 1 and len(live) < 8:
            if bm.allocate_with_prefix(step, [int(x) for x in rng.integers(0, 2, rng.integers(1, 24))]):
                live[step], front[step] = True, 0
        elif live:
            rid = int(rng.choice(list(live)))
            tokens = bm.request(rid)[1]
            if what == 2:
                n = int(rng.integers(0, tokens + 2))
                if bm.make_private(rid, n):
                    front[rid] = max(front[rid], n)
            elif what == 3:
                bm.append_slots(rid, int(rng.integers(0, 6)))
            elif what == 4:
                to = int(rng.integers(0, tokens + 1))
                try:
                    bm.truncate(rid, to)
                    front[rid] = min(front[rid], to)
                except KyroError:
                    pass
            else:
                bm.free(rid, cache_prompt=bool(rng.integers(0, 2)))
                del live[rid]
        if rng.integers(0, 2):
            bm.take_copies()
        bm.check()
        for rid in live:
            blocks, tokens = bm.request(rid)[:2]
            written = set(blocks[: -(-front[rid] // 4)]) | (set(blocks[tokens // 4:]) if tokens % 4 else set())
            others = [b for o in live if o != rid for b in bm.block_table[o]]
            assert not written & set(others)


@pytest.mark.parametrize("batch, heads, fits", [(2**22 - 1, 1, True), (2**22, 1, False), (2**20, 3, True), (2**20, 4, False),
                                                (3, 2**30, False)])
def test_sequences_and_heads_that_one_launch_carries(batch, heads, fits):
    """A grid has fewer than 2^32 threads: at most 2^22 - 1 workgroups of 1024."""
    rc, msg = evict(batch_size=batch, num_state_rows=batch, num_kv_heads=heads, weights=1 << 40, positions=1 << 50,
                    out_weights=1 << 40, out_positions=1 << 50, context_lens=1 << 30, out_context_lens=2 << 30)
    if fits:
        assert rc == _lib.KYRO_EINVAL and "null kyro_ctx" in msg, msg
    else:
        assert rc == _lib.KYRO_EUNSUPPORTED and "one launch" in msg, msg
