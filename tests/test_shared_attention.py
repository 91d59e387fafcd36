"""Attention over shared prefixes without a GPU: what the entry point refuses, and its scratch."""
import ctypes

import pytest

from kyro_amd import _lib

GOOD = dict(block_size=16, num_heads=8, head_dim=128, num_kv_heads=2, batch_size=4, total_q=4, max_blocks_per_seq=40, num_blocks=99,
            dtype=_lib.KYRO_BF16, out_dtype=_lib.KYRO_F32, causal=1, scale=0.0, path=0, num_splits=0, max_q_len=1, kv_reuse=0, schedule=0)
PTRS = dict(query=1 << 20, q_start_loc=None, key_cache=2 << 20, value_cache=3 << 20, block_table=4 << 20, context_lens=5 << 20,
            group_starts=6 << 20, group_blocks=7 << 20, out=8 << 20)


def call(groups=1, **change):
    """No address is dereferenced: every check here is the host's, and a good call ends at its null context."""
    p = _lib.PagedAttentionParams(**{k: change.get(k, v) for k, v in GOOD.items()})
    rc = _lib.lib().kyro_paged_attention_shared(None, ctypes.byref(p), groups, *[change.get(k, v) for k, v in PTRS.items()])
    return rc, _lib.last_error()


@pytest.mark.parametrize("change", [{}, dict(groups=0, group_starts=None, group_blocks=None), dict(batch_size=0, total_q=0),
                                    dict(total_q=30, q_start_loc=9 << 20, max_q_len=0), dict(head_dim=72), dict(block_size=8),
                                    dict(groups=9), dict(key_cache=(2 << 20) + 8)], ids=str)
def test_good_calls_only_lack_their_context(change):
    rc, msg = call(**change)
    assert rc == _lib.KYRO_EINVAL and "null kyro_ctx" in msg, msg


@pytest.mark.parametrize("change, status, text", [
    (dict(groups=-1), "EINVAL", "num_groups"), (dict(path=1), "EINVAL", "AUTO"), (dict(schedule=2), "EINVAL", "AUTO"),
    (dict(num_splits=2), "EINVAL", "AUTO"), (dict(num_heads=7), "EINVAL", "num_kv_heads"), (dict(head_dim=68), "EUNSUPPORTED", "head_dim 68"),
    (dict(dtype=2), "EINVAL", "dtype"), (dict(total_q=5), "EINVAL", "batch_size"), (dict(kv_reuse=3), "EINVAL", "kv_reuse"),
    (dict(group_starts=None), "EINVAL", "null device pointer"), (dict(group_blocks=None), "EINVAL", "null device pointer"),
    (dict(out=None), "EINVAL", "null device pointer")], ids=str)
def test_refusals(change, status, text):
    rc, msg = call(**change)
    assert rc == getattr(_lib, "KYRO_" + status) and text in msg, msg


def workspace(groups=1, **change):
    p = _lib.PagedAttentionParams(**dict(GOOD, **change))
    n = ctypes.c_size_t(7)
    rc = _lib.lib().kyro_paged_attention_shared_workspace(None, ctypes.byref(p), 1, groups, ctypes.byref(n))
    return rc, n.value


def test_workspace():
    plain = ctypes.c_size_t()
    p = _lib.PagedAttentionParams(**dict(GOOD, kv_reuse=1))
    assert _lib.lib().kyro_paged_attention_workspace(None, ctypes.byref(p), 1, ctypes.byref(plain)) == _lib.KYRO_OK
    assert workspace(groups=0) == (_lib.KYRO_OK, plain.value)  # no groups: the other entry point's launch
    assert workspace()[1] > plain.value
    assert workspace(batch_size=0, total_q=0) == (_lib.KYRO_OK, 0)
    assert workspace(groups=-1) == (_lib.KYRO_EINVAL, 0) and workspace(head_dim=12) == (_lib.KYRO_EUNSUPPORTED, 0)
    assert _lib.lib().kyro_paged_attention_shared_workspace(None, None, 1, 1, ctypes.byref(plain)) == _lib.KYRO_EINVAL
    assert _lib.lib().kyro_paged_attention_shared_workspace(None, ctypes.byref(p), 1, 1, None) == _lib.KYRO_EINVAL
    # 64 sequences of 8 rows, 32/8 heads: tens of MB
    assert workspace(num_heads=32, num_kv_heads=8, batch_size=64, total_q=512, max_q_len=8)[1] < 100 << 20
