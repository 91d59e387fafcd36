"""kyro_qkv_append without a GPU: what the entry point refuses, and the rotation tables in 64 bits."""
import ctypes
import math

import numpy as np
import pytest
import torch

import kyro_amd
from kyro_amd import _lib

GOOD = dict(block_size=16, num_heads=8, num_kv_heads=2, head_dim=64, batch_size=2, total_q=2, max_blocks_per_seq=4,
            num_blocks=9, src_dtype=_lib.KYRO_BF16, cache_dtype=_lib.KYRO_BF16, rotary_dim=64, interleaved=0,
            max_position=128, norm=1, weight_dtype=_lib.KYRO_BF16, eps=1e-6, weight_offset=0.0, query_stride=0,
            key_stride=0, value_stride=0)
# Addresses that no call dereferences: every check here is the host's, and a call that passes them all
# ends at its null context.
POINTERS = dict(query=1 << 20, key=2 << 20, value=3 << 20, q_start_loc=None, positions=None, block_table=4 << 20,
                context_lens=5 << 20, cos=6 << 20, sin=7 << 20, q_weight=8 << 20, k_weight=9 << 20,
                key_cache=10 << 20, value_cache=11 << 20, out_query=12 << 20)


def call(**change):
    params = _lib.QkvAppendParams(**{k: change.get(k, v) for k, v in GOOD.items()})
    ptrs = [change.get(k, v) for k, v in POINTERS.items()]
    return _lib.lib().kyro_qkv_append(None, ctypes.byref(params), *ptrs), _lib.last_error()


def test_a_good_call_only_lacks_its_context():
    rc, msg = call()
    assert rc == _lib.KYRO_EINVAL and "null kyro_ctx" in msg
    for change in (dict(interleaved=1, rotary_dim=62), dict(rotary_dim=0, cos=None, sin=None), dict(total_q=0, batch_size=0),
                   dict(norm=0, q_weight=None, k_weight=None), dict(query_stride=768, key_stride=768, value_stride=768),
                   dict(out_query=1 << 20), dict(head_dim=72, rotary_dim=20), dict(total_q=7, q_start_loc=13 << 20)):
        rc, msg = call(**change)
        assert rc == _lib.KYRO_EINVAL and "null kyro_ctx" in msg, (change, msg)


@pytest.mark.parametrize("change, status, text", [
    (dict(block_size=0), "EINVAL", "sizes"), (dict(num_blocks=0), "EINVAL", "sizes"), (dict(total_q=-1), "EINVAL", "sizes"),
    (dict(num_heads=7), "EINVAL", "num_kv_heads"), (dict(head_dim=60), "EUNSUPPORTED", "head_dim 60"),
    (dict(head_dim=264), "EUNSUPPORTED", "head_dim 264"), (dict(rotary_dim=66), "EINVAL", "rotary_dim"),
    (dict(rotary_dim=31), "EINVAL", "rotary_dim"), (dict(rotary_dim=62), "EUNSUPPORTED", "multiple of 4"),
    (dict(src_dtype=2), "EINVAL", "dtype"), (dict(cache_dtype=5), "EINVAL", "dtype"), (dict(weight_dtype=-1), "EINVAL", "dtype"),
    (dict(cos=None), "EINVAL", "cos"), (dict(max_position=0), "EINVAL", "max_position"),
    (dict(eps=-1.0), "EINVAL", "eps"), (dict(eps=0.0), "EINVAL", "eps"), (dict(eps=1e-39), "EINVAL", "eps"),
    (dict(eps=math.nan), "EINVAL", "eps"), (dict(weight_offset=math.inf), "EINVAL", "offset"),
    (dict(norm=0), "EINVAL", "norm weights"), (dict(k_weight=None), "EINVAL", "norm weights"),
    (dict(total_q=3), "EINVAL", "batch_size"), (dict(query_stride=500), "EINVAL", "strides"),
    (dict(key_stride=132), "EINVAL", "strides"), (dict(value_stride=-128), "EINVAL", "strides"),
    (dict(query=None), "EINVAL", "null device pointer"), (dict(block_table=None), "EINVAL", "null device pointer"),
    (dict(key=(2 << 20) + 8), "EINVAL", "16-byte"), (dict(sin=(7 << 20) + 4), "EINVAL", "16-byte"),
    (dict(out_query=(1 << 20) + 64), "EINVAL", "overlaps"), (dict(out_query=2 << 20), "EINVAL", "overlaps"),
    (dict(out_query=1 << 20, query_stride=768), "EINVAL", "overlaps"),
    (dict(out_query=1 << 20, src_dtype=_lib.KYRO_F32), "EINVAL", "overlaps"),
    (dict(total_q=2**31 - 1, q_start_loc=13 << 20, out_query=1 << 45, key=1 << 46, value=1 << 47), "EUNSUPPORTED", "one launch")])
def test_refusals(change, status, text):
    rc, msg = call(**change)
    assert rc == getattr(_lib, "KYRO_" + status) and text in msg, msg


def test_null_params():
    assert _lib.lib().kyro_qkv_append(None, None, *([None] * 14)) == _lib.KYRO_EINVAL


def test_struct_mirrors_the_header():
    from tests.test_abi import struct_fields

    assert [f[0] for f in _lib.QkvAppendParams._fields_] == struct_fields("kyro_qkv_append_params")


def test_rope_tables_hold_far_angles():
    """Angles in 64 bits, rounded once: at most half a step of a float32 in [-1, 1] (2^-25) from the cosine."""
    cos, sin = kyro_amd.rope_tables(200_001, 64, 10000.0)
    assert cos.shape == sin.shape == (200_001, 32) and cos.dtype == torch.float32
    for pos in (0, 1, 99_999, 200_000):
        angle = pos * 10000.0 ** (-np.arange(0, 64, 2) / 64)
        assert np.abs(cos[pos].double().numpy() - np.cos(angle)).max() <= 2.0 ** -25 + 1e-10
        assert np.abs(sin[pos].double().numpy() - np.sin(angle)).max() <= 2.0 ** -25 + 1e-10


def test_rope_tables_own_frequencies_and_refusals():
    cos, sin = kyro_amd.rope_tables(4, 4, inv_freq=[1.0, 0.5], scale=2.0)
    assert torch.allclose(cos[3], 2 * torch.cos(torch.tensor([3.0, 1.5])))
    assert torch.allclose(sin[3], 2 * torch.sin(torch.tensor([3.0, 1.5])))
    for bad in (dict(max_position=0, rotary_dim=4), dict(max_position=4, rotary_dim=3),
                dict(max_position=4, rotary_dim=4, inv_freq=[1.0])):
        with pytest.raises(ValueError):
            kyro_amd.rope_tables(**bad)


# ------------------------------------------------------------------------------------ the Python entry's own checks

class OnGpu(torch.Tensor):
    """A host tensor that says it is on a GPU: the library behind the checks is a stub here."""

    def get_device(self):
        return 0

    @property
    def device(self):
        return torch.device("cuda", 0)

    @property
    def is_cuda(self):
        return True


class Recorder:
    """Stands for the library and a context: keeps the parameters of a call that passes the checks."""

    handle, params = None, None

    def set_stream(self, stream):
        pass

    def kyro_qkv_append(self, handle, params, *pointers):
        self.params = _lib.QkvAppendParams.from_buffer_copy(params)
        return _lib.KYRO_OK


@pytest.fixture
def recorder(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(_lib, "lib", lambda: r)
    monkeypatch.setattr(_lib, "context", lambda idx: r)
    monkeypatch.setattr(_lib, "current_stream", lambda idx: 0)
    return r


def python_call(rows=5, heads=8, **change):
    """append_qkv_async of one sequence's rows with host tensors in place of the GPU's."""
    t = dict(query=torch.zeros(rows, heads, 64), key=torch.zeros(rows, 2, 64), value=torch.zeros(rows, 2, 64),
             key_cache=torch.zeros(9, 2, 16, 64), value_cache=torch.zeros(9, 2, 16, 64),
             block_table=torch.zeros(1, 4, dtype=torch.int64), context_lens=torch.full((1,), rows),
             q_start_loc=torch.tensor([0, rows], dtype=torch.int32), out=torch.zeros(rows, heads, 64))
    t.update(change)
    return kyro_amd.PagedKVCache(16, 2, 64).append_qkv_async(**{k: v.as_subclass(OnGpu) for k, v in t.items()})


@pytest.mark.parametrize("name,heads", [("query", 8), ("key", 2), ("value", 2)])
def test_rows_that_share_memory_are_refused(recorder, name, heads):
    """The library reads a stride of 0 as that of dense rows: rows of an expanded tensor would be read behind it."""
    for bad in (torch.zeros(1, heads, 64).expand(5, heads, 64), torch.zeros(heads + 4, 64).as_strided((5, heads, 64), (64, 64, 1))):
        with pytest.raises(ValueError, match=f"{name}'s rows"):
            python_call(**{name: bad})
    assert recorder.params is None
    # With one query head as well, where torch leaves the head stride open.
    if name == "query":
        with pytest.raises(ValueError, match="query's rows"):
            kv = kyro_amd.PagedKVCache(16, 1, 64)
            one = {k: torch.zeros(5, 1, 64).as_subclass(OnGpu) for k in ("key", "value", "out")}
            caches = {k: torch.zeros(9, 1, 16, 64).as_subclass(OnGpu) for k in ("key_cache", "value_cache")}
            kv.append_qkv_async(torch.zeros(1, 1, 64).expand(5, 1, 64).as_subclass(OnGpu), **one, **caches,
                                block_table=torch.zeros(1, 4, dtype=torch.int64).as_subclass(OnGpu),
                                context_lens=torch.full((1,), 5).as_subclass(OnGpu),
                                q_start_loc=torch.tensor([0, 5], dtype=torch.int32).as_subclass(OnGpu))


def test_row_strides_that_reach_the_library(recorder):
    packed = torch.zeros(5, 12, 64)
    python_call(query=packed[:, :8], key=packed[:, 8:10], value=packed[:, 10:])
    p = recorder.params
    assert (p.query_stride, p.key_stride, p.value_stride) == (768, 768, 768)
    python_call()
    p = recorder.params
    assert (p.query_stride, p.key_stride, p.value_stride) == (512, 128, 128)
    # One row has no next one: any stride is as good as the dense one.
    python_call(rows=1, query=torch.zeros(1, 8, 64).as_strided((1, 8, 64), (0, 64, 1)), key=torch.zeros(2, 64).expand(1, 2, 64))
    p = recorder.params
    for stride, heads in ((p.query_stride, 8), (p.key_stride, 2), (p.value_stride, 2)):
        assert stride in (0, heads * 64)


FAR = dict(query=1 << 40, key=2 << 40, value=3 << 40, out_query=4 << 40, q_start_loc=13 << 20)


@pytest.mark.parametrize("sizes, fits", [
    # A grid has fewer than 2^32 threads: at most 2^24 - 1 workgroups of four waves. A wave takes a row of 64 heads
    # of 8 elements (rotary_dim 0), or one head of 256 on 32 lanes.
    (dict(num_heads=1, num_kv_heads=1, head_dim=8, total_q=2**26 - 4), True),
    (dict(num_heads=1, num_kv_heads=1, head_dim=8, total_q=2**26 - 3), False),
    (dict(num_heads=62, num_kv_heads=1, head_dim=8, total_q=2**26 - 4), True),
    (dict(num_heads=63, num_kv_heads=1, head_dim=8, total_q=2**25), False),
    # heads that pass 32 bits when they are added up
    (dict(num_heads=2**29, num_kv_heads=2**29, head_dim=8, total_q=1), True),
    (dict(num_heads=2**30, num_kv_heads=2**30, head_dim=8, total_q=1), False),
    (dict(num_heads=2**31 - 1, num_kv_heads=2**31 - 1, head_dim=8, total_q=1), False)])
def test_what_one_launch_carries(sizes, fits):
    rc, msg = call(**FAR, rotary_dim=0, cos=None, sin=None, norm=0, q_weight=None, k_weight=None, **sizes)
    if fits:
        assert rc == _lib.KYRO_EINVAL and "null kyro_ctx" in msg, msg
    else:
        assert rc == _lib.KYRO_EUNSUPPORTED and "one launch" in msg, msg
