"""Paged KV write — host mirror of KVCacheManager::append_kv for a block-table cache.

The reference keeps one growing [1, seq, Hkv, D] tensor per request and appends the new rows
with a concatenation before attention (src/model/kv_cache.rs:49-75, called at
src/model/llama.rs:80-84). Here the cache is the paged [num_blocks, Hkv, block_size, D] layout
that :class:`kyro_amd.PagedAttention` reads, and a batch of sequences appends in one launch:
new row j of a sequence with q_len new rows and context length ctx (counted after the append,
as attention counts it) lands at token position ctx - q_len + j.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.KYRO_F32, torch.bfloat16: _lib.KYRO_BF16}


def _require(t, name, dtypes, ndim, device):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, expected one of {dtypes}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must be {ndim}-D, got shape {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def rope_tables(max_position: int, rotary_dim: int, base: float = 10000.0, *, inv_freq=None, scale: float = 1.0,
                device=None):
    """(cos, sin) of every position's angles, [max_position, rotary_dim / 2] float32 each, for
    :meth:`PagedKVCache.append_qkv` (RotaryEmbedding, src/model/layers.rs:21-62). Frequency i is
    base^(-2 i / rotary_dim), or ``inv_freq`` (rotary_dim / 2 numbers) for a model that scales them;
    ``scale`` multiplies both tables. The angles are computed in 64 bits: in 32, position 100000 would be
    off by 0.004 radians."""
    max_position, rotary_dim = int(max_position), int(rotary_dim)
    if max_position <= 0 or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("max_position must be positive and rotary_dim a positive even number")
    if inv_freq is None:
        freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    else:
        freq = torch.as_tensor(inv_freq, dtype=torch.float64, device="cpu").reshape(-1)
        if freq.numel() != rotary_dim // 2:
            raise ValueError(f"inv_freq has {freq.numel()} entries, expected {rotary_dim // 2}")
    angle = torch.outer(torch.arange(max_position, dtype=torch.float64), freq)
    return tuple((f(angle) * scale).to(torch.float32).to(device) for f in (torch.cos, torch.sin))


def _rows(t, name, dtype, shape, device):
    """Element stride between the rows of a [rows, heads, D] tensor whose heads are dense (a slice of a
    wider projection's output may be)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    n, h, d = shape
    st = t.stride()
    if (d > 1 and st[2] != 1) or (h > 1 and st[1] != d):
        raise ValueError(f"{name}'s heads must be dense: strides (any, {d}, 1), got {st}")
    if n > 1 and st[0] < h * d:  # an expanded tensor's 0 would stand for dense rows in the library
        raise ValueError(f"{name}'s rows must not share memory: a row stride of at least {h * d}, got {st[0]}")
    return st[0]


class PagedKVCache:
    """Writes new K/V rows into block-table caches (kv_cache.rs:21-35 holds num_kv_heads and
    head_dim; the block size is the paged layout's)."""

    def __init__(self, block_size: int, num_kv_heads: int, head_dim: int):
        self.block_size = int(block_size)
        self.num_kv_heads = int(num_kv_heads)
        self.head_dim = int(head_dim)

    def append_kv_async(self, key, value, key_cache, value_cache, block_table, context_lens, *,
                        q_start_loc=None, max_q_len=None):
        """Queues the write on torch's current stream; see :meth:`append_kv`."""
        dev = key.device
        if dev.type != "cuda":
            raise ValueError("append_kv runs on a GPU device; got " + str(dev))
        _require(key, "key", (torch.float32, torch.bfloat16), 3, dev)
        _require(value, "value", (key.dtype,), 3, dev)
        _require(key_cache, "key_cache", (torch.float32, torch.bfloat16), 4, dev)
        _require(value_cache, "value_cache", (key_cache.dtype,), 4, dev)
        _require(block_table, "block_table", (torch.int64,), 2, dev)
        _require(context_lens, "context_lens", (torch.int64,), 1, dev)
        total_q, hkv, d = key.shape
        if tuple(value.shape) != tuple(key.shape):
            raise ValueError("key and value must have the same shape")
        if hkv != self.num_kv_heads or d != self.head_dim:
            raise ValueError(f"key rows are [{hkv}, {d}], expected [{self.num_kv_heads}, {self.head_dim}]")
        nb = key_cache.shape[0]
        want = (nb, self.num_kv_heads, self.block_size, self.head_dim)
        if tuple(key_cache.shape) != want or tuple(value_cache.shape) != want:
            raise ValueError(f"caches must be {want}")
        B = context_lens.shape[0]
        if block_table.shape[0] != B:
            raise ValueError("block_table and context_lens disagree on the batch size")
        if q_start_loc is not None:
            _require(q_start_loc, "q_start_loc", (torch.int32,), 1, dev)
            if q_start_loc.shape[0] != B + 1:
                raise ValueError("q_start_loc must have batch+1 entries")
            if max_q_len is None:
                max_q_len = int((q_start_loc[1:] - q_start_loc[:-1]).max().item()) if B else 0
        else:
            if total_q != B:
                raise ValueError("without q_start_loc key must have one row per sequence")
            max_q_len = 1
        params = _lib.KvAppendParams(self.block_size, self.num_kv_heads, self.head_dim, B, total_q,
                                     block_table.shape[1], nb, _DTYPES[key.dtype],
                                     _DTYPES[key_cache.dtype], int(max_q_len))
        ctx = _lib.context(dev.index or 0)
        ctx.set_stream(_lib.current_stream(dev.index or 0))
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        _lib.check(_lib.lib().kyro_paged_kv_append(
            ctx.handle, ctypes.byref(params), ptr(key), ptr(value), ptr(q_start_loc),
            ptr(block_table), ptr(context_lens), ptr(key_cache), ptr(value_cache)))

    def append_qkv_async(self, query, key, value, key_cache, value_cache, block_table, context_lens, *, cos=None,
                         sin=None, positions=None, q_weight=None, k_weight=None, norm_eps=None, weight_offset=0.0,
                         interleaved=False, q_start_loc=None, out=None):
        """Queues the pass on torch's current stream and returns the query; see :meth:`append_qkv`."""
        # One expression for a call whose tensors are as they should be; _qkv_require names what is not.
        hkv, bs, d = self.num_kv_heads, self.block_size, self.head_dim
        try:
            idx, src, dst = query.get_device(), query.dtype, key_cache.dtype
            total_q, heads, _ = query.shape
            B, width = block_table.shape
            kv, cache, rows = key.shape, key_cache.shape, total_q
            (q_stride, qh, q1), (k_stride, kh, k1), (v_stride, vh, v1) = query.stride(), key.stride(), value.stride()
            nb = cache[0]
            plain = (idx >= 0 and src in _DTYPES and dst in _DTYPES and key.dtype == src and value.dtype == src
                     and query.shape[2] == d and kv == (rows, hkv, d) and value.shape == kv and rows > 0
                     and q1 == 1 and k1 == 1 and v1 == 1 and qh == d and kh == d and vh == d
                     and q_stride >= heads * d and k_stride >= hkv * d and v_stride >= hkv * d
                     and key.get_device() == idx and value.get_device() == idx
                     and cache == (nb, hkv, bs, d) and value_cache.shape == cache and value_cache.dtype == dst
                     and key_cache.is_contiguous() and value_cache.is_contiguous()
                     and key_cache.get_device() == idx and value_cache.get_device() == idx
                     and block_table.dtype == torch.int64 and block_table.is_contiguous()
                     and block_table.get_device() == idx and context_lens.dtype == torch.int64
                     and context_lens.shape == (B,) and context_lens.is_contiguous() and context_lens.get_device() == idx
                     and (rows == B if q_start_loc is None else
                          q_start_loc.dtype == torch.int32 and q_start_loc.shape == (B + 1,)
                          and q_start_loc.is_contiguous() and q_start_loc.get_device() == idx)
                     and (positions is None or (positions.dtype == torch.int64 and positions.shape == (rows,)
                                                and positions.is_contiguous() and positions.get_device() == idx)))
        except (AttributeError, ValueError, IndexError):  # not a tensor, or not of the right rank
            plain = False
        if not plain:
            q_stride, k_stride, v_stride = self._qkv_require(query, key, value, key_cache, value_cache, block_table,
                                                             context_lens, q_start_loc, positions)
            idx, src, dst = query.get_device(), query.dtype, key_cache.dtype
            (total_q, heads, _), (B, width), nb = query.shape, block_table.shape, key_cache.shape[0]
        if total_q == 1:  # torch gives a single row any stride
            q_stride = k_stride = v_stride = 0
        rotary = max_position = 0
        weight_dtype = src
        try:
            if cos is not None:
                max_position, half = turn = cos.shape
                rotary = 2 * half
                plain = (cos.dtype == torch.float32 and sin.dtype == torch.float32 and sin.shape == turn
                         and cos.is_contiguous() and sin.is_contiguous() and cos.get_device() == idx
                         and sin.get_device() == idx)
            else:
                plain = sin is None
            if q_weight is not None:
                weight_dtype = q_weight.dtype
                plain = (plain and norm_eps is not None and weight_dtype in _DTYPES and k_weight.dtype == weight_dtype
                         and q_weight.shape == (d,) and k_weight.shape == (d,) and q_weight.is_contiguous()
                         and k_weight.is_contiguous() and q_weight.get_device() == idx and k_weight.get_device() == idx)
            else:
                plain = plain and k_weight is None
        except (AttributeError, ValueError):
            plain = False
        if not plain:
            self._turn_require(query.device, cos, sin, q_weight, k_weight, norm_eps)
        if out is None:
            out = query.new_empty((total_q, heads, d), dtype=dst)
        else:
            _require(out, "out", (dst,), 3, query.device)
            if out.shape != query.shape:
                raise ValueError("out has the wrong shape")
        params = _lib.pack_qkv_append(bs, heads, hkv, d, B, total_q, width, nb, _DTYPES[src], _DTYPES[dst], rotary,
                                      1 if interleaved else 0, max_position, 0 if norm_eps is None else 1,
                                      _DTYPES[weight_dtype], 0.0 if norm_eps is None else norm_eps, weight_offset,
                                      q_stride, k_stride, v_stride)
        ctx = _lib.context(idx)
        ctx.set_stream(_lib.current_stream(idx))
        _lib.check(_lib.lib().kyro_qkv_append(
            ctx.handle, params, query.data_ptr(), key.data_ptr(), value.data_ptr(),
            None if q_start_loc is None else q_start_loc.data_ptr(), None if positions is None else positions.data_ptr(),
            block_table.data_ptr(), context_lens.data_ptr(), None if cos is None else cos.data_ptr(),
            None if sin is None else sin.data_ptr(), None if q_weight is None else q_weight.data_ptr(),
            None if k_weight is None else k_weight.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
            out.data_ptr()))
        return out

    def _turn_require(self, dev, cos, sin, q_weight, k_weight, norm_eps):
        """Raises what is wrong with append_qkv's tables and weights."""
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin come together")
        if cos is not None:
            _require(cos, "cos", (torch.float32,), 2, dev)
            _require(sin, "sin", (torch.float32,), 2, dev)
            if cos.shape != sin.shape:
                raise ValueError("cos and sin must have the same shape")
        if (q_weight is None) != (k_weight is None):
            raise ValueError("q_weight and k_weight come together")
        if q_weight is not None:
            if norm_eps is None:
                raise ValueError("norm weights need norm_eps")
            _require(q_weight, "q_weight", (torch.float32, torch.bfloat16), 1, dev)
            _require(k_weight, "k_weight", (q_weight.dtype,), 1, dev)
            if q_weight.shape[0] != self.head_dim or k_weight.shape[0] != self.head_dim:
                raise ValueError(f"norm weights must have {self.head_dim} entries")

    def _qkv_require(self, query, key, value, key_cache, value_cache, block_table, context_lens, q_start_loc, positions):
        """Raises what is wrong with append_qkv's tensors; (query, key, value) row strides where nothing is."""
        if not isinstance(query, torch.Tensor):
            raise TypeError("query must be a torch.Tensor")
        dev = query.device
        if dev.type != "cuda":
            raise ValueError("append_qkv runs on a GPU device; got " + str(dev))
        if query.dtype not in _DTYPES:
            raise TypeError(f"query has dtype {query.dtype}, expected one of {tuple(_DTYPES)}")
        if query.dim() != 3:
            raise ValueError(f"query must be 3-D, got shape {tuple(query.shape)}")
        src, (total_q, heads, d) = query.dtype, query.shape
        hkv, bs = self.num_kv_heads, self.block_size
        if d != self.head_dim:
            raise ValueError(f"query heads have {d} elements, expected {self.head_dim}")
        strides = (_rows(query, "query", src, (total_q, heads, d), dev), _rows(key, "key", src, (total_q, hkv, d), dev),
                   _rows(value, "value", src, (total_q, hkv, d), dev))
        _require(key_cache, "key_cache", (torch.float32, torch.bfloat16), 4, dev)
        _require(value_cache, "value_cache", (key_cache.dtype,), 4, dev)
        _require(block_table, "block_table", (torch.int64,), 2, dev)
        _require(context_lens, "context_lens", (torch.int64,), 1, dev)
        want = (key_cache.shape[0], hkv, bs, d)
        if tuple(key_cache.shape) != want or tuple(value_cache.shape) != want:
            raise ValueError(f"caches must be {want}")
        B = context_lens.shape[0]
        if block_table.shape[0] != B:
            raise ValueError("block_table and context_lens disagree on the batch size")
        if q_start_loc is not None:
            _require(q_start_loc, "q_start_loc", (torch.int32,), 1, dev)
            if q_start_loc.shape[0] != B + 1:
                raise ValueError("q_start_loc must have batch+1 entries")
        elif total_q != B:
            raise ValueError("without q_start_loc query must have one row per sequence")
        if positions is not None:
            _require(positions, "positions", (torch.int64,), 1, dev)
            if positions.shape[0] != total_q:
                raise ValueError("positions must have one entry per row")
        return strides

    def append_qkv(self, query, key, value, key_cache, value_cache, block_table, context_lens, *, cos=None, sin=None,
                   positions=None, q_weight=None, k_weight=None, norm_eps=None, weight_offset=0.0, interleaved=False,
                   q_start_loc=None, out=None):
        """Head norms, rotation and :meth:`append_kv` of a step's new rows in one launch; returns the query
        that :class:`kyro_amd.PagedAttention` takes, [total_q, H, D] in the caches' dtype (or ``out``, which
        may be ``query`` itself where that is contiguous and of the caches' dtype).

        ``query`` [total_q, H, D], ``key`` and ``value`` [total_q, Hkv, D] are the projections' rows; they may
        be slices of one [total_q, H + 2 Hkv, D] output, but no expanded tensors, whose rows share memory.
        ``cos`` and ``sin`` (:func:`rope_tables`) turn the first ``2 * cos.shape[1]`` elements of each query
        and key head, element i with i + half of them, or neighbours with ``interleaved``; without them nothing
        turns. ``positions`` (int64 [total_q]) are the tables' rows; by default a row's slot in its sequence,
        which it no longer is after :meth:`kyro_amd.CacheEviction.evict`. ``norm_eps`` (> 0) asks for the
        root-mean-square norm of each query and key head, scaled by ``q_weight`` / ``k_weight``
        (+ ``weight_offset``) where given. The call
        synchronises, so a bad block id, context length or position raises KyroError here."""
        out = self.append_qkv_async(query, key, value, key_cache, value_cache, block_table, context_lens, cos=cos,
                                    sin=sin, positions=positions, q_weight=q_weight, k_weight=k_weight,
                                    norm_eps=norm_eps, weight_offset=weight_offset, interleaved=interleaved,
                                    q_start_loc=q_start_loc, out=out)
        _lib.context(query.device.index or 0).sync()
        return out

    def append_kv(self, key, value, key_cache, value_cache, block_table, context_lens, *,
                  q_start_loc=None, max_q_len=None):
        """Appends each sequence's new rows (``key``/``value`` [total_q, Hkv, D], rows of sequence b
        at [q_start_loc[b], q_start_loc[b+1]) or row b without q_start_loc) to the caches in place
        and synchronises, so a bad block id or context length raises KyroError here.
        ``context_lens`` is each sequence's length after the append."""
        self.append_kv_async(key, value, key_cache, value_cache, block_table, context_lens,
                             q_start_loc=q_start_loc, max_q_len=max_q_len)
        _lib.context(key.device.index or 0).sync()
