"""Caches that keep the tokens attention uses: accumulated attention weights, and eviction by them.

The reference's caches only grow (src/model/kv_cache.rs:49-75). Here a sequence's paged cache can be held to a
budget: every step adds up the softmax weight each cached token receives, and a cache over the budget keeps,
for each kv head, its first tokens, its newest, and those of the most weight. Kept tokens from behind the
budget move into the slots of the ones that go, so caches, block tables and context lengths stay what
:class:`kyro_amd.PagedAttention` reads.

    state = ev.new_state(rows, max_tokens, device)               # weights, positions, beside each layer's cache
    kv.append_qkv(..., positions=positions)                      # rows rotated by their own positions
    ev.accumulate(query, key_cache, block_table, context_lens, *state, row_positions=positions)
    bm.make_private(rid); copy_blocks(key_cache, value_cache, bm.take_copies())
    context_lens = ev.evict(key_cache, value_cache, block_table, context_lens, *state, budget=2048)
    bm.truncate(rid, 2048)
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .kv_cache import _DTYPES, _require


class CacheEviction:
    """The geometry of one layer's cache (as :class:`kyro_amd.PagedAttention`)."""

    def __init__(self, block_size: int, num_heads: int, head_dim: int, num_kv_heads: int):
        self.block_size = int(block_size)
        self.num_heads = int(num_heads)
        self.head_dim = int(head_dim)
        self.num_kv_heads = int(num_kv_heads)

    def new_state(self, rows: int, max_tokens: int, device):
        """(weights, positions) for ``rows`` sequences of up to ``max_tokens`` cached tokens: no weight yet, and
        every token at the position of its slot."""
        shape = (int(rows), self.num_kv_heads, int(max_tokens))
        weights = torch.zeros(shape, dtype=torch.float32, device=device)
        positions = torch.arange(shape[2], dtype=torch.int32, device=device).expand(shape).contiguous()
        return weights, positions

    def _cache(self, cache, name, dtypes, dev):
        _require(cache, name, dtypes, 4, dev)
        want = (cache.shape[0], self.num_kv_heads, self.block_size, self.head_dim)
        if tuple(cache.shape) != want:
            raise ValueError(f"{name} must be {want}, got {tuple(cache.shape)}")

    def _state(self, t, name, dtype, dev, like=None):
        _require(t, name, (dtype,), 3, dev)
        if t.shape[1] != self.num_kv_heads or (like is not None and t.shape != like.shape):
            raise ValueError(f"{name} must be [rows, {self.num_kv_heads}, max_tokens]"
                             + ("" if like is None else f" like weights, {tuple(like.shape)}") + f", got {tuple(t.shape)}")

    def _batch(self, block_table, context_lens, state_rows, weights, dev):
        _require(block_table, "block_table", (torch.int64,), 2, dev)
        _require(context_lens, "context_lens", (torch.int64,), 1, dev)
        B = context_lens.shape[0]
        if block_table.shape[0] != B:
            raise ValueError("block_table and context_lens disagree on the batch size")
        if state_rows is not None:
            _require(state_rows, "state_rows", (torch.int32,), 1, dev)
            if state_rows.shape[0] != B:
                raise ValueError("state_rows must have one entry per sequence")
        elif weights.shape[0] < B:
            raise ValueError("without state_rows weights needs a row per sequence")
        return B

    def accumulate_async(self, query, key_cache, block_table, context_lens, weights, positions, *, q_start_loc=None,
                         max_q_len=None, row_positions=None, state_rows=None, causal=True, scale=None, out=None):
        """Queues the work on torch's current stream and returns the weights; see :meth:`accumulate`."""
        dev = query.device
        if dev.type != "cuda":
            raise ValueError("accumulate runs on a GPU device; got " + str(dev))
        _require(query, "query", (torch.float32, torch.bfloat16), 3, dev)
        self._cache(key_cache, "key_cache", (query.dtype,), dev)
        total_q, h, d = query.shape
        if (h, d) != (self.num_heads, self.head_dim):
            raise ValueError(f"query shape {tuple(query.shape)} does not match (*, {self.num_heads}, {self.head_dim})")
        self._state(weights, "weights", torch.float32, dev)
        self._state(positions, "positions", torch.int32, dev, weights)
        if out is None:
            out = weights
        else:
            self._state(out, "out", torch.float32, dev, weights)
        B = self._batch(block_table, context_lens, state_rows, weights, dev)
        if q_start_loc is not None:
            _require(q_start_loc, "q_start_loc", (torch.int32,), 1, dev)
            if q_start_loc.shape[0] != B + 1:
                raise ValueError("q_start_loc must have batch+1 entries")
            if max_q_len is None:
                max_q_len = int((q_start_loc[1:] - q_start_loc[:-1]).max().item()) if B else 1
        else:
            if total_q != B:
                raise ValueError("query rows must equal the batch size without q_start_loc")
            max_q_len = 1
        if row_positions is not None:
            _require(row_positions, "row_positions", (torch.int64,), 1, dev)
            if row_positions.shape[0] != total_q:
                raise ValueError("row_positions must have one entry per row")
        params = _lib.AttnWeightsParams(
            self.block_size, h, d, self.num_kv_heads, B, total_q, block_table.shape[1], key_cache.shape[0],
            _DTYPES[query.dtype], 1 if causal else 0, float(scale) if scale else 0.0, int(max_q_len), weights.shape[0],
            weights.shape[2])
        ctx = _lib.context(dev.index or 0)
        ctx.set_stream(_lib.current_stream(dev.index or 0))
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        _lib.check(_lib.lib().kyro_attn_weights(
            ctx.handle, ctypes.byref(params), query.data_ptr(), ptr(q_start_loc), ptr(row_positions),
            key_cache.data_ptr(), block_table.data_ptr(), context_lens.data_ptr(), ptr(state_rows),
            weights.data_ptr(), out.data_ptr(), positions.data_ptr()))
        return out

    def accumulate(self, query, key_cache, block_table, context_lens, weights, positions, *, q_start_loc=None,
                   max_q_len=None, row_positions=None, state_rows=None, causal=True, scale=None, out=None):
        """Adds to ``weights`` [rows, Hkv, max_tokens] what each cached token receives of the attention of
        ``query``'s rows (the arguments of :meth:`kyro_amd.PagedAttention.forward`, after the append), summed over
        the rows and over each kv head's query heads, and returns them. The step's own new tokens start from
        zero, and their entries of ``positions`` (int32, like weights) become ``row_positions`` (int64
        [total_q]; None: the slots). ``state_rows`` (int32 [B]) names the rows of weights and positions that the
        sequences own; by default sequence b owns row b. ``out`` receives the weights instead of weights itself.
        The call synchronises, so errors the device detects raise KyroError here."""
        out = self.accumulate_async(query, key_cache, block_table, context_lens, weights, positions,
                                    q_start_loc=q_start_loc, max_q_len=max_q_len, row_positions=row_positions,
                                    state_rows=state_rows, causal=causal, scale=scale, out=out)
        _lib.context(query.device.index or 0).sync()
        return out

    def evict_async(self, key_cache, value_cache, block_table, context_lens, weights, positions, *, budget, sink=4,
                    recent=0, state_rows=None, out=None):
        """Queues the work on torch's current stream and returns the new context lengths; see :meth:`evict`."""
        dev = key_cache.device
        if dev.type != "cuda":
            raise ValueError("evict runs on a GPU device; got " + str(dev))
        self._cache(key_cache, "key_cache", (torch.float32, torch.bfloat16), dev)
        self._cache(value_cache, "value_cache", (key_cache.dtype,), dev)
        if value_cache.shape != key_cache.shape:
            raise ValueError("key_cache and value_cache shapes differ")
        self._state(weights, "weights", torch.float32, dev)
        self._state(positions, "positions", torch.int32, dev, weights)
        out_weights, out_positions = (weights, positions) if out is None else out
        if out is not None:
            self._state(out_weights, "out[0]", torch.float32, dev, weights)
            self._state(out_positions, "out[1]", torch.int32, dev, weights)
        B = self._batch(block_table, context_lens, state_rows, weights, dev)
        lens = torch.empty_like(context_lens)
        params = _lib.KvEvictParams(
            self.block_size, self.num_kv_heads, self.head_dim, B, block_table.shape[1], key_cache.shape[0],
            _DTYPES[key_cache.dtype], int(budget), int(sink), int(recent), weights.shape[0], weights.shape[2])
        ctx = _lib.context(dev.index or 0)
        ctx.set_stream(_lib.current_stream(dev.index or 0))
        _lib.check(_lib.lib().kyro_kv_evict(
            ctx.handle, ctypes.byref(params), key_cache.data_ptr(), value_cache.data_ptr(), block_table.data_ptr(),
            context_lens.data_ptr(), state_rows.data_ptr() if state_rows is not None else None, weights.data_ptr(),
            positions.data_ptr(), out_weights.data_ptr(), out_positions.data_ptr(), lens.data_ptr()))
        return lens

    def evict(self, key_cache, value_cache, block_table, context_lens, weights, positions, *, budget, sink=4, recent=0,
              state_rows=None, out=None):
        """Cuts every sequence of more than ``budget`` tokens to it, in place, and returns the new context lengths
        (min(length, budget)). Each kv head keeps the tokens at positions below ``sink``, the ``recent`` newest
        positions, and of the others those of the most weight (ties: the lower slot). Kept tokens in slots >=
        budget move, in ascending order, into the slots of the ones that go; all others stay where they are. K, V,
        weight and position move together. ``out`` (weights, positions) receives the kept entries instead of the
        inputs. A sequence's blocks must be its own: :meth:`kyro_amd.BlockManager.make_private`. The call
        synchronises, so errors the device detects raise KyroError here."""
        lens = self.evict_async(key_cache, value_cache, block_table, context_lens, weights, positions, budget=budget,
                                sink=sink, recent=recent, state_rows=state_rows, out=out)
        _lib.context(key_cache.device.index or 0).sync()
        return lens
