"""Caches that keep the tokens attention uses: accumulated attention weights, and eviction by them.

The reference's caches only grow (src/model/kv_cache.rs:49-75). Here a sequence's paged cache can be held to a
budget: every step adds up the softmax weight each cached token receives, and a cache over the budget keeps,
for each kv head, its first tokens, its newest, and those of the most weight. Kept tokens from behind the
budget move into the slots of the ones that go, so caches, block tables and context lengths stay what
:class:`kyro_amd.PagedAttention` reads.

    state = ev.new_state(rows, max_tokens, device)               # weights, positions, beside each layer's cache
    kv.append_qkv(..., positions=positions)                      # rows rotated by their own positions
    ev.accumulate(query, key_cache, block_table, context_lens, *state, row_positions=positions)
    bm.make_private(rid, 2048); copy_blocks(key_cache, value_cache, bm.take_copies())
    context_lens = ev.evict(key_cache, value_cache, block_table, context_lens, *state, budget=2048)
    bm.truncate(rid, 2048)
"""
from __future__ import annotations

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
        # One expression for a call whose tensors are as they should be; _accumulate_require names what is not.
        hkv, bs, h, d = self.num_kv_heads, self.block_size, self.num_heads, self.head_dim
        if out is None:
            out = weights
        try:
            idx, dtype = query.get_device(), query.dtype
            total_q = query.shape[0]
            B, width = block_table.shape
            cache, state = key_cache.shape, weights.shape
            nb = cache[0]
            plain = (idx >= 0 and dtype in _DTYPES and query.shape == (total_q, h, d) and query.is_contiguous()
                     and key_cache.dtype == dtype and cache == (nb, hkv, bs, d) and key_cache.is_contiguous()
                     and key_cache.get_device() == idx and len(state) == 3 and state[1] == hkv
                     and weights.dtype == torch.float32 and out.dtype == torch.float32 and positions.dtype == torch.int32
                     and out.shape == state and positions.shape == state and weights.is_contiguous()
                     and out.is_contiguous() and positions.is_contiguous() and weights.get_device() == idx
                     and out.get_device() == idx and positions.get_device() == idx
                     and block_table.dtype == torch.int64 and block_table.is_contiguous()
                     and block_table.get_device() == idx and context_lens.dtype == torch.int64
                     and context_lens.shape == (B,) and context_lens.is_contiguous() and context_lens.get_device() == idx
                     and (total_q == B if q_start_loc is None else
                          max_q_len is not None and q_start_loc.dtype == torch.int32 and q_start_loc.shape == (B + 1,)
                          and q_start_loc.is_contiguous() and q_start_loc.get_device() == idx)
                     and (state[0] >= B if state_rows is None else
                          state_rows.dtype == torch.int32 and state_rows.shape == (B,) and state_rows.is_contiguous()
                          and state_rows.get_device() == idx)
                     and (row_positions is None or (
                         row_positions.dtype == torch.int64 and row_positions.shape == (total_q,)
                         and row_positions.is_contiguous() and row_positions.get_device() == idx)))
        except (AttributeError, ValueError, IndexError):  # not a tensor, or not of the right rank
            plain = False
        if not plain:
            max_q_len = self._accumulate_require(query, key_cache, block_table, context_lens, weights, positions, out,
                                                 q_start_loc, max_q_len, row_positions, state_rows)
            idx, dtype, total_q = query.get_device(), query.dtype, query.shape[0]
            (B, width), state, nb = block_table.shape, weights.shape, key_cache.shape[0]
        params = _lib.pack_attn_weights(bs, h, d, hkv, B, total_q, width, nb, _DTYPES[dtype], 1 if causal else 0,
                                        scale or 0.0, 1 if q_start_loc is None else max_q_len, state[0], state[2])
        ctx = _lib.context(idx)
        ctx.set_stream(_lib.current_stream(idx))
        _lib.check(_lib.lib().kyro_attn_weights(
            ctx.handle, params, query.data_ptr(), None if q_start_loc is None else q_start_loc.data_ptr(),
            None if row_positions is None else row_positions.data_ptr(), key_cache.data_ptr(), block_table.data_ptr(),
            context_lens.data_ptr(), None if state_rows is None else state_rows.data_ptr(), weights.data_ptr(),
            out.data_ptr(), positions.data_ptr()))
        return out

    def _accumulate_require(self, query, key_cache, block_table, context_lens, weights, positions, out, q_start_loc,
                            max_q_len, row_positions, state_rows):
        """Raises what is wrong with accumulate's tensors; the most rows of a sequence where nothing is."""
        if not isinstance(query, torch.Tensor):
            raise TypeError("query must be a torch.Tensor")
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
        self._state(out, "out", torch.float32, dev, weights)
        B = self._batch(block_table, context_lens, state_rows, weights, dev)
        if row_positions is not None:
            _require(row_positions, "row_positions", (torch.int64,), 1, dev)
            if row_positions.shape[0] != total_q:
                raise ValueError("row_positions must have one entry per row")
        if q_start_loc is None:
            if total_q != B:
                raise ValueError("query rows must equal the batch size without q_start_loc")
            return 1
        _require(q_start_loc, "q_start_loc", (torch.int32,), 1, dev)
        if q_start_loc.shape[0] != B + 1:
            raise ValueError("q_start_loc must have batch+1 entries")
        if max_q_len is None:
            max_q_len = int((q_start_loc[1:] - q_start_loc[:-1]).max().item()) if B else 1
        return int(max_q_len)

    def accumulate(self, query, key_cache, block_table, context_lens, weights, positions, *, q_start_loc=None,
                   max_q_len=None, row_positions=None, state_rows=None, causal=True, scale=None, out=None):
        """Adds to ``weights`` [rows, Hkv, max_tokens] what each cached token receives of the attention of
        ``query``'s rows (the arguments of :meth:`kyro_amd.PagedAttention.forward`, after the append), summed over
        the rows and over each kv head's query heads, and returns them. The step's own new tokens start from
        zero, and their entries of ``positions`` (int32, like weights) become ``row_positions`` (int64
        [total_q]; None: the slots). Every row weighs: after a verify step call it once acceptance is known, with
        the rows and context lengths that stay. ``state_rows`` (int32 [B]) names the rows of weights and positions
        that the sequences own; by default sequence b owns row b. ``out`` receives the weights of every sequence's
        tokens (of one without rows as they are) instead of weights itself; its other entries stay. The call
        synchronises, so errors the device detects raise KyroError here."""
        out = self.accumulate_async(query, key_cache, block_table, context_lens, weights, positions,
                                    q_start_loc=q_start_loc, max_q_len=max_q_len, row_positions=row_positions,
                                    state_rows=state_rows, causal=causal, scale=scale, out=out)
        _lib.context(query.device.index or 0).sync()
        return out

    def evict_async(self, key_cache, value_cache, block_table, context_lens, weights, positions, *, budget, sink=4,
                    recent=0, state_rows=None, out=None):
        """Queues the work on torch's current stream and returns the new context lengths; see :meth:`evict`."""
        # One expression for a call whose tensors are as they should be; _evict_require names what is not.
        hkv, bs, d = self.num_kv_heads, self.block_size, self.head_dim
        out_weights, out_positions = (weights, positions) if out is None else out
        try:
            idx, dtype = key_cache.get_device(), key_cache.dtype
            B, width = block_table.shape
            cache, state = key_cache.shape, weights.shape
            nb = cache[0]
            plain = (idx >= 0 and dtype in _DTYPES and cache == (nb, hkv, bs, d) and key_cache.is_contiguous()
                     and value_cache.shape == cache and value_cache.dtype == dtype and value_cache.is_contiguous()
                     and value_cache.get_device() == idx and len(state) == 3 and state[1] == hkv
                     and weights.dtype == torch.float32 and out_weights.dtype == torch.float32
                     and positions.dtype == torch.int32 and out_positions.dtype == torch.int32
                     and out_weights.shape == state and positions.shape == state and out_positions.shape == state
                     and weights.is_contiguous() and out_weights.is_contiguous() and positions.is_contiguous()
                     and out_positions.is_contiguous() and weights.get_device() == idx
                     and out_weights.get_device() == idx and positions.get_device() == idx
                     and out_positions.get_device() == idx and block_table.dtype == torch.int64
                     and block_table.is_contiguous() and block_table.get_device() == idx
                     and context_lens.dtype == torch.int64 and context_lens.shape == (B,)
                     and context_lens.is_contiguous() and context_lens.get_device() == idx
                     and (state[0] >= B if state_rows is None else
                          state_rows.dtype == torch.int32 and state_rows.shape == (B,) and state_rows.is_contiguous()
                          and state_rows.get_device() == idx))
        except (AttributeError, ValueError, IndexError):  # not a tensor, or not of the right rank
            plain = False
        if not plain:
            self._evict_require(key_cache, value_cache, block_table, context_lens, weights, positions, out_weights,
                                out_positions, state_rows)
            idx, dtype, nb = key_cache.get_device(), key_cache.dtype, key_cache.shape[0]
            (B, width), state = block_table.shape, weights.shape
        lens = torch.empty_like(context_lens)
        params = _lib.pack_kv_evict(bs, hkv, d, B, width, nb, _DTYPES[dtype], budget, sink, recent, state[0], state[2])
        ctx = _lib.context(idx)
        ctx.set_stream(_lib.current_stream(idx))
        _lib.check(_lib.lib().kyro_kv_evict(
            ctx.handle, params, key_cache.data_ptr(), value_cache.data_ptr(), block_table.data_ptr(),
            context_lens.data_ptr(), None if state_rows is None else state_rows.data_ptr(), weights.data_ptr(),
            positions.data_ptr(), out_weights.data_ptr(), out_positions.data_ptr(), lens.data_ptr()))
        return lens

    def _evict_require(self, key_cache, value_cache, block_table, context_lens, weights, positions, out_weights,
                       out_positions, state_rows):
        """Raises what is wrong with evict's tensors."""
        if not isinstance(key_cache, torch.Tensor):
            raise TypeError("key_cache must be a torch.Tensor")
        dev = key_cache.device
        if dev.type != "cuda":
            raise ValueError("evict runs on a GPU device; got " + str(dev))
        self._cache(key_cache, "key_cache", (torch.float32, torch.bfloat16), dev)
        self._cache(value_cache, "value_cache", (key_cache.dtype,), dev)
        if value_cache.shape != key_cache.shape:
            raise ValueError("key_cache and value_cache shapes differ")
        self._state(weights, "weights", torch.float32, dev)
        self._state(positions, "positions", torch.int32, dev, weights)
        self._state(out_weights, "out[0]", torch.float32, dev, weights)
        self._state(out_positions, "out[1]", torch.int32, dev, weights)
        self._batch(block_table, context_lens, state_rows, weights, dev)

    def evict(self, key_cache, value_cache, block_table, context_lens, weights, positions, *, budget, sink=4, recent=0,
              state_rows=None, out=None):
        """Cuts every sequence of more than ``budget`` tokens to it, in place, and returns the new context lengths
        (min(length, budget)). Each kv head keeps the tokens at positions below ``sink``, the ``recent`` newest
        positions, and of the others those of the most weight (ties: the lower slot). Kept tokens in slots >=
        budget move, in ascending order, into the slots of the ones that go; all others stay where they are. K, V,
        weight and position move together. ``out`` (weights, positions) receives the kept entries instead of the
        inputs. The blocks of a sequence's first ``budget`` slots must be its own:
        :meth:`kyro_amd.BlockManager.make_private`. The call synchronises, so errors the device detects raise
        KyroError here."""
        lens = self.evict_async(key_cache, value_cache, block_table, context_lens, weights, positions, budget=budget,
                                sink=sink, recent=recent, state_rows=state_rows, out=out)
        _lib.context(key_cache.device.index or 0).sync()
        return lens
