"""Block tables that live on the GPU: what each request holds, a pool of free blocks, and the tables of a step.

The reference's scheduler keeps block tables on the host (src/scheduler/block_manager.rs:15-153), and so does
:class:`kyro_amd.BlockManager`, which has to know how many drafts a verify step accepted before it can lay out the
next. Here requests and free blocks are device tensors, so that steps follow each other without a host in between:

    bm = BlockManager(16, num_gpu_blocks)
    tables = RequestTables.new(16, rows=256, max_blocks=2048, pool=bm.allocate(POOL_ID, 16 * 30000),
                               num_blocks=num_gpu_blocks, device=device)
    tables.admit(row, blocks_of_a_cached_prefix, tokens_cached)          # on the host, once a request
    step = tables.extend_async(state_rows, new_rows, total_q=total_q)    # each step
    q = kv.append_qkv_async(q, k, v, key_cache, value_cache, step.block_table, step.context_lens, cos=cos, sin=sin,
                            positions=step.positions, q_start_loc=step.q_start_loc)
    out = attn.forward_async(q, key_cache, value_cache, step.block_table, step.context_lens,
                             q_start_loc=step.q_start_loc, max_q_len=max_q_len)
    res = verify_drafts_async(...)
    tables.keep_async(state_rows, step.context_lens, step.q_start_loc, res.accepted, plus=1)
"""
from __future__ import annotations

from typing import NamedTuple

import numpy as np
import torch

from . import _lib
from .kv_cache import _require


class StepTables(NamedTuple):
    """What the calls of a step read: see :meth:`RequestTables.extend`."""

    block_table: torch.Tensor   # [B, max_blocks_per_seq] int64
    context_lens: torch.Tensor  # [B] int64, the new rows included
    q_start_loc: torch.Tensor   # [B + 1] int32
    positions: torch.Tensor     # [total_q] int64: a row's position in its request
    slots: torch.Tensor         # [total_q] int64: block * block_size + offset, its place in the caches


class RequestTables:
    """``requests`` [rows, 4] int32: tokens, blocks held, blocks at the front that are not the pool's, unused.
    ``blocks`` [rows, max_blocks] int64: the ids a request holds, in order. ``pool`` [capacity] int64: ids of free
    blocks, of which the first ``pool_count`` ([1] int32) count. All contiguous, on one GPU, and written in place."""

    def __init__(self, block_size: int, requests, blocks, pool, pool_count, num_blocks: int):
        self.block_size = int(block_size)
        self.num_blocks = int(num_blocks)
        if not isinstance(requests, torch.Tensor):
            raise TypeError("requests must be a torch.Tensor")
        dev = requests.device
        _require(requests, "requests", (torch.int32,), 2, dev)
        _require(blocks, "blocks", (torch.int64,), 2, dev)
        _require(pool, "pool", (torch.int64,), 1, dev)
        _require(pool_count, "pool_count", (torch.int32,), 1, dev)
        if requests.shape[1] != 4 or blocks.shape[0] != requests.shape[0] or pool_count.shape[0] != 1:
            raise ValueError(f"requests must be [rows, 4], blocks [rows, max_blocks] and pool_count [1], got "
                             f"{tuple(requests.shape)}, {tuple(blocks.shape)}, {tuple(pool_count.shape)}")
        self.requests, self.blocks, self.pool, self.pool_count = requests, blocks, pool, pool_count
        self.device = dev
        self._index = requests.get_device()

    @classmethod
    def new(cls, block_size: int, *, rows: int, max_blocks: int, pool, num_blocks: int, device):
        """State for ``rows`` requests of up to ``max_blocks`` blocks; ``pool``: the ids of the free blocks."""
        ids = torch.as_tensor(np.asarray(pool, dtype=np.int64).reshape(-1))
        return cls(block_size, torch.zeros((int(rows), 4), dtype=torch.int32, device=device),
                   torch.zeros((int(rows), int(max_blocks)), dtype=torch.int64, device=device), ids.to(device),
                   torch.tensor([ids.numel()], dtype=torch.int32, device=device), num_blocks)

    def admit(self, row: int, blocks=(), tokens: int = 0) -> None:
        """A new request in a row that holds none: ``tokens`` cached tokens in ``blocks`` (ids, host), which stay
        whose they are, as the prefix that a block manager's request or its prefix cache holds. Its first new rows
        may not lie in a block that others read."""
        ids = np.asarray(blocks, dtype=np.int64).reshape(-1)
        row, tokens = int(row), int(tokens)
        if not 0 <= row < self.requests.shape[0]:
            raise ValueError(f"row {row} is not in [0, {self.requests.shape[0]})")
        if ids.size > self.blocks.shape[1] or not 0 <= tokens <= ids.size * self.block_size:
            raise ValueError(f"{tokens} tokens in {ids.size} blocks of {self.block_size} (at most {self.blocks.shape[1]})")
        if ids.size:
            self.blocks[row, : ids.size] = torch.as_tensor(ids, device=self.device)
        self.requests[row] = torch.tensor([tokens, ids.size, ids.size, 0], dtype=torch.int32, device=self.device)

    def _vector(self, t, name, dtype, n):
        # One expression for a tensor as it should be; _require names what is not.
        if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.numel() == n and t.dim() == 1
                and t.get_device() == self._index and t.is_contiguous()):
            return
        _require(t, name, (dtype,), 1, self.device)
        if t.shape[0] != n:
            raise ValueError(f"{name} must have {n} entries, got {t.shape[0]}")

    def _batch(self, state_rows, entries):
        if state_rows is not None:
            self._vector(state_rows, "state_rows", torch.int32, entries)
        elif entries > self.requests.shape[0]:
            raise ValueError("without state_rows every entry of the batch needs a request of the state")

    def _context(self, context=None):
        idx = self._index
        if idx < 0:
            raise ValueError("RequestTables runs on a GPU device; got " + str(self.device))
        ctx = context if context is not None else _lib.context(idx)
        ctx.set_stream(_lib.current_stream(idx))
        return ctx

    def _params(self, entries, width=0, max_rows=0, plus=0):
        return _lib.pack_tables(self.block_size, entries, width, self.requests.shape[0], self.blocks.shape[1],
                                self.num_blocks, self.pool.shape[0], max_rows, plus)

    def extend_async(self, state_rows, new_rows, *, total_q, max_blocks_per_seq=None, out=None,
                     context=None) -> StepTables:
        """Queues the work on torch's current stream; see :meth:`extend`. ``context`` (a ``kyro_amd.Context``) runs
        the call on that context and its arena instead of the process-wide one, for programs that keep a context a
        stream."""
        if not isinstance(new_rows, torch.Tensor):
            raise TypeError("new_rows must be a torch.Tensor")
        entries = new_rows.shape[0] if new_rows.dim() == 1 else -1
        self._vector(new_rows, "new_rows", torch.int32, entries)
        self._batch(state_rows, entries)
        total_q = int(total_q)
        width = self.blocks.shape[1] if max_blocks_per_seq is None else int(max_blocks_per_seq)
        if out is None:
            # One allocation for all but the row ranges: five of them cost 7.0 us a call, this 4.8.
            new = self.requests.new_empty
            table, ctx_lens, positions, slots = torch.split_with_sizes(
                new((entries * width + entries + 2 * total_q,), dtype=torch.int64),
                (entries * width, entries, total_q, total_q))
            out = StepTables(table.view(entries, width), ctx_lens, new((entries + 1,)), positions, slots)
        else:
            out = StepTables(*out)
            _require(out.block_table, "out.block_table", (torch.int64,), 2, self.device)
            if out.block_table.shape != (entries, width):
                raise ValueError(f"out.block_table must be {(entries, width)}, got {tuple(out.block_table.shape)}")
            self._vector(out.context_lens, "out.context_lens", torch.int64, entries)
            self._vector(out.q_start_loc, "out.q_start_loc", torch.int32, entries + 1)
            self._vector(out.positions, "out.positions", torch.int64, total_q)
            self._vector(out.slots, "out.slots", torch.int64, total_q)
        if entries == 0:
            out.q_start_loc.zero_()
            out.positions.fill_(-1)
            out.slots.fill_(-1)
            return out
        ctx = self._context(context)
        _lib.check(_lib.lib().kyro_tables_extend(
            ctx.handle, self._params(entries, width, total_q), None if state_rows is None else state_rows.data_ptr(),
            new_rows.data_ptr(), self.requests.data_ptr(), self.blocks.data_ptr(), self.pool.data_ptr(),
            self.pool_count.data_ptr(), out.block_table.data_ptr(), out.context_lens.data_ptr(),
            out.q_start_loc.data_ptr(), out.positions.data_ptr(), out.slots.data_ptr()))
        return out

    def extend(self, state_rows, new_rows, *, total_q, max_blocks_per_seq=None, out=None) -> StepTables:
        """Room for ``new_rows`` (int32 [B]) more rows of the batch's requests ``state_rows`` (int32 [B]; None: request
        b; negative: padding), and the tables of the step: blocks come off the pool in the order of the batch where
        those held do not reach. ``total_q`` bounds the rows in all (positions and slots behind the last one are -1),
        ``max_blocks_per_seq`` is the width of the block table (None: the state's). The requests' lengths
        change with :meth:`keep`; until then the call can be repeated. ``out`` (a :class:`StepTables`) is written
        instead of new tensors. An entry without room has context length 0. The call synchronises, so a pool
        with too few blocks raises KyroError (KYRO_ENOSPACE) here, and so does a bad state row, record or
        length."""
        step = self.extend_async(state_rows, new_rows, total_q=total_q, max_blocks_per_seq=max_blocks_per_seq, out=out)
        _lib.context(self.device.index or 0).sync()
        return step

    def keep_async(self, state_rows, context_lens, q_start_loc, kept, *, plus=0, out=None, context=None):
        """Queues the work on torch's current stream; see :meth:`keep` (``context`` as for :meth:`extend_async`)."""
        if not isinstance(context_lens, torch.Tensor):
            raise TypeError("context_lens must be a torch.Tensor")
        entries = context_lens.shape[0] if context_lens.dim() == 1 else -1
        self._vector(context_lens, "context_lens", torch.int64, entries)
        self._vector(q_start_loc, "q_start_loc", torch.int32, entries + 1)
        self._vector(kept, "kept", torch.int32, entries)
        self._batch(state_rows, entries)
        if out is None:
            out = torch.empty_like(context_lens)
        else:
            self._vector(out, "out", torch.int64, entries)
        if entries == 0:
            return out
        ctx = self._context(context)
        _lib.check(_lib.lib().kyro_tables_keep(
            ctx.handle, self._params(entries, plus=int(plus)), None if state_rows is None else state_rows.data_ptr(),
            context_lens.data_ptr(), q_start_loc.data_ptr(), kept.data_ptr(), self.requests.data_ptr(),
            self.blocks.data_ptr(), self.pool.data_ptr(), self.pool_count.data_ptr(), out.data_ptr()))
        return out

    def keep(self, state_rows, context_lens, q_start_loc, kept, *, plus=0, out=None):
        """Of a step's rows (``context_lens`` and ``q_start_loc`` as :meth:`extend` gave them) the first ``kept`` (int32
        [B]) + ``plus`` of each entry stay: the requests' lengths count them, and blocks behind them go back to the pool.
        After :func:`kyro_amd.verify_drafts` that is ``res.accepted`` and 1. Returns the lengths that stay (int64
        [B], 0 for an entry of context length 0, as extend leaves one out, whose request is left alone); ``out`` may be ``context_lens``. The call synchronises, so
        errors the device detects raise KyroError here."""
        out = self.keep_async(state_rows, context_lens, q_start_loc, kept, plus=plus, out=out)
        _lib.context(self.device.index or 0).sync()
        return out

    def release_async(self, state_rows, *, context=None) -> None:
        """Queues the work on torch's current stream; see :meth:`release` (``context`` as for :meth:`extend_async`)."""
        if not isinstance(state_rows, torch.Tensor):
            raise TypeError("state_rows must be a torch.Tensor")
        entries = state_rows.shape[0] if state_rows.dim() == 1 else -1
        self._batch(state_rows, entries)
        if entries == 0:
            return
        ctx = self._context(context)
        _lib.check(_lib.lib().kyro_tables_release(
            ctx.handle, self._params(entries), state_rows.data_ptr(), self.requests.data_ptr(), self.blocks.data_ptr(),
            self.pool.data_ptr(), self.pool_count.data_ptr()))

    def release(self, state_rows) -> None:
        """Ends the requests ``state_rows`` (int32 [n]): their blocks, but for the shared ones, go back to the pool
        and their records become 0. Synchronises."""
        self.release_async(state_rows)
        _lib.context(self.device.index or 0).sync()
