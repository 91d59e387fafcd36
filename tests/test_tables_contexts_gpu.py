"""Tables of two servers at once, a stream and a context each: extend and release keep what they hand from one launch to
the next in the context's scratch."""
import numpy as np
import pytest
import torch

import kyro_amd
from kyro_amd import RequestTables

pytestmark = pytest.mark.gpu


class Server:
    def __init__(self, gpu, seed, B, width):
        rng = np.random.default_rng(seed)
        self.width, self.gpu = width, gpu
        self.t = RequestTables.new(16, rows=B + 5, max_blocks=width, pool=rng.permutation(B * width), num_blocks=B * width, device=gpu)
        self.rows = torch.from_numpy(rng.permutation(B + 5)[:B].astype(np.int32)).to(gpu)
        self.new = [torch.from_numpy(rng.integers(1, 300, B).astype(np.int32)).to(gpu) for _ in range(4)]
        self.totals = [int(x.sum()) for x in self.new]

    def run(self, context):
        """Four steps of which all rows stay, and the end of every request; on the current stream."""
        got = []
        for new, total in zip(self.new, self.totals):
            step = self.t.extend_async(self.rows, new, total_q=total, max_blocks_per_seq=40000, context=context)
            lens = self.t.keep_async(self.rows, step.context_lens, step.q_start_loc, new, context=context)
            got += [*step[1:], step.block_table[:, : self.width].clone(), lens]
        self.t.release_async(self.rows, context=context)
        return got + [self.t.requests, self.t.blocks, self.t.pool, self.t.pool_count]


def test_two_contexts_at_once(gpu):
    shapes = [(1, 24, 100), (2, 9, 90)]
    alone = [[x.clone() for x in Server(gpu, *s).run(None)] for s in shapes]
    kyro_amd.sync()
    servers = [Server(gpu, *s) for s in shapes]
    streams, contexts = [torch.cuda.Stream(gpu) for _ in shapes], [kyro_amd.Context(0) for _ in shapes]
    torch.cuda.synchronize()
    got = []
    for s, stream, context in zip(servers, streams, contexts):
        with torch.cuda.stream(stream):
            got.append(s.run(context))
    for c in contexts:
        c.sync()
    for a, b in zip(alone, got):
        assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))
