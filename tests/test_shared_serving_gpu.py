"""Steps as a server runs them, all of it on the GPU: tables extended, new keys and values appended, attention over
shared prefixes, drafts verified, and the rows that stay kept; against a model of the requests on the host."""
import numpy as np
import pytest
import torch

import kyro_amd
from kyro_amd import BlockManager, PagedAttention, PagedKVCache, RequestTables, StepTables, verify_drafts_async

pytestmark = pytest.mark.gpu

BS, H, HKV, D, V, DRAFTS = 16, 8, 2, 128, 64, 3
DOCUMENT, SYSTEM = 150, 90  # tokens that four requests, and two others, start with: 9 and 5 whole blocks
POOL = 10_000


class Server:
    """Seven requests, an entry of padding, and what the host knows of them."""

    def __init__(self, gpu, seed):
        self.gpu = gpu
        self.rng = np.random.default_rng(seed)
        self.gen = torch.Generator().manual_seed(seed)
        num_blocks = 256
        bm = BlockManager(BS, num_blocks)
        prompts = {}
        doc, system = self.rng.integers(0, 1000, DOCUMENT), self.rng.integers(1000, 2000, SYSTEM)
        for rid, (front, own) in enumerate([(doc, 3), (system, 40), (doc, 20), (None, 35), (doc, 1), (system, 2), (doc, 17)]):
            tail = self.rng.integers(2000 + 100 * rid, 2100 + 100 * rid, own)
            prompts[rid] = tail if front is None else np.concatenate([front, tail])
        for rid, p in prompts.items():  # the cache has them from an earlier turn
            assert bm.allocate_with_prefix(1000 + rid, p) is not None
            bm.free(1000 + rid)
        for rid, p in prompts.items():
            assert bm.allocate_with_prefix(rid, np.append(p, 5000 + rid)) is not None
        bm.take_copies()
        ids = sorted(prompts)
        order, starts, blocks = bm.prefix_groups(ids)
        self.rids = [ids[i] for i in order]
        self.group_starts, self.group_blocks = torch.from_numpy(starts).to(gpu), torch.from_numpy(blocks).to(gpu)
        assert sorted(blocks.tolist()) == [0, SYSTEM // BS, DOCUMENT // BS]
        self.prefix = {}
        for g, nb in enumerate(blocks):
            for i in range(starts[g], starts[g + 1]):
                self.prefix[self.rids[i]] = int(nb)

        shape = (num_blocks, HKV, BS, D)
        self.kc = torch.full(shape, float("nan"), dtype=torch.bfloat16, device=gpu)
        self.vc = torch.full(shape, float("nan"), dtype=torch.bfloat16, device=gpu)
        pool = bm.allocate(POOL, BS * 60)
        self.tables = RequestTables.new(BS, rows=16, max_blocks=40, pool=pool, num_blocks=num_blocks, device=gpu)
        self.state = {rid: 2 * rid + 1 for rid in self.rids}
        self.k, self.v = {}, {}  # [tokens, HKV, D] of each request, on the host
        written = {}
        for rid in self.rids:
            held = bm.request(rid)[0][: self.prefix[rid]]
            for b in held:
                if b not in written:
                    written[b] = self.rows(2 * BS)
                    for cache, x in ((self.kc, written[b][:BS]), (self.vc, written[b][BS:])):
                        cache[b] = x.transpose(0, 1).to(gpu)
            none = torch.zeros((0, HKV, D), dtype=torch.bfloat16)
            self.k[rid] = torch.cat([none] + [written[b][:BS] for b in held])
            self.v[rid] = torch.cat([none] + [written[b][BS:] for b in held])
            self.tables.admit(self.state[rid], held, BS * len(held))
        self.chunk = {rid: len(prompts[rid]) - len(self.k[rid]) for rid in self.rids}
        self.state_rows = torch.tensor([self.state[r] for r in self.rids] + [-1], dtype=torch.int32, device=gpu)
        self.attn, self.kv = PagedAttention(BS, H, D, HKV), PagedKVCache(BS, HKV, D)

    def rows(self, n, heads=HKV):
        return torch.randn((n, heads, D), generator=self.gen).to(torch.bfloat16)

    def inputs(self, new):
        """A step's query, keys and values, and what the drafts are verified against, on the host."""
        B = len(self.rids) + 1
        q, k, v = self.rows(self.total, H), self.rows(self.total), self.rows(self.total)
        target, draft = torch.randn((B, DRAFTS + 1, V), generator=self.gen), torch.randn((B, DRAFTS, V), generator=self.gen)
        return [torch.tensor(new, dtype=torch.int32), q, k, v, target, draft,
                torch.randint(0, V, (B, DRAFTS), generator=self.gen, dtype=torch.int32),
                torch.rand((B, DRAFTS), generator=self.gen), torch.rand((B,), generator=self.gen)]

    def attend(self, tables, new, q, k, v, kc, vc, most, step=None, out=None):
        step = tables.extend_async(self.state_rows, new, total_q=self.total, max_blocks_per_seq=40, out=step)
        q = self.kv.append_qkv_async(q, k, v, kc, vc, step.block_table, step.context_lens, positions=step.positions,
                                     q_start_loc=step.q_start_loc)
        out = self.attn.forward_shared_async(q, kc, vc, step.block_table, step.context_lens, self.group_starts,
                                             self.group_blocks, q_start_loc=step.q_start_loc, max_q_len=most, out=out)
        return step, out

    def verify(self, tables, step, target, draft, tokens, u, ur):
        B = len(self.rids) + 1
        drafts = torch.full((B,), DRAFTS, dtype=torch.int32, device=self.gpu)
        ones = torch.ones(B, device=self.gpu)
        res = verify_drafts_async(target, draft, tokens, drafts, ones, u, ur)
        return res.accepted, tables.keep_async(self.state_rows, step.context_lens, step.q_start_loc, res.accepted, plus=1)

    total = 192  # the prompts have 162 rows that no whole cached block holds

    def check(self, step, out, new, q, k, v):
        """Attention of every row in 64 bits; a weight and nothing else is rounded, by at most 2^-8 of it (half a step of
        8 bits), and sums in 32 bits add less than 2^-12 of their terms' size."""
        starts = np.concatenate([[0], np.cumsum(new)])
        assert step.q_start_loc.tolist() == starts.tolist()
        out = out.double().cpu()
        for b, rid in enumerate(self.rids):
            q0, q1 = int(starts[b]), int(starts[b + 1])
            keys, values = (torch.cat([x[rid], y[q0:q1]]).double() for x, y in ((self.k, k), (self.v, v)))
            ctx = len(keys)
            assert int(step.context_lens[b]) == ctx and step.positions[q0:q1].tolist() == list(range(ctx - (q1 - q0), ctx))
            for j in range(q0, q1):
                n = ctx - (q1 - q0) + (j - q0) + 1
                qj = q[j].double().view(HKV, H // HKV, D)
                p = torch.softmax(torch.einsum("khd,tkd->kht", qj, keys[:n]) / D ** 0.5, -1)
                exact = torch.einsum("kht,tkd->khd", p, values[:n]).reshape(H, D)
                size = torch.einsum("kht,tkd->khd", p, values[:n].abs()).reshape(H, D)
                err = (out[j] - exact).abs()
                assert (err <= (2.0 ** -8 + 2.0 ** -12) * size + 1e-30).all(), (rid, j, float((err / size).max()))

    def stay(self, new, kept, k, v):
        starts = np.concatenate([[0], np.cumsum(new)])
        for b, rid in enumerate(self.rids):
            q0 = int(starts[b])
            for x, y in ((self.k, k), (self.v, v)):
                x[rid] = torch.cat([x[rid], y[q0:q0 + kept[b]]])


def prefill(s):
    """The prompts' rows that no cached block holds, all of which stay."""
    new = [s.chunk[r] for r in s.rids] + [0]
    host = s.inputs(new)
    dev = [x.to(s.gpu) for x in host]
    step, out = s.attend(s.tables, *dev[:4], s.kc, s.vc, max(new))
    lens = s.tables.keep_async(s.state_rows, step.context_lens, step.q_start_loc, dev[0], plus=0)
    torch.cuda.synchronize()
    s.check(step, out, new, *host[1:4])
    s.stay(new, new, *host[2:4])
    assert lens.tolist() == [len(s.k[r]) for r in s.rids] + [0]


@pytest.mark.parametrize("side", [False, True])
def test_a_server_s_steps(gpu, side):
    """Prompts behind cached prefixes, then verify steps; `side`: all on a stream of its own."""
    s = Server(gpu, 3)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream(gpu) if side else torch.cuda.current_stream(gpu)
    with torch.cuda.stream(stream):
        prefill(s)
        for _ in range(6):
            new = [DRAFTS + 1] * len(s.rids) + [0]
            host = s.inputs(new)
            dev = [x.to(gpu) for x in host]
            step, out = s.attend(s.tables, *dev[:4], s.kc, s.vc, DRAFTS + 1)
            accepted, lens = s.verify(s.tables, step, *dev[4:])
            torch.cuda.synchronize()
            s.check(step, out, new, *host[1:4])
            s.stay(new, (accepted[:-1] + 1).tolist(), *host[2:4])
            assert lens.tolist() == [len(s.k[r]) for r in s.rids] + [0]
        s.tables.release(s.state_rows[:-1].contiguous())
    assert int(s.tables.pool_count) == 60 and sorted(s.tables.pool.tolist()) == sorted(set(s.tables.pool.tolist()))


def test_a_captured_step_against_an_eager_one(gpu):
    """The whole step as a graph, replayed with other inputs each time; an eager step on copies of the state and the caches
    runs between the replays and has to give the same bits."""
    s = Server(gpu, 5)
    prefill(s)
    new = [DRAFTS + 1] * len(s.rids) + [0]
    static = [x.to(gpu) for x in s.inputs(new)]
    copies = RequestTables(BS, *(x.clone() for x in (s.tables.requests, s.tables.blocks, s.tables.pool, s.tables.pool_count)),
                           s.tables.num_blocks)
    kc, vc = s.kc.clone(), s.vc.clone()
    s.attend(copies, *static[:4], kc, vc, DRAFTS + 1)  # scratch grows to what the step needs; extend can be repeated
    torch.cuda.synchronize()
    B, long = len(s.rids) + 1, torch.int64
    given = StepTables(*(torch.zeros(n, dtype=t, device=gpu) for n, t in
                         (((B, 40), long), (B, long), (B + 1, torch.int32), (s.total, long), (s.total, long))))
    out = torch.zeros((s.total, H, D), device=gpu)
    stream = torch.cuda.Stream(gpu)
    stream.wait_stream(torch.cuda.current_stream(gpu))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step, _ = s.attend(s.tables, *static[:4], s.kc, s.vc, DRAFTS + 1, given, out)
        accepted, lens = s.verify(s.tables, step, *static[4:])
    for _ in range(5):
        host = s.inputs(new)
        for x, y in zip(static, host):
            x.copy_(y)
        graph.replay()
        eager = [x.to(gpu) for x in host]
        want, want_out = s.attend(copies, *eager[:4], kc, vc, DRAFTS + 1)
        want_accepted, want_lens = s.verify(copies, want, *eager[4:])
        torch.cuda.synchronize()
        rows = sum(new)
        for a, b in zip(step, want):
            assert torch.equal(a, b)
        assert torch.equal(out[:rows], want_out[:rows]) and torch.equal(accepted, want_accepted) and torch.equal(lens, want_lens)
        for a, b in ((s.tables.requests, copies.requests), (s.tables.blocks, copies.blocks), (s.tables.pool, copies.pool),
                     (s.tables.pool_count, copies.pool_count)):
            assert torch.equal(a, b)
        s.check(step, out, new, *host[1:4])
        s.stay(new, (accepted[:-1] + 1).tolist(), *host[2:4])


def test_two_contexts_at_once(gpu):
    """Batches that differ, on two streams with a context and so scratch each: what each gives alone."""
    gen = torch.Generator().manual_seed(9)
    attn = PagedAttention(BS, H, D, HKV)

    def batch(B, common, own, rows):
        blocks = common + own
        table = torch.randperm(B * blocks, generator=gen).view(B, blocks)
        table[:, :common] = table[0, :common]
        caches = torch.randn((2, B * blocks, HKV, BS, D), generator=gen).to(torch.bfloat16).to(gpu)
        q = torch.randn((B * rows, H, D), generator=gen).to(torch.bfloat16).to(gpu)
        i32 = dict(dtype=torch.int32, device=gpu)
        return ((q, caches[0], caches[1], table.to(gpu), torch.full((B,), blocks * BS - 3, device=gpu),
                 torch.tensor([0, B], **i32), torch.tensor([common], **i32)),
                dict(q_start_loc=torch.arange(0, B * rows + 1, rows, **i32), max_q_len=rows))

    batches = [batch(24, 60, 9, 2), batch(5, 100, 40, 7)]
    alone = [attn.forward_shared(*args, **kw) for args, kw in batches]
    streams = [torch.cuda.Stream(gpu) for _ in batches]
    contexts = [kyro_amd.Context(0) for _ in batches]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, (args, kw) in enumerate(batches):
            with torch.cuda.stream(streams[i]):
                outs[i].append(attn.forward_shared_async(*args, context=contexts[i], **kw))
    torch.cuda.synchronize()
    for c in contexts:
        c.sync()
    for i in range(2):
        assert all(torch.equal(x, alone[i]) for x in outs[i])


@pytest.mark.parametrize("B", [6, 400])
def test_a_group_whose_first_sequence_is_left_out(gpu, B):
    """As kyro_tables_extend leaves an entry that the pool had no room for, or padding: no context, no blocks. The others
    read the common tokens all the same."""
    gen = torch.Generator().manual_seed(B)
    attn = PagedAttention(BS, H, D, HKV)
    common, own = 20, 3
    table = torch.randperm(B * (common + own), generator=gen).view(B, -1) + 1
    table[:, :common] = table[1, :common]
    lens = torch.full((B,), (common + own) * BS - 5)
    table[0], lens[0] = 0, 0
    caches = torch.randn((2, B * (common + own) + 1, HKV, BS, D), generator=gen).to(torch.bfloat16).to(gpu)
    q = torch.randn((B, H, D), generator=gen).to(torch.bfloat16).to(gpu)
    groups = [torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([0, B], [common])]
    args = q, caches[0], caches[1], table.to(gpu), lens.to(gpu)
    got = attn.forward_shared(*args, *groups)
    q, k, v = (x.float() for x in args[:3])
    exact, size = attn.forward(q, k, v, *args[3:]), attn.forward(q, k, v.abs(), *args[3:])
    # A weight is rounded once, by at most 2^-8 of it; sums in 32 bits, here and in `exact`, add less than 2^-11 of their
    # terms' size.
    assert ((got - exact).abs() <= (2.0 ** -8 + 2.0 ** -11) * size).all()
    assert not got[0].any() and exact[1:].any()
