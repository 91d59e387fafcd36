"""Accumulated attention weights (CacheEviction.accumulate) and eviction (CacheEviction.evict) against plain
implementations in 64 bits, at the sizes, masks and states where they can go wrong."""
import numpy as np
import pytest
import torch

import kyro_amd

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def caches(gpu, B, ctx, bs, hkv, D, dtype, seed=0, width=None, n=2):
    g = torch.Generator().manual_seed(seed)
    width = max(1, -(-int(max(ctx)) // bs)) if width is None else width
    nb = B * width + 2
    table = torch.randperm(nb, generator=g)[: B * width].view(B, width).to(gpu)
    return [torch.randn(nb, hkv, bs, D, generator=g).to(dtype).to(gpu) for _ in range(n)], table, g


# ------------------------------------------------------------------------------------ weights

def case(gpu, *, rows, old, H=8, hkv=2, D=64, bs=16, dtype=BF16, seed=0, width=None, extra_rows=0, sharp=1.5,
         state_rows=None, num_state=None, max_tokens=None):
    rows, old = list(rows), list(old)
    B, ctx = len(rows), [o + r for o, r in zip(old, rows)]
    (kc,), table, g = caches(gpu, B, ctx, bs, hkv, D, dtype, seed, width, 1)
    total = sum(rows) + extra_rows
    max_tokens = max_tokens or table.shape[1] * bs
    num_state = num_state or B
    c = dict(query=(torch.randn(total, H, D, generator=g) * sharp).to(dtype).to(gpu), key_cache=kc, block_table=table,
             context_lens=torch.tensor(ctx, device=gpu),
             weights=torch.rand(num_state, hkv, max_tokens, generator=g).to(gpu),
             positions=torch.randint(0, 99, (num_state, hkv, max_tokens), generator=g, dtype=torch.int32).to(gpu),
             q_start_loc=torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device=gpu))
    if state_rows is not None:
        c["state_rows"] = torch.tensor(state_rows, dtype=torch.int32, device=gpu)
    return c


def plain_weights(c, causal=True, scale=None):
    """(weights, positions, how far a right answer may be off) in 64 bits.

    A score is off by at most D roundings of the partial sums of |q k| plus its own, its scaling and the
    subtraction; softmax turns twice that (the score's and the row's log sum) into a relative error. The row's
    sum adds at most 1024 / 64 tiles x 4 in a lane, 6 merges of lanes and waves and 16 and more of chunks: 128
    steps cover it with the exponentials' own. Then one step per row added, and one for the old weight."""
    q, hkv = c["query"].double(), c["key_cache"].shape[1]
    H, D, bs = q.shape[1], q.shape[2], c["key_cache"].shape[2]
    scale = D ** -0.5 if scale is None else scale
    w, pos = c["weights"].double().clone(), c["positions"].clone()
    tol = torch.zeros_like(w)
    starts, ctx = c["q_start_loc"].tolist(), c["context_lens"].tolist()
    states = c["state_rows"].tolist() if c.get("state_rows") is not None else range(len(ctx))
    for b, (n_ctx, st) in enumerate(zip(ctx, states)):
        n = starts[b + 1] - starts[b]
        if n == 0:
            continue
        tok = torch.arange(n_ctx, device=q.device)
        if n_ctx == 0:
            continue
        last = n_ctx - n + torch.arange(n, device=q.device) if causal else torch.full((n,), n_ctx - 1, device=q.device)
        for h in range(hkv):
            k = c["key_cache"][c["block_table"][b], h].reshape(-1, D)[:n_ctx].double()
            new, err = torch.zeros(n_ctx, dtype=torch.float64, device=q.device), torch.zeros(n_ctx, dtype=torch.float64, device=q.device)
            for g in range(h * (H // hkv), (h + 1) * (H // hkv)):
                x = q[starts[b]:starts[b + 1], g]
                s = (x @ k.T * scale).masked_fill(tok > last[:, None], -float("inf"))
                size = ((x.abs() @ k.abs().T) * abs(scale)).amax(1)
                p = torch.softmax(s, -1).nan_to_num()  # a row that sees nothing adds nothing
                new += p.sum(0)
                err += (p * (2 * (D + 4) * size + 128 + n * (H // hkv))[:, None]).sum(0) * U
            old = max(0, n_ctx - n)
            w[st, h, :old] += new[:old]
            w[st, h, old:n_ctx] = new[old:]
            tol[st, h, :n_ctx] = err + 2 * U * w[st, h, :n_ctx].abs() + 1e-37
            at = c["row_positions"][starts[b]:starts[b + 1]][old - (n_ctx - n):] if c.get("row_positions") is not None else tok[old:]
            pos[st, h, old:n_ctx] = at.int()
    return w, pos, tol


def check_weights(c, **more):
    want, pos, tol = plain_weights(c, **{k: v for k, v in more.items() if k in ("causal", "scale")})
    ev = kyro_amd.CacheEviction(c["key_cache"].shape[2], c["query"].shape[1], c["query"].shape[2], c["key_cache"].shape[1])
    before = c["weights"].clone()
    out = ev.accumulate(**c, **more)
    off = (out.double() - want).abs() - tol
    assert not off.isnan().any() and (off <= 0).all(), f"{off.max():.3g} past the bound"
    assert torch.equal(c["positions"], pos)
    if more.get("out") is not None:
        assert torch.equal(c["weights"], before)
    return out


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [8, 40, 64, 72, 80, 96, 112, 128, 160, 200, 256])
@pytest.mark.parametrize("bs", [16, 5])
def test_head_dims_and_blocks(gpu, dtype, D, bs):
    check_weights(case(gpu, rows=[1, 5, 0, 3], old=[0, 70, 9, 300], D=D, bs=bs, dtype=dtype, seed=D + bs))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H,hkv", [(1, 1), (8, 8), (7, 1), (32, 8), (64, 2), (40, 8)])
@pytest.mark.parametrize("rows", [(1, 1, 1), (9, 1, 4), (40, 33, 64)])
def test_groups_and_rows(gpu, dtype, H, hkv, rows):
    check_weights(case(gpu, rows=rows, old=[0, 15, 200], H=H, hkv=hkv, dtype=dtype, seed=H))


@pytest.mark.parametrize("ctx", [1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 1000, 1024, 1025, 4097])
def test_one_row_of_every_length(gpu, ctx):
    check_weights(case(gpu, rows=[1], old=[ctx - 1], seed=ctx))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,old", [((300, 0, 17), (0, 50, 1000)), ((130,), (2000,)), ((512, 511), (0, 1)),
                                      ((1, 257, 64, 2), (3000, 0, 64, 128))])
def test_prompts(gpu, dtype, rows, old):
    check_weights(case(gpu, rows=rows, old=old, D=128, H=8, hkv=2, dtype=dtype, seed=len(rows)))


def test_many_sequences_and_wide_tables(gpu):
    """More sequences than a strip of the walk holds, tables far wider than the contexts."""
    g = np.random.default_rng(0)
    rows = g.integers(0, 4, 150)
    check_weights(case(gpu, rows=rows, old=g.integers(0, 90, 150), H=4, hkv=2, D=32, width=64, seed=1))
    check_weights(case(gpu, rows=[1, 2], old=[1000, 5], H=4, hkv=2, D=32, width=5000, seed=2))


def test_long_context(gpu):
    check_weights(case(gpu, rows=[1, 3], old=[70001, 33], H=4, hkv=1, D=64, seed=3))


def test_more_scores_than_are_kept(gpu):
    """16 rows of 64 kv heads at 70000 tokens: 286 MB of scores, of which 256 MiB are kept between the passes."""
    check_weights(case(gpu, rows=[1], old=[69999], H=1024, hkv=64, D=8, seed=5))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prompts_beside_decode_steps(gpu, dtype):
    """Sequences of many rows and of few in one call, each with its own kernels."""
    check_weights(case(gpu, rows=[1, 200, 9, 0, 1, 65], old=[900, 40, 333, 7, 0, 64], D=128, H=8, hkv=2, dtype=dtype, seed=6))


def test_many_rows_over_few_tokens(gpu):
    """The rows of a sum split into parts, joined in their order."""
    check_weights(case(gpu, rows=[700], old=[3], D=128, H=8, hkv=1, seed=7))
    check_weights(case(gpu, rows=[900, 2], old=[0, 100], D=80, H=4, hkv=1, dtype=F32, seed=8))


def test_not_causal_scale_out_and_row_positions(gpu):
    c = case(gpu, rows=[4, 1, 30], old=[10, 0, 99], seed=4)
    c["row_positions"] = torch.randint(0, 5000, (35,), device=gpu)
    out = torch.full_like(c["weights"], 7.0)
    want_rest = c["weights"].clone()
    got = check_weights({**c, "weights": c["weights"]}, causal=False, scale=0.3,
                        out=torch.where(torch.zeros_like(out, dtype=torch.bool), out, want_rest))
    assert got.data_ptr() != c["weights"].data_ptr()


def test_entries_behind_the_tokens_and_other_rows_stay(gpu):
    c = case(gpu, rows=[2, 3], old=[5, 40], state_rows=[4, 1], num_state=6, max_tokens=100, width=9, extra_rows=3)
    check_weights(c)  # compares the whole state


@pytest.mark.parametrize("rows", [(1, 1, 4, 6), (1, 130, 4, 300)])
def test_padded_batches_and_contexts_shorter_than_their_rows(gpu, rows):
    """Empty contexts with a row each, as a padded batch has them, and rows that see no token."""
    c = case(gpu, rows=rows, old=[0, 30, 60, 0], seed=9)
    c["context_lens"] = torch.tensor([0, 30 + rows[1], 2, rows[3] - 3], device=gpu)
    c["row_positions"] = torch.randint(0, 5000, (sum(rows),), device=gpu)
    check_weights(c)
    assert (c["weights"][0] <= 1).all()


def test_unseen_numbers_reach_nothing_from_prompts(gpu):
    """The same for the kernels of many rows: a row of NaN reaches the tokens it sees and no others."""
    c = case(gpu, rows=[200, 90], old=[50, 7], D=128, H=2, hkv=2, extra_rows=5)
    c["query"][290:] = float("nan")
    for b, n in enumerate([250, 97]):
        t = torch.arange(n, 16 * c["block_table"].shape[1], device=gpu)
        c["key_cache"][c["block_table"][b, t // 16], :, t % 16] = float("nan")
    check_weights(c)
    c["query"][250, 1] = float("nan")  # the second sequence's row 50: sees tokens 0 to 57
    out = kyro_amd.CacheEviction(16, 2, 128, 2).accumulate(**c)
    assert out[1, 1, :58].isnan().all() and out[1, 1, 58:].isfinite().all()
    assert out[0].isfinite().all() and out[1, 0].isfinite().all()


@pytest.mark.parametrize("n,hkv", [(3, 2), (3, 8), (7, 2), (7, 8), (20, 2), (100, 2), (70, 8)])
def test_a_score_of_minus_infinity_is_a_weight_of_zero(gpu, n, hkv):
    """Every row scores one token -infinity. The zeros that fill up the operands of the products would make it
    NaN (0 * infinity): they are no rows."""
    c = case(gpu, rows=[n], old=[50], H=8, hkv=hkv, D=64, seed=n)
    c["query"][..., 0] = -1
    c["key_cache"][c["block_table"][0, 0], :, 5, 0] = float("inf")
    c["weights"].zero_()
    out = kyro_amd.CacheEviction(16, 8, 64, hkv).accumulate(**c)
    assert (out[0, :, 5] == 0).all() and out.isfinite().all()
    # each row of a kv head's 8 / hkv heads shares out a weight of 1, within 2^-24 x (the bound of plain_weights) of it
    assert ((out[0].double().sum(-1) / (n * 8 // hkv) - 1).abs() < 1e-4).all()


def test_one_row_without_q_start(gpu):
    c = case(gpu, rows=[1, 1, 1], old=[5, 0, 300])
    d = {k: v.clone() for k, v in c.items() if k != "q_start_loc"}
    want = check_weights(c)
    got = kyro_amd.CacheEviction(16, 8, 64, 2).accumulate(**d)
    assert torch.equal(got, want)


def test_same_result_every_time(gpu):
    c = case(gpu, rows=[8] * 9, old=range(100, 1000, 100), H=32, hkv=8, D=128)
    outs = [kyro_amd.CacheEviction(16, 32, 128, 8).accumulate(**{**c, "out": torch.zeros_like(c["weights"])}) for _ in range(3)]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_unseen_numbers_reach_nothing(gpu):
    """NaN and infinities behind a sequence's last token, in its last page, in other blocks and in rows of no
    sequence; and a NaN that is seen reaches exactly the tokens its row sees."""
    c = case(gpu, rows=[2, 4], old=[9, 18], extra_rows=2, width=3, H=2, hkv=2)
    used = torch.zeros(c["key_cache"].shape[0], 16, dtype=torch.bool)
    for b, n in enumerate([11, 22]):
        for t in range(n):
            used[c["block_table"][b, t // 16], t % 16] = True
    bad = ~used.to(gpu)[:, None, :, None].expand_as(c["key_cache"])
    c["key_cache"][bad] = torch.where(torch.rand(int(bad.sum()), device=gpu) < 0.5, float("nan"), float("inf")).to(BF16)
    c["query"][6:] = float("nan")
    check_weights(c)
    c["query"][3, 0] = float("nan")  # the second sequence's row 1, head 0: sees tokens 0 to 19
    out = kyro_amd.CacheEviction(16, 2, 64, 2).accumulate(**c)
    assert out[1, 0, :20].isnan().all() and out[1, 0, 20:].isfinite().all()
    assert out[0].isfinite().all() and out[1, 1].isfinite().all()


def test_scores_of_great_size(gpu):
    """One token takes all: no overflow in 2^x, no row lost."""
    c = case(gpu, rows=[3], old=[60], H=2, hkv=2, dtype=F32, sharp=300.0)
    out = kyro_amd.CacheEviction(16, 2, 64, 2).accumulate(**{**c, "out": torch.zeros_like(c["weights"])})
    gained = (out - c["weights"])[0, :, :60].double().sum(-1) + out[0, :, 60:63].double().sum(-1)
    assert (gained - 3).abs().max() < 1e-3 and out.isfinite().all()


def test_bad_sequences_are_reported_and_left_out(gpu):
    for what in ("context", "cap", "layout", "row", "twice"):
        c = case(gpu, rows=[2, 3, 1, 5], old=[20, 5, 7, 9], state_rows=[0, 1, 2, 3], max_tokens=40, width=4)
        bad = [1]
        if what == "context":
            c["context_lens"][1] = -1
        elif what == "cap":
            c["context_lens"][1] = 41
        elif what == "layout":
            c["q_start_loc"][4] = 99
            bad = [3]
        elif what == "row":
            c["state_rows"][1] = 4
        else:
            c["state_rows"][3] = 1
            bad = [1, 3]
        good = [b for b in range(4) if b not in bad]
        if what == "layout":
            alone = dict(c, q_start_loc=torch.tensor([0, 2, 5, 6, 6], dtype=torch.int32, device=gpu))
        else:
            alone = dict(c)
        before = c["weights"].clone(), c["positions"].clone()
        ev = kyro_amd.CacheEviction(16, 8, 64, 2)
        match = {"context": "context length", "cap": "context length", "layout": "q_start_loc", "row": "state row", "twice": "state row"}
        with pytest.raises(kyro_amd.KyroError, match=match[what]):
            ev.accumulate(**c, max_q_len=5)
        for b in bad:
            assert torch.equal(c["weights"][b], before[0][b]) and torch.equal(c["positions"][b], before[1][b]), what
        want = plain_weights({**alone, "weights": before[0], "positions": before[1],
                              "context_lens": torch.where(torch.tensor([b in bad for b in range(4)], device=gpu), 23, c["context_lens"]),
                              "state_rows": torch.arange(4, dtype=torch.int32, device=gpu)})
        for b in good:
            assert ((c["weights"][b].double() - want[0][b]).abs() <= want[2][b]).all(), what
        kyro_amd.sync()


def test_bad_block_is_reported_and_not_seen(gpu):
    c = case(gpu, rows=[2], old=[40])
    c["block_table"][0, 1] = -5
    with pytest.raises(kyro_amd.KyroError, match="block_table"):
        kyro_amd.CacheEviction(16, 8, 64, 2).accumulate(**{**c, "out": torch.zeros_like(c["weights"])})
    out = torch.zeros_like(c["weights"])
    with pytest.raises(kyro_amd.KyroError):
        kyro_amd.CacheEviction(16, 8, 64, 2).accumulate(**{**c, "weights": torch.zeros_like(out), "out": out})
    assert (out[0, :, 16:32] == 0).all()
    assert ((out[0].double().sum(-1) - 2 * 4).abs() < 1e-4).all()  # two rows of four heads share their whole weight


def test_weights_refused_tensors(gpu):
    c = case(gpu, rows=[2, 3], old=[5, 40])
    ev = kyro_amd.CacheEviction(16, 8, 64, 2)

    def refused(error, **change):
        with pytest.raises(error):
            ev.accumulate(**{**c, **change})

    refused(TypeError, query=c["query"].half())
    refused(TypeError, key_cache=c["key_cache"].float())
    refused(ValueError, query=c["query"][:, :4])
    refused(ValueError, query=c["query"].transpose(0, 1))
    refused(ValueError, weights=c["weights"][..., :-1])
    refused(ValueError, positions=c["positions"][..., :-1].contiguous())
    refused(TypeError, positions=c["positions"].long())
    refused(TypeError, weights=c["weights"].double())
    refused(ValueError, out=c["weights"][:1])
    refused(ValueError, q_start_loc=c["q_start_loc"][:2])
    refused(ValueError, q_start_loc=None)
    refused(ValueError, row_positions=torch.zeros(3, dtype=torch.int64, device=gpu))
    refused(TypeError, state_rows=torch.zeros(2, dtype=torch.int64, device=gpu))
    refused(ValueError, block_table=c["block_table"][:1])
    refused(ValueError, weights=c["weights"][:1], positions=c["positions"][:1])
    check_weights(c)


# ------------------------------------------------------------------------------------ eviction

def ecase(gpu, ctx, *, hkv=2, D=64, bs=16, dtype=BF16, seed=0, width=None, max_tokens=None, kind="spread", again=0):
    (kc, vc), table, g = caches(gpu, len(ctx), ctx, bs, hkv, D, dtype, seed, width)
    max_tokens = max_tokens or table.shape[1] * bs
    shape = (len(ctx), hkv, max_tokens)
    w = torch.exp(3 * torch.randn(shape, generator=g))
    if kind == "ties":
        w = torch.randint(0, 3, shape, generator=g).float()
    elif kind == "equal":
        w = torch.ones(shape)
    elif kind == "odd":
        odd = torch.tensor([float("nan"), float("inf"), -float("inf"), -1.0, -0.0, 0.0, 1e-40, -1e-40, 3.0])
        w = odd[torch.randint(0, 9, shape, generator=g)]
    pos = torch.arange(max_tokens, dtype=torch.int32).expand(shape).clone()
    if again:
        pos += 500
        pos[..., :again] = torch.stack([torch.randperm(500, generator=g)[:again] for _ in range(shape[0] * hkv)]).view(*shape[:2], again)
    return dict(key_cache=kc, value_cache=vc, block_table=table, context_lens=torch.tensor(ctx, device=gpu),
                weights=w.to(gpu), positions=pos.to(gpu))


def plain_evict(c, budget, sink, recent, out=None):
    kc, vc = c["key_cache"].cpu().clone(), c["value_cache"].cpu().clone()
    w, pos, table, bs = c["weights"].cpu(), c["positions"].cpu().numpy(), c["block_table"].cpu().numpy(), c["key_cache"].shape[2]
    ow, op = (w.clone(), torch.from_numpy(pos.copy())) if out is None else (out[0].cpu().clone(), out[1].cpu().clone())
    lens = c["context_lens"].tolist()
    states = c["state_rows"].tolist() if c.get("state_rows") is not None else range(len(lens))
    for b, (n, st) in enumerate(zip(lens, states)):
        for h in range(w.shape[1]):
            x, p = w[st, h, :n].double().numpy().copy(), pos[st, h, :n].astype(np.int64)
            x[np.isnan(x)] = -np.inf
            keep = min(n, budget)
            source = np.arange(keep)
            if n > budget:
                safe = (p < sink) | (p > p.max() - recent)
                order = sorted(range(n), key=lambda t: (not safe[t], -x[t], t))[:budget]
                kept = np.zeros(n, bool)
                kept[order] = True
                source[~kept[:budget]] = budget + np.flatnonzero(kept[budget:])
            for t, s in enumerate(source):
                if t != s:
                    to, frm = (table[b, t // bs], h, t % bs), (table[b, s // bs], h, s % bs)
                    kc[to], vc[to] = kc[frm], vc[frm]
            ow[st, h, :keep], op[st, h, :keep] = w[st, h][source], torch.from_numpy(pos[st, h][source])
    return kc, vc, ow, op, [min(n, budget) for n in lens]


def same(a, b):
    a, b = a.cpu(), b.cpu()
    kind = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.view(kind), b.view(kind))  # bit for bit, NaN too


def check_evict(c, budget, sink=4, recent=0, out=None):
    want = plain_evict(c, budget, sink, recent, out)
    ev = kyro_amd.CacheEviction(c["key_cache"].shape[2], c["key_cache"].shape[1], c["key_cache"].shape[3], c["key_cache"].shape[1])
    before = c["weights"].clone(), c["positions"].clone()
    lens = ev.evict(**c, budget=budget, sink=sink, recent=recent, out=out)
    got = out or (c["weights"], c["positions"])
    assert lens.tolist() == want[4]
    for name, x, y in zip(("key cache", "value cache", "weights", "positions"), (c["key_cache"], c["value_cache"], *got), want):
        assert same(x, y), name
    if out is not None:
        assert same(c["weights"], before[0]) and same(c["positions"], before[1])
    return lens


@pytest.mark.parametrize("dtype,D,bs,hkv", [(BF16, 128, 16, 8), (F32, 80, 32, 3), (BF16, 8, 5, 1), (F32, 256, 16, 2),
                                            (BF16, 72, 1, 2), (F32, 8, 64, 1)])
@pytest.mark.parametrize("budget,sink,recent", [(100, 4, 16), (1, 0, 0), (1, 1, 0), (257, 0, 257), (64, 64, 0), (300, 10, 50)])
def test_evict_sizes(gpu, dtype, D, bs, hkv, budget, sink, recent):
    check_evict(ecase(gpu, [0, 1, 99, 100, 101, 300, 777], hkv=hkv, D=D, bs=bs, dtype=dtype, seed=budget), budget, sink, recent)


@pytest.mark.parametrize("kind", ["ties", "equal", "odd"])
@pytest.mark.parametrize("budget", [33, 500, 1023])
def test_evict_ties_and_odd_weights(gpu, kind, budget):
    check_evict(ecase(gpu, [1024, 40, 600], kind=kind, seed=budget), budget, 2, 5)


@pytest.mark.parametrize("ctx,budget", [([12288], 5000), ([12289], 5000), ([30000, 20], 29000), ([70001], 64)])
def test_evict_around_the_keys_that_fit(gpu, ctx, budget):
    """Keys in LDS up to 12288 tokens, read again for each pass beyond."""
    check_evict(ecase(gpu, ctx, hkv=1, D=8, seed=budget), budget, 4, 30)


def test_evict_moved_tokens_again(gpu):
    """Protection goes by position, wherever earlier evictions have put a token; twice in a row."""
    c = ecase(gpu, [300, 333], again=200)
    check_evict(c, 200, 4, 120)
    c["context_lens"] = torch.tensor([150, 200], device=gpu)
    check_evict(c, 150, 4, 60)


def test_evict_out_of_place_can_be_repeated(gpu):
    c = ecase(gpu, [300, 50, 128], kind="ties")
    out = torch.full_like(c["weights"], -7.0), torch.full_like(c["positions"], -7)
    check_evict(c, 128, 4, 16, out=out)
    k, v = c["key_cache"].clone(), c["value_cache"].clone()
    check_evict(c, 128, 4, 16, out=out)
    assert same(k, c["key_cache"]) and same(v, c["value_cache"])


def test_evict_state_rows_and_wide_state(gpu):
    c = ecase(gpu, [300, 222], width=40, max_tokens=310)
    for n in ("weights", "positions"):
        c[n] = torch.cat([c[n], c[n].flip(0), c[n]])
    c["state_rows"] = torch.tensor([5, 2], dtype=torch.int32, device=gpu)
    check_evict(c, 100, 4, 30)


def test_evict_bad_sequences_are_left(gpu):
    for what in ("context", "block", "row", "twice"):
        c = ecase(gpu, [200, 220, 240])
        c["state_rows"] = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
        bad = [1]
        if what == "context":
            c["context_lens"][1] = -3
        elif what == "block":
            c["block_table"][1, 13] = c["key_cache"].shape[0]  # its last page
        elif what == "row":
            c["state_rows"][1] = -1
        else:
            c["state_rows"][1] = 0
            bad = [0, 1]
        good = [b for b in range(3) if b not in bad]
        part = {k: (v[good] if k in ("block_table", "context_lens", "state_rows") else v) for k, v in c.items()}
        want = plain_evict(part, 100, 4, 10)
        lens0 = c["context_lens"].tolist()
        match = {"context": "context length", "block": "block_table", "row": "state row", "twice": "state row"}[what]
        ev = kyro_amd.CacheEviction(16, 2, 64, 2)
        lens = ev.evict_async(**c, budget=100, sink=4, recent=10)
        with pytest.raises(kyro_amd.KyroError, match=match):
            kyro_amd.sync()
        assert lens.tolist() == [100 if b in good else lens0[b] for b in range(3)]
        for x, y in zip((c["key_cache"], c["value_cache"], c["weights"], c["positions"]), want):
            assert same(x, y), what


def test_evict_refused_tensors(gpu):
    c = ecase(gpu, [200, 220])
    ev = kyro_amd.CacheEviction(16, 2, 64, 2)

    def refused(error, **change):
        with pytest.raises(error):
            ev.evict(**{**dict(c, budget=100), **change})

    refused(kyro_amd.KyroError, budget=0)
    refused(kyro_amd.KyroError, sink=60, recent=41)
    refused(TypeError, key_cache=c["key_cache"].half())
    refused(TypeError, value_cache=c["value_cache"].float())
    refused(ValueError, value_cache=c["value_cache"][:-1])
    refused(ValueError, key_cache=c["key_cache"].transpose(1, 2))
    refused(TypeError, positions=c["positions"].long())
    refused(ValueError, context_lens=c["context_lens"][:1])
    refused(TypeError, state_rows=torch.zeros(2, device=gpu))
    refused(ValueError, out=(c["weights"][:1], c["positions"]))
    refused(kyro_amd.KyroError, out=(c["positions"].view(F32), c["positions"]))
    check_evict(c, 100)


def test_evict_cache_past_32_bits(gpu):
    nb = 2 ** 32 // (2 * 16 * 128) + 40
    c = ecase(gpu, [300, 100], D=128)
    big = [torch.empty((nb, 2, 16, 128), dtype=BF16, device=gpu) for _ in range(2)]
    shift = nb - c["key_cache"].shape[0]
    for x, y in zip(big, (c["key_cache"], c["value_cache"])):
        x[shift:] = y
        x[:64] = 3
    far = dict(c, key_cache=big[0], value_cache=big[1], block_table=c["block_table"] + shift, weights=c["weights"].clone(),
               positions=c["positions"].clone())
    kyro_amd.CacheEviction(16, 2, 128, 2).evict(**far, budget=90, recent=10)
    check_evict(c, 90, 4, 10)
    assert same(big[0][shift:], c["key_cache"]) and same(big[1][shift:], c["value_cache"]) and (big[0][:64] == 3).all()


# ------------------------------------------------------------------------------------ together

def test_graphs_replay_as_eager(gpu):
    """Both calls captured, replayed with other inputs and eager work between: the eager results."""
    ev = kyro_amd.CacheEviction(16, 8, 64, 2)
    c = case(gpu, rows=[3, 1], old=[200, 90])
    (_, vc), _, _ = caches(gpu, 2, [203, 91], 16, 2, 64, BF16)
    out = torch.zeros_like(c["weights"]), torch.zeros_like(c["positions"])
    w2 = torch.zeros_like(c["weights"])
    k0, v0 = c["key_cache"].clone(), vc.clone()

    def work(c, w2, out, vc):
        ev.accumulate_async(**c, max_q_len=3, out=w2)
        return ev.evict_async(c["key_cache"], vc, c["block_table"], c["context_lens"], w2, c["positions"], budget=80, recent=8,
                              out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(c, w2, out, vc)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            lens = work(c, w2, out, vc)
    torch.cuda.current_stream().wait_stream(side)
    for turn in range(4):
        c["query"].copy_(torch.randn(c["query"].shape, device=gpu))
        c["weights"].uniform_()
        c["key_cache"].copy_(k0), vc.copy_(v0)
        graph.replay()
        torch.cuda.synchronize()
        d = dict(c, key_cache=k0.clone(), positions=c["positions"].clone())
        e_out, e_w2, e_vc = (torch.zeros_like(out[0]), torch.zeros_like(out[1])), torch.zeros_like(w2), v0.clone()
        e_lens = work(d, e_w2, e_out, e_vc)
        kyro_amd.sync()
        for x, y in ((w2, e_w2), (out[0], e_out[0]), (out[1], e_out[1]), (lens, e_lens), (c["key_cache"], d["key_cache"]), (vc, e_vc)):
            assert torch.equal(x, y)


def test_a_run_of_steps_under_a_budget(gpu):
    """A sequence as a serving program runs it: rows rotated and appended by position, attended, weighed, and the
    cache cut to its budget whenever it is over, against the same steps with the kept tokens in lists, in 64 bits.
    The block manager's request shares its prompt with the prefix cache at first."""
    H, hkv, D, bs, budget, steps = 4, 2, 32, 4, 24, 30
    g = torch.Generator().manual_seed(1)
    bm = kyro_amd.BlockManager(bs, 64)
    prompt = list(range(10))
    bm.allocate_with_prefix(1, prompt)
    bm.free(1)
    bm.allocate_with_prefix(2, prompt)
    kc, vc = (torch.zeros(64, hkv, bs, D, device=gpu) for _ in range(2))
    kyro_amd.copy_blocks(kc, vc, bm.take_copies())
    shared = bm.block_table[2][0]
    kv, ev = kyro_amd.PagedKVCache(bs, hkv, D), kyro_amd.CacheEviction(bs, H, D, hkv)
    attn = kyro_amd.PagedAttention(bs, H, D, hkv)
    weights, positions = ev.new_state(1, 64, gpu)
    cos, sin = kyro_amd.rope_tables(200, D, device=gpu)
    table, ctx = torch.zeros(1, 16, dtype=torch.int64, device=gpu), torch.zeros(1, dtype=torch.int64, device=gpu)
    model = [[] for _ in range(hkv)]  # per kv head, by slot: (position, key, value, weight)
    cut = 0
    for step in range(steps):
        n = 10 if step == 0 else 1 + step % 3
        first = 0 if step == 0 else pos_next
        pos_next = first + n
        if step:
            assert bm.append_slots(2, n)
        bm.write_tables([2], table, ctx)
        q, k, v = (torch.randn(n, heads, D, generator=g).to(gpu) for heads in (H, hkv, hkv))
        pos = torch.arange(first, first + n, device=gpu)
        starts = torch.tensor([0, n], dtype=torch.int32, device=gpu)
        qr = kv.append_qkv(q, k, v, kc, vc, table, ctx, cos=cos, sin=sin, positions=pos, q_start_loc=starts, norm_eps=1e-6)
        got = attn.forward(qr, kc, vc, table, ctx, q_start_loc=starts)
        ev.accumulate(qr, kc, table, ctx, weights, positions, q_start_loc=starts, row_positions=pos)
        ang = pos.double().cpu()[:, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)

        def turn(x):
            x = x.double().cpu()
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
            a, b = x[..., : D // 2], x[..., D // 2:]
            c, s = ang.cos()[:, None], ang.sin()[:, None]
            return torch.cat((a * c - b * s, b * c + a * s), -1)

        q64, k64, v64 = turn(q), turn(k), v.double().cpu()
        for h in range(hkv):
            held = len(model[h])
            model[h] += [[first + j, k64[j, h], v64[j, h], 0.0] for j in range(n)]
            K, V = (torch.stack([e[i] for e in model[h]]) for i in (1, 2))
            for gq in range(2 * h, 2 * h + 2):
                s = q64[:, gq] @ K.T / D ** 0.5
                s[torch.arange(held + n) > held + torch.arange(n)[:, None]] = -float("inf")
                p = torch.softmax(s, -1)
                # f32 attention over up to 30 tokens: the library's own bound
                assert (got[:, gq].double().cpu() - p @ V).abs().max() < 1e-3
                for e, x in zip(model[h], p.sum(0).tolist()):
                    e[3] += x
            mine = weights[0, h, : len(model[h])].double().cpu()
            # at most 60 rows have been added, each within the scores' error: 2 (32 + 4) 2^-24 max |s|, |s| < 12
            assert (mine - torch.tensor([e[3] for e in model[h]], dtype=torch.float64)).abs().max() < 1e-3
            assert positions[0, h, : len(model[h])].tolist() == [e[0] for e in model[h]]
        if int(ctx) > budget:
            cut += 1
            assert bm.make_private(2)
            kyro_amd.copy_blocks(kc, vc, bm.take_copies())
            before = kc[shared].clone()
            bm.write_tables([2], table, ctx)
            lens = ev.evict(kc, vc, table, ctx, weights, positions, budget=budget, sink=2, recent=6)
            bm.truncate(2, int(lens))
            bm.check()
            assert torch.equal(kc[shared], before)  # the prefix cache's block is as it was
            for h in range(hkv):
                # What stayed is the library's to say where weights nearly tie; that it is a right choice is not.
                stay = set(positions[0, h, :budget].tolist())
                newest = max(e[0] for e in model[h])
                gone = [e for e in model[h] if e[0] not in stay]
                kept = [e for e in model[h] if e[0] in stay]
                assert len(kept) == budget and all(2 <= e[0] <= newest - 6 for e in gone)
                free = [e[3] for e in kept if 2 <= e[0] <= newest - 6]
                assert not gone or not free or max(e[3] for e in gone) <= min(free) + 2e-3
                where = {e[0]: e for e in kept}
                model[h] = [where[p] for p in positions[0, h, :budget].tolist()]
    assert cut >= 10
    bm.free(2)
    bm.check()


# ------------------------------------------------------------------------------------ weights that go elsewhere

@pytest.mark.parametrize("what,rows,old,more", [
    # 8 / 2 heads: 4 rows of a kv head for each of a sequence.
    ("scores kept", (1, 0, 4, 0), (70, 33, 300, 0), {}),
    ("scores computed again", (1, 0, 9, 0), (70, 33, 300, 16), {}),
    ("f32, scores computed again", (0, 12, 0), (1, 900, 64), dict(dtype=F32)),
    ("rows through LDS", (100, 0, 100), (70, 33, 300), {}),
    ("both forms", (100, 0, 1, 0, 7), (70, 333, 300, 5, 0), {}),
    ("rows in parts", (0, 700, 0), (3, 3, 3), dict(D=128, hkv=1)),
    ("f32 rows in parts", (400, 0), (3, 90), dict(D=80, hkv=1, dtype=F32)),
    ("a long sequence without rows", (0, 1), (5000, 20), {}),
    ("no rows at all", (0, 0, 0), (17, 0, 400), {})])
def test_weights_go_elsewhere_whole(gpu, what, rows, old, more):
    """Entries of every sequence's tokens, also of one without rows, come from `weights`; what is behind them
    in `out`, and state rows of no sequence, stay as they are."""
    n = len(rows)
    c = case(gpu, rows=rows, old=old, state_rows=[(2 * b + 1) % (2 * n + 1) for b in range(n)], num_state=2 * n + 1,
             width=-(-(max(old) + max(rows)) // 16) + 3, seed=n, **more)
    before, pos = c["weights"].clone(), c["positions"].clone()
    want, want_pos, tol = plain_weights(c)
    out = torch.full_like(before, 7.0)
    kyro_amd.CacheEviction(16, 8, c["query"].shape[2], c["key_cache"].shape[1]).accumulate(**c, out=out)
    held = torch.zeros_like(out, dtype=torch.bool)
    for b in range(n):
        held[(2 * b + 1) % (2 * n + 1), :, :old[b] + rows[b]] = True
    assert (out[~held] == 7).all() and torch.equal(c["weights"], before) and torch.equal(c["positions"], want_pos)
    assert ((out.double() - want).abs() <= tol)[held].all()
    for b in range(n):
        if rows[b] == 0:
            r = (2 * b + 1) % (2 * n + 1)
            assert torch.equal(out[r, :, :old[b]], before[r, :, :old[b]]) and torch.equal(c["positions"][r], pos[r])


def test_bad_sequences_without_rows_are_reported_and_left_out(gpu):
    for what, match in (("context", "context length"), ("cap", "context length"), ("row", "state row"), ("twice", "state row")):
        for rows in ((0, 2, 0), (0, 0, 0)):
            c = case(gpu, rows=rows, old=[20, 7, 9], state_rows=[0, 1, 2], max_tokens=40, width=4)
            if what in ("context", "cap"):
                c["context_lens"][0] = -1 if what == "context" else 41
            else:
                c["state_rows"][0] = 3 if what == "row" else 2
            out = torch.full_like(c["weights"], 7.0)
            with pytest.raises(kyro_amd.KyroError, match=match):
                kyro_amd.CacheEviction(16, 8, 64, 2).accumulate(**c, max_q_len=2, out=out)
            assert (out[0] == 7).all()
            assert (out[2] == 7).all() if what == "twice" else torch.equal(out[2, :, :9], c["weights"][2, :, :9])
            kyro_amd.sync()


def test_padded_batch_without_rows_needs_no_state_row(gpu):
    """Empty sequences of no rows have nothing to take along: their state rows are not looked at."""
    c = case(gpu, rows=[3, 0, 0], old=[20, 0, 0], state_rows=[1, -1, -1], num_state=2)
    out = torch.full_like(c["weights"], 7.0)
    kyro_amd.CacheEviction(16, 8, 64, 2).accumulate(**c, out=out)
    assert (out[0] == 7).all() and (out[1, :, :23] != 7).all()


def test_evict_with_only_the_front_private(gpu):
    """A shared prompt of 50 tokens cut to 13: four of its 13 blocks are copied, the others stay shared and are
    only read, and what the other holder reads is as it was."""
    bm = kyro_amd.BlockManager(4, 60)
    prompt = list(range(50))
    bm.allocate_with_prefix(1, prompt)
    bm.free(1)
    for rid in (2, 3):
        assert bm.allocate_with_prefix(rid, prompt)[1] == 50
    c = ecase(gpu, [50], bs=4, seed=3)
    g = torch.Generator().manual_seed(8)
    for name in ("key_cache", "value_cache"):
        c[name] = torch.randn(60, 2, 4, 64, generator=g).to(BF16).to(gpu)
    kyro_amd.copy_blocks(c["key_cache"], c["value_cache"], bm.take_copies())
    assert bm.make_private(2, 13)
    copies = bm.take_copies()
    assert len(copies) == 4
    kyro_amd.copy_blocks(c["key_cache"], c["value_cache"], copies)
    bm.write_tables([2], c["block_table"], c["context_lens"])
    other = bm.block_table[3]
    assert bm.block_table[2][4:12] == other[4:12]
    kyro_amd.sync()
    before = c["key_cache"][other].clone(), c["value_cache"][other].clone()
    lens = check_evict(c, 13, 2, 3)
    assert torch.equal(c["key_cache"][other], before[0]) and torch.equal(c["value_cache"][other], before[1])
    bm.truncate(2, int(lens))
    bm.check()


@pytest.mark.parametrize("n,hkv", [(3, 8), (3, 2), (7, 2), (9, 2), (100, 2), (70, 8)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_row_of_nan_gives_nan_where_it_scores_minus_infinity(gpu, n, hkv, dtype):
    """Token 5 scores -infinity and token 7 NaN with every row: the softmax of a row is NaN over all it sees, in
    every form of the kernels, and a row of numbers beside it is not."""
    c = case(gpu, rows=[n, n], old=[50, 50], H=8, hkv=hkv, D=64, dtype=dtype, seed=n)
    c["query"][..., 0] = -1
    for b in range(2):
        c["key_cache"][c["block_table"][b, 0], :, 5, 0] = float("inf")
    c["key_cache"][c["block_table"][1, 0], :, 7, 1] = float("nan")
    c["key_cache"][c["block_table"][1, (49 + n) // 16], :, (49 + n) % 16, 0] = float("inf")  # seen by the last row
    c["weights"].zero_()
    out = kyro_amd.CacheEviction(16, 8, 64, hkv).accumulate(**c)
    assert out[1, :, :50 + n].isnan().all() and out[0].isfinite().all() and (out[0, :, 5] == 0).all()


@pytest.mark.parametrize("n,hkv", [(3, 8), (3, 2), (9, 2), (100, 2)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_row_of_minus_infinities_adds_nothing(gpu, n, hkv, dtype):
    """As one that sees no token: in every form, and beside a sequence of numbers."""
    c = case(gpu, rows=[n, n], old=[150, 150], H=8, hkv=hkv, D=64, dtype=dtype, seed=n)
    c["query"][..., 0] = -1
    c["key_cache"][c["block_table"][1], ..., 0] = float("inf")
    before = c["weights"].clone()
    out = kyro_amd.CacheEviction(16, 8, 64, hkv).accumulate(**c)
    assert torch.equal(out[1, :, :150], before[1, :, :150]) and (out[1, :, 150:150 + n] == 0).all()
    # The other's rows share out a weight of 1 each, within 2^-24 x 4000 (plain_weights: 136 |q| |k| / 8 + 128 + 400);
    # adding it to up to 250 weights below 1 and gains rounds each by half a step of a number below 128, 2^-18.
    gain = out[0].double().sum(-1) - before[0, :, :150].double().sum(-1) - before[0, :, 150 + n:].double().sum(-1)
    assert ((gain / (n * 8 // hkv) - 1).abs() < 4000 * U + 250 * 2.0 ** -18 / (n * 8 // hkv)).all()


# ------------------------------------------------------------------------------------ every form of the kernels

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 72, 96, 112, 128, 160, 192, 200, 256])
def test_head_dims_of_many_rows(gpu, dtype, D):
    """Rows through LDS: each number of steps a product has, whole rows and padded ones, in parts of the rows and
    (with more tokens) without, beside sequences of few rows."""
    check_weights(case(gpu, rows=[75, 3, 0, 33], old=[130, 300, 9, 0], H=8, hkv=2, D=D, dtype=dtype, seed=D))
    check_weights(case(gpu, rows=[300], old=[77], H=4, hkv=1, D=D, dtype=dtype, seed=D + 1))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [32, 192])
@pytest.mark.parametrize("n", [1, 3, 8, 16])
def test_head_dims_of_few_rows(gpu, dtype, D, n):
    check_weights(case(gpu, rows=[n, 0, n], old=[90, 5, 400], H=8, hkv=2, D=D, dtype=dtype, seed=D + n))


def test_many_rows_that_are_not_split(gpu):
    """Runs of tokens enough for the CUs: the rows of a sum in one part, in place and elsewhere."""
    for dtype in (BF16, F32):
        c = case(gpu, rows=[70, 66], old=[20000, 17000], H=8, hkv=8, D=64, dtype=dtype, seed=2)
        out = torch.full_like(c["weights"], 7.0)
        kyro_amd.CacheEviction(16, 8, 64, 8).accumulate(**{**c, "positions": c["positions"].clone()}, out=out)
        got = check_weights(c)
        for b, n in enumerate(c["context_lens"].tolist()):
            assert torch.equal(out[b, :, :n], got[b, :, :n]) and (out[b, :, n:] == 7).all()


LIMITS = [1024, 4096, 16384, 32768, 65536]  # tokens up to which a selecting thread holds 1, 4, 16, 32 and 64 keys


@pytest.mark.parametrize("n", [m for limit in LIMITS for m in (limit, limit + 1)] + [70001])
@pytest.mark.parametrize("part", [0.43, 0.999, 0.002])
@pytest.mark.parametrize("elsewhere", [False, True])
def test_evict_on_both_sides_of_every_form(gpu, n, part, elsewhere):
    """Few moves, and more than a selecting workgroup makes itself (1024)."""
    c = ecase(gpu, [n], hkv=1, D=8, seed=n)
    out = (torch.full_like(c["weights"], -7.0), torch.full_like(c["positions"], -7)) if elsewhere else None
    budget = int(n * part) + 1
    check_evict(c, budget, min(4, budget), min(50, budget - min(4, budget)), out=out)


@pytest.mark.parametrize("kind", ["ties", "equal", "odd"])
@pytest.mark.parametrize("n", [4000, 16000, 30000, 60000, 66000])
def test_evict_ties_and_odd_weights_of_every_form(gpu, kind, n):
    check_evict(ecase(gpu, [n], hkv=1, D=8, kind=kind, seed=n), n // 3, 2, 5)


@pytest.mark.parametrize("width", [300, 1100, 2100, 4200])
def test_evict_short_contexts_in_wide_tables(gpu, width):
    """The table's width chooses the kernel, a context's length the form within it."""
    check_evict(ecase(gpu, [900, 3000, 40, 4700], D=8, width=width, seed=width), 500, 4, 20)


def test_evict_many_caches_of_many_moves(gpu):
    """From 128 caches on the selecting workgroups make up to 1024 moves, and leave the others."""
    check_evict(ecase(gpu, [6000, 5000] + [10] * 126, hkv=1, D=8, seed=4), 2600, 4, 20)
    check_evict(ecase(gpu, [6000, 5000] + [10] * 126, hkv=1, D=8, seed=5, dtype=F32, kind="ties"), 2600, 4, 20)


@pytest.mark.parametrize("rows,old", [((200, 150), (64, 500)), ((200, 1, 0, 9), (64, 500, 33, 20)), ((300, 300), (3, 5))])
def test_graphs_of_prompts_replay_as_eager(gpu, rows, old):
    """The kernels of many rows, their parts, and few rows beside them, captured and replayed with other inputs."""
    ev = kyro_amd.CacheEviction(16, 8, 128, 2)
    c = case(gpu, rows=rows, old=old, D=128, seed=1)
    out = torch.zeros_like(c["weights"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ev.accumulate_async(**c, max_q_len=max(rows), out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ev.accumulate_async(**c, max_q_len=max(rows), out=out)
    torch.cuda.current_stream().wait_stream(side)
    for turn in range(4):
        c["query"].copy_(torch.randn(c["query"].shape, device=gpu))
        c["key_cache"].copy_(torch.randn(c["key_cache"].shape, device=gpu))
        c["weights"].uniform_()
        out.fill_(turn)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.full_like(out, turn)
        ev.accumulate(**{**c, "positions": c["positions"].clone()}, out=eager)
        assert torch.equal(out, eager)


def test_a_verify_step_weighs_its_accepted_rows(gpu):
    """Every row of a call weighs, so a step that rejects drafts is weighed once its acceptance is known: with the
    rows that stay, at the lengths that stay. The same as if the rejected rows had never been."""
    c = case(gpu, rows=[5, 5, 5], old=[100, 7, 40], seed=11)
    stay = [3, 5, 1]
    rows = torch.cat([torch.arange(5 * b, 5 * b + n) for b, n in enumerate(stay)]).to(gpu)
    c["query"] = c["query"][rows]
    c["q_start_loc"] = torch.tensor([0, 3, 8, 9], dtype=torch.int32, device=gpu)
    c["context_lens"] -= torch.tensor([2, 0, 4], device=gpu)
    before = c["weights"].clone()
    check_weights(c)
    for b, n in enumerate((103, 12, 41)):
        assert torch.equal(c["weights"][b, :, n:], before[b, :, n:])
