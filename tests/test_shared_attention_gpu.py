"""Attention over shared prefixes against attention in 64 bits over each sequence's whole context."""
import ctypes

import numpy as np
import pytest
import torch

import kyro_amd
from kyro_amd import _lib, workloads as wl
from tests import helpers as h

pytestmark = pytest.mark.gpu

DIMS = [("bf16", D) for D in (64, 80, 96, 112, 128, 160, 192, 224, 256)] + [("f32", D) for D in (64, 80, 96, 112, 128)]

# (heads, kv heads), group starts, common tokens of each group (rounded down to blocks), each sequence's tokens beyond
# its group's, its rows (of them; a context may be shorter than its rows), None: every sequence `rows` long.
SHAPES = {
    # one group, one row each; tails of one token, around a tile and a slot
    "decode": ((8, 2), [0, 7], [500], [1, 15, 16, 17, 64, 65, 130], [1] * 7),
    # a verify step: 8 rows, 32 per kv head
    "verify": ((8, 2), [0, 6], [320], [8, 9, 31, 40, 71, 200], [8] * 6),
    # groups of one and of none, common tokens of none and of less than a tile, sequences before and behind the groups
    "groups": ((14, 2), [2, 5, 6, 6, 9, 12], [200, 400, 64, 0, 40], [30, 70, 5, 1, 90, 20, 3, 33, 50, 9, 12, 7, 64, 100],
               [1, 3, 5, 1, 0, 2, 1, 4, 9, 1, 1, 1, 6, 2]),
    # row groups of 128 in one sequence and across sequences, ragged
    "prompts": ((4, 1), [0, 4], [700], [33, 100, 77, 260], [33, 100, 1, 250]),
    # long: common tokens and one own tail split into parts
    "long": ((4, 1), [0, 3, 5], [6000, 3000], [10, 2000, 60, 5, 9], [1, 2, 1, 5, 1]),
    # many heads that each have their own keys
    "mha": ((6, 6), [0, 5], [250], [4, 8, 1, 20, 70], [1, 1, 1, 4, 1]),
}


def make(name, dtype, D, block=16, seed=0, short=()):
    """A case whose groups' tables start with the same blocks; `short`: sequences cut to fewer tokens than their group
    has in common."""
    (H, Hkv), starts, common, tails, rows = SHAPES[name]
    blocks = [c // block for c in common]
    ctx = list(tails)
    for g, nb in enumerate(blocks):
        for b in range(starts[g], starts[g + 1]):
            ctx[b] += nb * block
    case = wl.make_attention_case(context_lens=ctx, q_lens=rows, num_heads=H, num_kv_heads=Hkv, head_dim=D, block_size=block,
                                  dtype=dtype, seed=seed + D)
    for g, nb in enumerate(blocks):
        case.block_table[starts[g]:starts[g + 1], :nb] = case.block_table[starts[g], :nb] if starts[g] < len(ctx) else 0
    for b, n in short:
        case.context_lens[b] = n
    return case, np.array(starts, np.int32), np.array(blocks, np.int32)


def reference(case, causal=True):
    """(attention, sums of weight times |value|) in 64 bits."""
    H, Hkv, D = case.num_heads, case.num_kv_heads, case.head_dim
    cast = wl.bf16_bits_to_f32 if case.dtype == "bf16" else np.asarray
    out = torch.zeros(case.query.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b in range(case.batch):
        ctx, q0, q1 = int(case.context_lens[b]), int(case.q_start_loc[b]), int(case.q_start_loc[b + 1])
        n = q1 - q0
        if n == 0 or ctx == 0:
            continue
        ids = case.block_table[b, :-(-ctx // case.block_size)]
        k, v = (torch.from_numpy(cast(x[ids])).double().transpose(0, 1).reshape(Hkv, -1, D)[:, :ctx]
                for x in (case.key_cache, case.value_cache))
        q = torch.from_numpy(cast(case.query[q0:q1])).double().view(n, Hkv, H // Hkv, D).permute(1, 2, 0, 3)
        s = torch.matmul(q.reshape(Hkv, -1, D), k.transpose(1, 2)).view(Hkv, H // Hkv, n, ctx) / D ** 0.5
        if causal:
            s = s.masked_fill(torch.arange(ctx) > ctx - n + torch.arange(n).view(-1, 1), float("-inf"))
        p = torch.softmax(s, -1).nan_to_num().view(Hkv, -1, ctx)  # a row that sees nothing: 0
        for to, x in ((out, v), (mag, v.abs())):
            to[q0:q1] = torch.matmul(p, x).view(Hkv, H // Hkv, n, D).permute(2, 0, 1, 3).reshape(n, H, D)
    return out, mag


def run(gpu, case, starts, blocks, t=None, **kw):
    t = h.attention_tensors(case, gpu) if t is None else t
    attn = kyro_amd.PagedAttention(case.block_size, case.num_heads, case.head_dim, case.num_kv_heads)
    return attn.forward_shared(t["query"], t["key_cache"], t["value_cache"], t["block_table"], t["context_lens"],
                               h.to_device(starts, gpu), h.to_device(blocks, gpu), q_start_loc=t["q_start_loc"], **kw)


def check(out, case, ref, rows=None):
    """bf16: a weight is rounded once, by at most half a step, torch.finfo(torch.bfloat16).eps / 2 = 2^-8 of it (8 bits
    hold a value, the first of them implied), and sums in 32 bits of up to some thousand terms add less than 2^-12 of
    the terms' size; the output's own rounding is 2^-8 of it. f32: as the other attention tests."""
    exact, mag = ref
    err = (out.double().cpu() - exact).abs()
    if case.dtype == "bf16":
        bound = (2.0 ** -8 + 2.0 ** -12) * mag + (2.0 ** -8 * exact.abs() if out.dtype == torch.bfloat16 else 0) + 1e-30
    else:
        bound = torch.full_like(mag, h.ATOL_F32_SUMS) + (2.0 ** -8 * exact.abs() if out.dtype == torch.bfloat16 else 0)
    bad = ~(err <= bound)
    if rows is not None:
        bad = bad[rows]
    assert not bad.any(), f"{int(bad.sum())} values off, worst {float((err - bound).max()):.3g} past the bound"


@pytest.mark.parametrize("name", sorted(SHAPES))
@pytest.mark.parametrize("dtype,D", DIMS, ids=lambda x: str(x))
def test_shared_parity(gpu, name, dtype, D):
    case, starts, blocks = make(name, dtype, D, block=32 if D % 96 == 0 else 16)
    check(run(gpu, case, starts, blocks), case, reference(case))


@pytest.mark.parametrize("name,dtype,D,block", [("groups", "bf16", 128, 16), ("prompts", "bf16", 64, 64), ("verify", "f32", 96, 32),
                                                ("decode", "bf16", 256, 16), ("decode", "f32", 128, 16)])
def test_nan_past_the_context_and_outputs_in_bf16(gpu, name, dtype, D, block):
    """Every cache slot that no sequence holds is NaN, those of a sequence's last block past its context among them."""
    case, starts, blocks = make(name, dtype, D, block=block, seed=3)
    t = h.attention_tensors(case, gpu)
    used = torch.zeros(case.key_cache.shape[0], block, dtype=torch.bool)
    for b in range(case.batch):
        for i in range(int(case.context_lens[b])):
            used[int(case.block_table[b, i // block]), i % block] = True
    for x in ("key_cache", "value_cache"):
        t[x] = t[x].masked_fill((~used).to(gpu)[:, None, :, None], float("nan"))
    for causal in (True, False):
        out = run(gpu, case, starts, blocks, t, causal=causal, out_dtype=torch.bfloat16)
        check(out, case, reference(case, causal))


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_contexts_that_end_in_the_common_tokens(gpu, dtype, D, causal):
    """A sequence of no tokens, ones that end inside the common tokens, at their end, one row before it, and rows that
    see nothing; the rest of the group shares on."""
    case, starts, blocks = make("verify", dtype, D, short=((0, 0), (1, 100), (2, 320), (3, 327), (4, 3)))
    t = h.attention_tensors(case, gpu)
    out = torch.full_like(t["query"], float("nan"), dtype=torch.float32)
    check(run(gpu, case, starts, blocks, t, causal=causal, out=out), case, reference(case, causal))


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 128)])
def test_without_row_ranges_scale_and_reuse_hint(gpu, dtype, D):
    case, starts, blocks = make("decode", dtype, D)
    t = h.attention_tensors(case, gpu)
    ref = reference(case)
    attn = kyro_amd.PagedAttention(case.block_size, case.num_heads, D, case.num_kv_heads)
    args = (t["query"], t["key_cache"], t["value_cache"], t["block_table"], t["context_lens"], h.to_device(starts, gpu),
            h.to_device(blocks, gpu))
    outs = [attn.forward_shared(*args, kv_reuse=r) for r in ("auto", "shared", "stream")]
    check(outs[0], case, ref)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    half = attn.forward_shared(t["query"] * 2, *args[1:], scale=0.5 * D ** -0.5)
    check(half, case, ref)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 128)])
def test_no_groups_and_no_rows(gpu, dtype, D):
    case, _, _ = make("verify", dtype, D)
    none = np.zeros(0, np.int32)
    check(run(gpu, case, np.zeros(1, np.int32), none), case, reference(case))
    empty = wl.make_attention_case(context_lens=[40, 0], q_lens=[0, 0], num_heads=8, num_kv_heads=2, head_dim=D, dtype=dtype)
    assert run(gpu, empty, np.array([0, 2], np.int32), np.array([1], np.int32), max_q_len=1).shape == (0, 8, D)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 64)])
def test_groups_out_of_order_latch(gpu, dtype, D):
    """Faulty groups are reported, and everything is computed without them; a group with too many blocks alone shares
    nothing."""
    case, starts, blocks = make("groups", dtype, D, seed=5)
    ref = reference(case)
    width = case.block_table.shape[1]
    for s, nb in (([2, 5, 4, 6, 9, 12], blocks), ([-1, 5, 6, 6, 9, 12], blocks), ([2, 5, 6, 6, 9, 15], blocks),
                  (starts, [12, 25, width + 1, 0, 2]), (starts, [-3, 25, 4, 0, 2])):
        t = h.attention_tensors(case, gpu)
        out = torch.full_like(t["query"], float("nan"), dtype=torch.float32)
        with pytest.raises(kyro_amd.KyroError, match="group_starts"):
            run(gpu, case, np.array(s, np.int32), np.array(nb, np.int32), t, out=out)
        check(out, case, ref)


def test_faulty_sequences_latch(gpu):
    """A bad block among a sequence's own, a context past its table and rows out of order: reported, and the other
    sequences are computed as before. A bad common block's tokens count for none of the group's rows."""
    case, starts, blocks = make("verify", "bf16", 128, seed=7)
    ref = reference(case)
    for fault in ("own block", "context", "rows", "common block"):
        t = h.attention_tensors(case, gpu)
        hurt = {2}
        if fault == "own block":
            t["block_table"][2, 20] = case.key_cache.shape[0]
        elif fault == "context":
            t["context_lens"][2] = case.block_table.shape[1] * 16 + 1
        elif fault == "rows":
            t["q_start_loc"][3] = t["q_start_loc"][2] - 1
            hurt = {2, 3}  # both have the entry as a bound
        else:
            t["block_table"][:, 3] = -1
            hurt = set(range(6))
        out = torch.zeros_like(t["query"], dtype=torch.float32)
        with pytest.raises(kyro_amd.KyroError):
            run(gpu, case, starts, blocks, t, max_q_len=8, out=out)
        rows = torch.cat([torch.arange(8 * b, 8 * b + 8) for b in range(6) if b not in hurt] or [torch.zeros(0, dtype=torch.long)])
        check(out, case, ref, rows)
    gone = wl.AttentionCase(**{**case.__dict__, "block_table": np.delete(case.block_table, 3, 1), "context_lens": case.context_lens - 16})
    check(out, gone, reference(gone))


@pytest.mark.parametrize("B,G", [(1500, 1), (1500, 1200)])
def test_more_sequences_and_groups_than_the_plan_holds_in_lds(gpu, B, G):
    rng = np.random.RandomState(B + G)
    starts = np.concatenate([[0], np.sort(rng.randint(0, B + 1, G - 1)), [B]]).astype(np.int32)
    rows = rng.randint(0, 3, B)
    own = rng.randint(1, 40, B) + 2
    case = wl.make_attention_case(context_lens=96 + own, q_lens=rows, num_heads=2, num_kv_heads=1, head_dim=64, dtype="bf16", seed=B)
    for g in range(G):
        if starts[g] < starts[g + 1]:
            case.block_table[starts[g]:starts[g + 1], :6] = case.block_table[starts[g], :6]
    check(run(gpu, case, starts, np.full(G, 6, np.int32)), case, reference(case))


@pytest.mark.parametrize("B,most", [(300, 140), (40, 2000), (1100, 40)])
def test_more_row_groups_than_the_plan_holds_in_lds(gpu, B, most):
    """Sequences of none to several row groups (32 rows of a kv head each), some of which share."""
    rng = np.random.default_rng(B)
    rows = rng.integers(0, most, B)
    rows[rng.integers(0, B, B // 4)] = 0
    SHAPES["row_groups"] = ((4, 1), [0, B // 3, B // 3 + 1, B - 2], [130, 0, 64], (rows + rng.integers(0, 60, B)).tolist(), rows.tolist())
    try:
        case, starts, blocks = make("row_groups", "bf16", 64)
    finally:
        del SHAPES["row_groups"]
    check(run(gpu, case, starts, blocks), case, reference(case))


@pytest.mark.parametrize("dtype,D,block", [("bf16", 72, 16), ("bf16", 128, 8), ("f32", 256, 16), ("f32", 40, 24)])
def test_other_geometries_run_without_the_groups(gpu, dtype, D, block):
    case, starts, blocks = make("verify", dtype, D, block=block, seed=9)
    t = h.attention_tensors(case, gpu)
    attn = kyro_amd.PagedAttention(block, case.num_heads, D, case.num_kv_heads)
    want = attn.forward(t["query"], t["key_cache"], t["value_cache"], t["block_table"], t["context_lens"], q_start_loc=t["q_start_loc"],
                        kv_reuse="shared")
    assert torch.equal(run(gpu, case, starts, blocks, t), want)


def test_misaligned_caches_run_without_the_groups(gpu):
    case, starts, blocks = make("verify", "bf16", 128, seed=11)
    t = h.attention_tensors(case, gpu)
    for x in ("key_cache", "value_cache"):
        flat = torch.zeros(t[x].numel() + 8, dtype=torch.bfloat16, device=gpu)
        flat[4:4 + t[x].numel()] = t[x].flatten()
        t[x] = flat[4:4 + t[x].numel()].view(t[x].shape)
    check(run(gpu, case, starts, blocks, t), case, reference(case))


def test_the_common_tokens_are_read_once(gpu):
    """The tables of all but the group's first sequence name other, wrong blocks for the common tokens, which a kernel
    that walked them for each sequence would read."""
    case, starts, blocks = make("verify", "bf16", 128, seed=13)
    ref = reference(case)
    t = h.attention_tensors(case, gpu)
    t["block_table"][1:, : int(blocks[0])] = t["block_table"][0, -1]
    check(run(gpu, case, starts, blocks, t), case, ref)


@pytest.mark.parametrize("name", ["verify", "long", "groups"])
def test_same_result_every_time_and_from_a_graph(gpu, name):
    case, starts, blocks = make(name, "bf16", 128, seed=17)
    t = h.attention_tensors(case, gpu)
    attn = kyro_amd.PagedAttention(16, case.num_heads, 128, case.num_kv_heads)
    args = (t["query"], t["key_cache"], t["value_cache"], t["block_table"], t["context_lens"], h.to_device(starts, gpu),
            h.to_device(blocks, gpu))
    kw = dict(q_start_loc=t["q_start_loc"], max_q_len=case.max_q_len)
    eager = attn.forward_shared(*args, **kw)
    for _ in range(3):
        assert torch.equal(attn.forward_shared(*args, **kw), eager)
    out = torch.zeros_like(eager)
    s = torch.cuda.Stream(gpu)
    s.wait_stream(torch.cuda.current_stream(gpu))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        attn.forward_shared_async(*args, out=out, **kw)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert torch.equal(attn.forward_shared(*args, **kw), eager)


def test_a_capture_without_scratch_is_refused_and_the_size_query_suffices(gpu):
    case, starts, blocks = make("verify", "bf16", 128, seed=19)
    t = h.attention_tensors(case, gpu)
    attn = kyro_amd.PagedAttention(16, case.num_heads, 128, case.num_kv_heads)
    args = (t["query"], t["key_cache"], t["value_cache"], t["block_table"], t["context_lens"], h.to_device(starts, gpu),
            h.to_device(blocks, gpu))
    kw = dict(q_start_loc=t["q_start_loc"], max_q_len=8)
    ctx = kyro_amd.Context(0)
    eager = attn.forward_shared(*args, **kw)
    out = torch.zeros_like(eager)
    s = torch.cuda.Stream(gpu)
    s.wait_stream(torch.cuda.current_stream(gpu))
    ctx.set_stream(s.cuda_stream)  # which waits for the context's own stream, as no call inside a capture may
    with pytest.raises(kyro_amd.KyroError, match="kyro_ctx_reserve"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
            attn.forward_shared_async(*args, out=out, context=ctx, **kw)
    p = _lib.PagedAttentionParams(16, case.num_heads, 128, case.num_kv_heads, 6, 48, case.block_table.shape[1], case.key_cache.shape[0],
                                  _lib.KYRO_BF16, _lib.KYRO_F32, 1, 0.0, 0, 0, 8, 0, 0)
    n = ctypes.c_size_t()
    _lib.check(_lib.lib().kyro_paged_attention_shared_workspace(ctx.handle, ctypes.byref(p), 1, 1, ctypes.byref(n)))
    ctx.reserve(n.value)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        attn.forward_shared_async(*args, out=out, context=ctx, **kw)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
