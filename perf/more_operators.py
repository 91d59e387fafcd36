"""The operators of a serving step on caches whose sequences share prefixes, with block tables that live on
the GPU, as cases that can be timed and compared with their plain forms.

    share     PagedAttention.forward_shared_async   one layer's attention where groups of sequences hold the same
                                                    first blocks, which are read and multiplied once a group
    extend    RequestTables.extend_async            a step's new rows: blocks from the pool, block table, context
                                                    lengths, row ranges, positions and cache slots
    keep      RequestTables.keep_async              after acceptance: the rows that stay count, the blocks of the
                                                    others go back to the pool

A case is a dict of plain values; `listed` gives the ones that are always measured, `draw` more of the same
ranges. Lengths follow from the case alone, values and orders from the seed. With `own` false the operators run
in their plain form, elementary torch operations in 32 bits (whole numbers in 64); with `own` true through the
library. `exact` computes them in 64 bits. Inputs are made on the GPU.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}


def _share(name, batch, heads, kv_heads, dim, groups, prefix, tail, rows, loose=0, dtype="bf16", block=16):
    """`groups` groups of about as many sequences, `loose` more sequences that share nothing. `prefix` (least, most
    over the groups) tokens in common, in whole blocks; `tail` (least, most over the batch) tokens of a sequence's
    own before its new ones, `rows` new ones."""
    case = {"op": "share", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block,
            "groups": groups, "prefix_min": prefix[0], "prefix_max": prefix[1], "tail_min": tail[0], "tail_max": tail[1],
            "rows_min": rows[0], "rows_max": rows[1], "loose": loose, "dtype": dtype}
    return dict(case, name=name) if name else case


def _tables(op, name, batch, old, rows, requests, width, block=16, padding=0):
    """`batch` of `requests` requests of `old` (least, most) tokens bring `rows` new ones; `padding` more entries of
    the batch are empty. `width`: blocks of a row of the tables."""
    case = {"op": op, "batch": batch, "old_min": old[0], "old_max": old[1], "rows_min": rows[0], "rows_max": rows[1],
            "requests": requests, "width": width, "block": block, "padding": padding}
    return dict(case, name=name) if name else case


def listed():
    return [
        # Four samples of one prompt, a token each: all latency.
        _share("share_samples", 4, 32, 8, 128, 1, (1000, 1000), (1, 120), (1, 1)),
        # Decode of 64 conversations behind one system prompt.
        _share("share_decode", 64, 32, 8, 128, 1, (8192, 8192), (16, 1000), (1, 1)),
        # The verify step of 64 sequences with 7 drafts behind one.
        _share("share_verify", 64, 32, 8, 128, 1, (4096, 4096), (100, 1500), (8, 8)),
        # Questions about one long document.
        _share("share_document", 32, 32, 8, 128, 1, (32768, 32768), (20, 300), (1, 1)),
        # Mixed drafts behind prompts of four applications, and sequences of none.
        _share("share_mixed", 128, 64, 8, 128, 4, (600, 6000), (1, 1200), (1, 9), loose=16),
        # Eight new questions, 100 to 300 tokens each, read behind the same 6000 tokens.
        _share("share_prompts", 8, 32, 8, 128, 1, (6000, 6000), (0, 0), (100, 300)),
        # f32 caches, blocks of 32, odd sizes.
        _share("share_f32", 24, 14, 2, 96, 2, (700, 1900), (5, 333), (5, 5), dtype="f32", block=32),
        # One conversation, one token: all latency.
        _tables("extend", "extend_one", 1, (999, 999), (1, 1), 16, 256),
        # The verify step of 64 sequences with 7 drafts at about 4096 tokens.
        _tables("extend", "extend_verify", 64, (3000, 4088), (8, 8), 96, 264),
        # Chunks of many prompts beside decoding sequences, tables of 131072 tokens.
        _tables("extend", "extend_chunks", 256, (1000, 100000), (1, 2000), 300, 8192, padding=8),
        # After the verify step: some of the 7 drafts stay.
        _tables("keep", "keep_verify", 64, (3000, 4088), (8, 8), 96, 264),
        # Long drafts of many sequences, most rejected.
        _tables("keep", "keep_drafts", 1024, (100, 8000), (1, 64), 1200, 520, padding=8),
    ]


# ------------------------------------------------------------------------------------ drawn cases

def _spread(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("share", "share", "share", "extend", "keep"))
    if op == "share":
        return _draw_share(rng)
    block = rng.choice((16, 16, 32, 64, 8, 1, 24))
    batch = _spread(rng, 1, 1024)
    most = _spread(rng, 16, 120000)
    rows = rng.choice(((1, 1), (8, 8), (1, 9), (1, _spread(rng, 16, 2000)))) if op == "extend" else \
        rng.choice(((1, 1), (8, 8), (1, 9), (1, 64)))
    while batch * (most / block + rows[1] / 8 + 8) > 2.2e6:
        batch, most = max(1, batch // 2), max(16, most * 3 // 4)
    width = -(-(most + rows[1]) // block) + rng.choice((0, 3, 100))
    return _tables(op, None, batch, (most // rng.choice((1, 3, 20)), most), rows, batch + rng.choice((0, 7, 200)), width, block,
                   padding=rng.choice((0, 0, 5)))


def _draw_share(rng):
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    dim = rng.choice((64, 128, 128, 128, 80, 96, 256) if dtype == "bf16" else (64, 80, 96, 128))
    kv_heads = rng.choice((1, 2, 4, 8, 8, 16, 32))
    group = rng.choice((1, 4, 7, 8) if kv_heads <= 8 else (1, 2))
    block = rng.choice((16, 16, 16, 32, 64))
    size = _SIZE[dtype]
    batch = _spread(rng, 2, 160)
    groups = rng.choice((1, 1, 1, 2, 5))
    rows = rng.choice(((1, 1), (1, 1), (8, 8), (1, 9), (5, 5), (1, _spread(rng, 16, 300))))
    prefix, tail = _spread(rng, 128, 32768), _spread(rng, 8, 2000)
    prefix_min, tail_min = prefix // rng.choice((1, 1, 4)), tail // rng.choice((1, 4, 100))
    loose = rng.choice((0, 0, 1, batch // 3))
    while True:
        groups = max(1, min(groups, (batch - loose) // 2 or 1))
        loose = min(loose, max(0, batch - groups))
        case = _share(None, batch, kv_heads * group, kv_heads, dim, groups, (min(prefix_min, prefix), prefix), (min(tail_min, tail), tail),
                      rows, loose, dtype, block)
        # At most the largest listed case's products (in f32 an eighth) and bytes.
        if work(case)["flops"] <= (6.5e10 if dtype == "bf16" else 8e9) and work(case)["bytes"] <= 3.4e8 and \
                (batch + 1) * (prefix + tail + rows[1]) * kv_heads * dim * size <= 6e9:
            return case
        if rows[1] > 16:
            rows = (rows[0], rows[1] * 2 // 3)
        elif batch > 8:
            batch, loose = batch * 2 // 3, loose * 2 // 3
        else:
            prefix, tail = max(64, prefix * 2 // 3), max(1, tail * 2 // 3)


# ------------------------------------------------------------------------------------ sizes of a case

def _between(least, most, n):
    """n whole numbers from least to most, evenly spaced."""
    return [most if n == 1 else least + (most - least) * i // (n - 1) for i in range(n)]


def _share_sizes(case):
    """Sequences of each group (the last ones share nothing), blocks in common, and for each sequence its group, new
    rows and tokens with them."""
    groups, shared = case["groups"], case["batch"] - case["loose"]
    members = [shared // groups + (g < shared % groups) for g in range(groups)]
    blocks = [max(1, p // case["block"]) for p in _between(case["prefix_min"], case["prefix_max"], groups)]
    if case["loose"]:
        members, blocks = members + [case["loose"]], blocks + [0]
    rows = _between(case["rows_max"], case["rows_min"], case["batch"])
    tails = _between(case["tail_min"], case["tail_max"], case["batch"])
    group_of = [g for g, n in enumerate(members) for _ in range(n)]
    # Members of a group are spread over the range of lengths.
    order = [i * 7919 % case["batch"] if math.gcd(7919, case["batch"]) == 1 else i for i in range(case["batch"])]
    rows, tails = [rows[i] for i in order], [tails[i] for i in order]
    ctx = [blocks[g] * case["block"] + t + r for g, t, r in zip(group_of, tails, rows)]
    return members, blocks, group_of, rows, ctx


def _table_sizes(case):
    """(new rows, tokens before) of each entry of the batch that is not empty; the longest bring the fewest rows."""
    return (_between(case["rows_max"], case["rows_min"], case["batch"]),
            _between(case["old_min"], case["old_max"], case["batch"]))


def work(case):
    if case["op"] == "share":
        members, blocks, group_of, rows, ctx = _share_sizes(case)
        size, dim = _SIZE[case["dtype"]], case["dim"]
        tokens = sum(blocks) * case["block"] + sum(c - blocks[g] * case["block"] for g, c in zip(group_of, ctx))
        seen = sum(r * c - r * (r - 1) // 2 for r, c in zip(rows, ctx)) * case["heads"]
        return {"bytes": 2 * tokens * case["kv_heads"] * dim * size + 2 * sum(rows) * case["heads"] * dim * size,
                "flops": 4 * seen * dim}
    rows, old = _table_sizes(case)
    bs = case["block"]
    held = sum(-(-o // bs) for o in old)
    fresh = sum(-(-(o + r) // bs) for o, r in zip(old, rows)) - held
    entries = case["batch"] + case["padding"]
    if case["op"] == "extend":
        return {"bytes": 8 * (held + 2 * fresh + entries * case["width"]) + 16 * sum(rows) + entries * (4 + 4 + 32 + 12), "flops": 0}
    return {"bytes": 8 * fresh + entries * (4 + 4 + 4 + 8 + 32 + 8), "flops": 0}  # about half of the new blocks go back


# ------------------------------------------------------------------------------------ inputs

def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _starts(rows):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 13)
    rng = np.random.RandomState(int(seed) % 2**31)
    return (_prepare_share if case["op"] == "share" else _prepare_tables)(case, gen, rng)


def _prepare_share(case, gen, rng):
    dtype, block, kv_heads, dim = _DTYPES[case["dtype"]], case["block"], case["kv_heads"], case["dim"]
    members, blocks, group_of, rows, ctx = _share_sizes(case)
    width = max(-(-c // block) for c in ctx)
    total = sum(blocks) + sum(-(-c // block) - blocks[g] for g, c in zip(group_of, ctx)) + 3
    ids = rng.permutation(total)
    table = np.zeros((case["batch"], width), np.int64)
    common, at = [], 0
    for n in blocks:
        common.append(ids[at:at + n])
        at += n
    for b, (g, c) in enumerate(zip(group_of, ctx)):
        n, mine = blocks[g], -(-c // block) - blocks[g]
        table[b, :n] = common[g]
        table[b, n:n + mine] = ids[at:at + mine]
        at += mine
    s = {"case": case, "blocks": blocks, "members": members, "rows": rows, "ctx_list": ctx, "most": max(rows),
         "tail_width": max(-(-c // block) - blocks[g] for g, c in zip(group_of, ctx))}
    s["table"], s["ctx"] = torch.from_numpy(table).cuda(), torch.tensor(ctx, dtype=torch.int64, device="cuda")
    s["starts"], s["group_starts"] = _starts(rows), _starts(members)
    s["group_blocks"] = torch.tensor(blocks, dtype=torch.int32, device="cuda")
    # Queries of a trained model are sharper than unit normal ones against unit normal keys.
    s["q"] = _normal(gen, (sum(rows), case["heads"], dim), dtype) * 1.5
    s["kc"], s["vc"] = (_normal(gen, (total, kv_heads, block, dim), dtype) for _ in range(2))
    return s


def _prepare_tables(case, gen, rng):
    block, width, entries = case["block"], case["width"], case["batch"] + case["padding"]
    rows, old = _table_sizes(case)
    order = rng.permutation(case["batch"])
    rows, old = [rows[i] for i in order], [old[i] for i in order]
    before = [-(-o // block) for o in old]
    after = [-(-(o + r) // block) for o, r in zip(old, rows)]
    own_ids, spare = sum(before), sum(after) - sum(before) + 100
    ids = rng.permutation(own_ids + spare + 5)
    owner = rng.permutation(case["requests"])[: case["batch"]]
    # A request: tokens, blocks held, blocks at the front that are no blocks of the pool (a shared prefix).
    requests = np.zeros((case["requests"], 4), np.int32)
    blocks = np.zeros((case["requests"], width), np.int64)
    pool = ids[own_ids:own_ids + spare].copy()
    taken, at = 0, 0
    for r, o, n, nb, na in zip(owner, old, rows, before, after):
        blocks[r, :nb] = ids[at:at + nb]
        at += nb
        requests[r, :3] = o, nb, nb // 2
        if case["op"] == "keep":  # after extend
            blocks[r, nb:na] = pool[len(pool) - 1 - taken - np.arange(na - nb)]
            taken += na - nb
            requests[r, 1] = na
    empty = [0] * case["padding"]
    s = {"case": case, "total": sum(rows)}
    s["requests"], s["blocks"], s["pool"] = (torch.from_numpy(x).cuda() for x in (requests, blocks, pool))
    s["count"] = torch.tensor([len(pool) - taken], dtype=torch.int32, device="cuda")
    s["state_rows"] = torch.tensor(list(owner) + [-1] * case["padding"], dtype=torch.int32, device="cuda")
    s["new"] = torch.tensor(rows + empty, dtype=torch.int32, device="cuda")
    if case["op"] == "keep":
        s["starts"] = _starts(rows + empty)
        s["ctx"] = torch.tensor([o + r for o, r in zip(old, rows)] + empty, dtype=torch.int64, device="cuda")
        # Of the rows after the first, which always stays, a geometric number does.
        accepted = np.minimum(rng.geometric(0.4, entries) - 1, np.maximum(np.array(rows + empty) - 1, 0))
        s["accepted"] = torch.from_numpy(accepted.astype(np.int32)).cuda()
    s["num_blocks"] = len(ids)
    return s


# ------------------------------------------------------------------------------------ the operators

def run(s):
    case = s["case"]
    if own:
        return _OWN[case["op"]](s, case)
    return _PLAIN[case["op"]](s, case)


def _own_share(s, c):
    import kyro_amd

    attn = kyro_amd.PagedAttention(c["block"], c["heads"], c["dim"], c["kv_heads"])
    return attn.forward_shared_async(s["q"], s["kc"], s["vc"], s["table"], s["ctx"], s["group_starts"], s["group_blocks"],
                                     q_start_loc=s["starts"], max_q_len=s["most"], out_dtype=s["q"].dtype)


def _handle(s, c):
    import kyro_amd

    if "handle" not in s:  # a program's, for as long as it serves
        s["handle"] = kyro_amd.RequestTables(c["block"], s["requests"], s["blocks"], s["pool"], s["count"], s["num_blocks"])
    return s["handle"]


def _own_extend(s, c):
    step = _handle(s, c).extend_async(s["state_rows"], s["new"], total_q=s["total"], max_blocks_per_seq=c["width"])
    return (step.block_table, step.context_lens, step.q_start_loc, step.positions, step.slots, s["requests"], s["blocks"],
            s["pool"], s["count"])


def _own_keep(s, c):
    ctx = _handle(s, c).keep_async(s["state_rows"], s["ctx"], s["starts"], s["accepted"], plus=1)
    return ctx, s["requests"], s["blocks"], s["pool"], s["count"]


def _softmax_parts(scores, values):
    """(largest score, sum of weights, weighted values) of scores [.., n, t] against values [.., t, D]; rows that see
    nothing have none."""
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0))
    return top, p.sum(-1, keepdim=True), torch.matmul(p, values)


def _plain_share(s, c):
    batch, heads, hkv, dim, block, most = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["block"], s["most"]
    group, scale = heads // hkv, dim ** -0.5
    starts = s["starts"].long()
    n = starts[1:] - starts[:-1]
    first = torch.repeat_interleave(s["group_blocks"].long(), s["group_starts"][1:].long() - s["group_starts"][:-1].long())
    # The common tokens of each group against all its rows.
    total = s["q"].shape[0]
    top = torch.full((total, heads, 1), -math.inf, device="cuda")
    sums = torch.zeros((total, heads, 1), device="cuda")
    acc = torch.zeros((total, heads, dim), device="cuda")
    seq = 0
    for members, blocks in zip(s["members"], s["blocks"]):
        r0, r1 = sum(s["rows"][:seq]), sum(s["rows"][:seq + members])
        if blocks and r1 > r0:
            keys, values = (x[s["table"][seq, :blocks]].transpose(0, 1).reshape(hkv, blocks * block, dim).float()
                            for x in (s["kc"], s["vc"]))
            q = s["q"][r0:r1].float().view(r1 - r0, hkv, group, dim).transpose(0, 1).reshape(hkv, -1, dim)
            parts = _softmax_parts(torch.matmul(q, keys.transpose(-1, -2)) * scale, values)
            for to, x in zip((top, sums, acc), parts):
                to[r0:r1] = x.view(hkv, r1 - r0, group, -1).transpose(0, 1).reshape(r1 - r0, heads, -1)
        seq += members
    # Each sequence's own tokens against its rows.
    width = s["tail_width"]
    at = (first[:, None] + torch.arange(width, device="cuda")).clamp(max=s["table"].shape[1] - 1)
    ids = s["table"].gather(1, at)
    keys, values = (x[ids].permute(0, 2, 1, 3, 4).reshape(batch, hkv, width * block, dim).float() for x in (s["kc"], s["vc"]))
    j = torch.arange(most, device="cuda")
    row = (starts[:-1, None] + j).clamp(max=total - 1)
    q = s["q"][row].float().view(batch, most, hkv, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, hkv, most * group, dim)
    scores = (torch.matmul(q, keys.transpose(-1, -2)) * scale).view(batch, hkv, most, group, width * block)
    tok = first[:, None] * block + torch.arange(width * block, device="cuda")
    sees = tok[:, None] <= ((s["ctx"] - n)[:, None] + j)[..., None]
    scores = scores.masked_fill(~sees[:, None, :, None], -math.inf).view(batch, hkv, most * group, width * block)
    parts = [x.view(batch, hkv, most, group, -1).permute(0, 2, 1, 3, 4).reshape(batch, most, heads, -1)[j < n[:, None]]
             for x in _softmax_parts(scores, values)]
    best = torch.maximum(top, parts[0])
    a, b = torch.exp(top - best), torch.exp(parts[0] - best)
    return ((acc * a + parts[2] * b) / (sums * a + parts[1] * b)).to(s["q"].dtype)


def _plain_extend(s, c):
    bs, width = c["block"], c["width"]
    r, new = s["state_rows"].long(), s["new"].long()
    real = r >= 0
    rec = s["requests"][r.clamp(min=0)].long()
    old, held = rec[:, 0], rec[:, 1]
    ctx = torch.where(real, old + new, 0)
    need = torch.where(real, ((ctx + bs - 1) // bs - held).clamp(min=0), 0)
    before = need.cumsum(0) - need
    i = torch.arange(width, device="cuda")
    popped = s["pool"][(s["count"].long() - 1 - before[:, None] - (i - held[:, None])).clamp(0, s["pool"].shape[0] - 1)]
    ids = torch.where(i < held[:, None], s["blocks"][r.clamp(min=0)], popped)
    table = torch.where(real[:, None] & (i < (held + need)[:, None]), ids, 0)
    b, at = (real[:, None] & (i >= held[:, None]) & (i < (held + need)[:, None])).nonzero(as_tuple=True)
    s["blocks"][r[b], at] = table[b, at]
    s["requests"][r[real], 1] = (held + need)[real].int()
    s["count"] -= need.sum().int()
    starts = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), new.cumsum(0)))
    row = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    positions = old[seq] + row - starts[seq]
    slots = table[seq, positions // bs] * bs + positions % bs
    return table, ctx, starts.int(), positions, slots, s["requests"], s["blocks"], s["pool"], s["count"]


def _plain_keep(s, c):
    bs = c["block"]
    r, starts = s["state_rows"].long(), s["starts"].long()
    real = r >= 0
    rec = s["requests"][r.clamp(min=0)].long()
    held = rec[:, 1]
    ctx = torch.where(real, s["ctx"] - (starts[1:] - starts[:-1]) + s["accepted"].long() + 1, 0)
    stay = torch.minimum(held, torch.maximum((ctx + bs - 1) // bs, rec[:, 2]))
    freed = torch.where(real, held - stay, 0)
    before = freed.cumsum(0) - freed
    i = torch.arange(int(c["rows_max"]) // bs + 2, device="cuda")
    b, k = (i < freed[:, None]).nonzero(as_tuple=True)
    s["pool"][s["count"].long() + before[b] + k] = s["blocks"][r[b], stay[b] + k]
    s["requests"][r[real], 0] = ctx[real].int()
    s["requests"][r[real], 1] = stay[real].int()
    s["count"] += freed.sum().int()
    return ctx, s["requests"], s["blocks"], s["pool"], s["count"]


_OWN = {"share": _own_share, "extend": _own_extend, "keep": _own_keep}
_PLAIN = {"share": _plain_share, "extend": _plain_extend, "keep": _plain_keep}


# ------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"share": _exact_share, "extend": _exact_extend, "keep": _exact_keep}[case["op"]](s, case)


def _exact_share(s, c):
    """Every sequence over its whole context, one kv head after the other."""
    group, block = c["heads"] // c["kv_heads"], c["block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, length) in enumerate(zip(s["rows"], s["ctx_list"])):
        ids = s["table"][b, : -(-length // block)]
        sees = torch.arange(length, device="cuda") <= length - n + torch.arange(n, device="cuda").repeat_interleave(group)[:, None]
        for h in range(c["kv_heads"]):
            keys = s["kc"][ids, h].reshape(-1, c["dim"])[:length].double()
            values = s["vc"][ids, h].reshape(-1, c["dim"])[:length].double()
            q = s["q"][first:first + n, h * group:(h + 1) * group].double().reshape(n * group, c["dim"])
            p = torch.softmax((q @ keys.T / math.sqrt(c["dim"])).masked_fill(~sees, -math.inf), -1)
            out[first:first + n, h * group:(h + 1) * group] = (p @ values).view(n, group, c["dim"])
        first += n
    return out


def _exact_extend(s, c):
    bs, width = c["block"], c["width"]
    requests, blocks, pool = s["requests"].cpu().numpy(), s["blocks"].cpu().numpy(), s["pool"].cpu().numpy()
    count = int(s["count"].item())
    rows, new = s["state_rows"].tolist(), s["new"].tolist()
    table, ctx = np.zeros((len(rows), width), np.int64), np.zeros(len(rows), np.int64)
    positions, slots = [], []
    for b, (r, n) in enumerate(zip(rows, new)):
        if r < 0:
            continue
        ctx[b] = requests[r, 0] + n
        while requests[r, 1] * bs < ctx[b]:
            count -= 1
            blocks[r, requests[r, 1]] = pool[count]
            requests[r, 1] += 1
        table[b, : requests[r, 1]] = blocks[r, : requests[r, 1]]
        at = np.arange(ctx[b] - n, ctx[b])
        positions.append(at)
        slots.append(blocks[r, at // bs] * bs + at % bs)
    return (table, ctx, np.concatenate([[0], np.cumsum(new)]).astype(np.int32), np.concatenate(positions), np.concatenate(slots),
            requests, blocks, pool, np.array([count], np.int32))


def _exact_keep(s, c):
    bs = c["block"]
    requests, blocks, pool = s["requests"].cpu().numpy(), s["blocks"].cpu().numpy(), s["pool"].cpu().numpy()
    count, starts = int(s["count"].item()), s["starts"].tolist()
    ctx = np.zeros(s["ctx"].shape[0], np.int64)
    for b, (r, length, accepted) in enumerate(zip(s["state_rows"].tolist(), s["ctx"].tolist(), s["accepted"].tolist())):
        if r < 0:
            continue
        ctx[b] = requests[r, 0] = length - (starts[b + 1] - starts[b]) + accepted + 1
        stay = max(-(-int(ctx[b]) // bs), int(requests[r, 2]))
        for i in range(stay, int(requests[r, 1])):
            pool[count] = blocks[r, i]
            count += 1
        requests[r, 1] = min(stay, int(requests[r, 1]))
    return ctx, requests, blocks, pool, np.array([count], np.int32)
