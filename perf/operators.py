"""The operators around the paged KV cache that a serving step calls next to attention, as cases that
can be timed and compared with their plain forms.

    rotate    PagedKVCache.append_qkv_async     one layer's new query, key and value rows: head norms and
                                                position rotation, the keys and values into the paged cache
    weigh     CacheEviction.accumulate_async    the attention weight that new rows give each cached token,
                                                added up for each kv head
    evict     CacheEviction.evict_async         caches longer than a budget keep the tokens of the most
                                                weight, the first and the newest ones

A case is a dict of plain values; `listed` gives the ones that are always measured, `draw` more of the
same ranges. Lengths follow from the case alone, values and orders from the seed. With `own` false the
operators run in their plain form, elementary torch operations in 32 bits; with `own` true through the
library. `exact` computes them in 64 bits. Inputs are made on the GPU.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}
_EPS = 1e-6
_BASE = 10000.0


def _rotate(name, batch, heads, kv_heads, dim, old, rows, src="bf16", dtype="bf16", block=16, rotary=None, norm=True,
            interleaved=False, packed=True, moved=False):
    """`old` and `rows` are (least, most) over the batch: tokens cached before, and new ones. `packed`: query, key and
    value are slices of one projection's output. `moved`: the cache has lost tokens, so positions are given."""
    case = {"op": "rotate", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block,
            "old_min": old[0], "old_max": old[1], "rows_min": rows[0], "rows_max": rows[1], "src": src, "dtype": dtype,
            "rotary": dim if rotary is None else rotary, "norm": norm, "interleaved": interleaved, "packed": packed,
            "moved": moved}
    return dict(case, name=name) if name else case


def _weigh(name, batch, heads, kv_heads, dim, old, rows, dtype="bf16", block=16):
    case = {"op": "weigh", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block,
            "old_min": old[0], "old_max": old[1], "rows_min": rows[0], "rows_max": rows[1], "dtype": dtype}
    return dict(case, name=name) if name else case


def _evict(name, batch, kv_heads, dim, ctx, budget, sink, recent, dtype="bf16", block=16, again=False):
    """`again`: the cache has been cut to the budget before, so its first `budget` slots are in no order."""
    case = {"op": "evict", "batch": batch, "kv_heads": kv_heads, "dim": dim, "block": block, "ctx_min": ctx[0],
            "ctx_max": ctx[1], "budget": budget, "sink": sink, "recent": recent, "dtype": dtype, "again": again}
    return dict(case, name=name) if name else case


def listed():
    return [
        # One conversation, one token: all latency.
        _rotate("rotate_one", 1, 32, 8, 128, (999, 999), (1, 1)),
        # The verify step of 64 sequences with 7 drafts, on caches that have lost tokens before.
        _rotate("rotate_verify", 64, 32, 8, 128, (500, 1000), (8, 8), moved=True),
        # Four new prompts of 2048 tokens.
        _rotate("rotate_prompts", 4, 32, 8, 128, (0, 0), (2048, 2048)),
        # A partial, interleaved rotation without norms, f32 rows into a bf16 cache, ragged chunks of prompts.
        _rotate("rotate_partial", 7, 14, 2, 96, (0, 700), (1, 777), src="f32", block=32, rotary=48, norm=False,
                interleaved=True, packed=False),
        # One conversation, one token.
        _weigh("weigh_one", 1, 32, 8, 128, (999, 999), (1, 1)),
        # The verify step of 64 sequences with 7 drafts at about 4096 tokens.
        _weigh("weigh_verify", 64, 32, 8, 128, (4088, 4088), (8, 8)),
        # Two prompts' next 512 tokens after 7680: the rows that decide what a long prompt keeps.
        _weigh("weigh_chunk", 2, 32, 8, 128, (7680, 7680), (512, 512)),
        # Every head its own keys, f32 caches, ragged.
        _weigh("weigh_f32", 16, 32, 32, 128, (507, 2043), (5, 5), dtype="f32"),
        # One conversation of 1000 tokens cut to 512.
        _evict("evict_one", 1, 8, 128, (1000, 1000), 512, 4, 128),
        # Steady serving: 64 sequences come back 256 tokens over a budget of 2048 they were cut to before.
        _evict("evict_steady", 64, 8, 128, (2304, 2304), 2048, 4, 256, again=True),
        # After long prompts: most of the cache goes.
        _evict("evict_prompts", 8, 8, 128, (6000, 16384), 1024, 4, 64),
        # Odd sizes on f32 caches; some sequences are below the budget and stay as they are.
        _evict("evict_f32", 9, 5, 80, (37, 1500), 701, 1, 33, dtype="f32", block=32),
    ]


# ------------------------------------------------------------------------------------ drawn cases

def _spread(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("rotate", "weigh", "weigh", "evict"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    dim = rng.choice((64, 128, 128, 128, 80, 96, 112, 72, 256, 40))
    kv_heads = rng.choice((1, 2, 4, 8, 8, 16, 32))
    group = rng.choice((1, 4, 7, 8) if kv_heads <= 8 else (1, 2))
    block = rng.choice((16, 16, 16, 32, 64, 8))
    if op == "rotate":
        batch = _spread(rng, 1, 128)
        most = rng.choice((1, 5, 8, _spread(rng, 16, 4096)))
        src = "f32" if dtype == "f32" else rng.choice(("bf16", "bf16", "f32"))
        while batch * most * (group + 2) * kv_heads * dim * (_SIZE[src] + _SIZE[dtype]) > 1.6e8 and batch * most > 1:
            batch, most = max(1, batch // 2), max(1, most * 3 // 4)
        old = _spread(rng, 1, 1024) - 1
        return _rotate(None, batch, kv_heads * group, kv_heads, dim, (old // rng.choice((1, 3)), old),
                       (max(1, most // rng.choice((1, 4))), most), src, dtype, block,
                       rotary=rng.choice((dim, dim, dim, dim // 2)), norm=rng.choice((True, True, False)),
                       interleaved=rng.choice((False, False, True)), packed=rng.choice((True, False)),
                       moved=rng.choice((True, False)))
    if op == "weigh":
        size = _SIZE[dtype]
        if rng.random() < 0.35:  # chunks of prompts, at most the products of the largest listed one
            batch, most = _spread(rng, 1, 6), _spread(rng, 64, 1024)
            old = rng.choice((0, _spread(rng, 1, 8000)))
            rows = (max(1, most // rng.choice((1, 2))), most)
            limit = 6e10 if dtype == "bf16" else 8e9
        else:
            batch, most = _spread(rng, 1, 96), _spread(rng, 32, 65536)
            rows = rng.choice(((1, 1), (1, 1), (5, 5), (8, 8), (1, 9)))
            old, limit = most, 6e10
        while True:
            case = _weigh(None, batch, kv_heads * group, kv_heads, dim, (old // rng.choice((1, 3, 12)), old), rows, dtype, block)
            if work(case)["flops"] <= limit and batch * (old + rows[1]) * kv_heads * dim * size <= 5.3e8:
                return case
            if batch > 1:
                batch = batch * 2 // 3
            elif old > 64:
                old = old * 3 // 4
            else:
                rows = (max(1, rows[0] // 2), max(1, rows[1] // 2))
    batch, ctx = _spread(rng, 1, 64), _spread(rng, 64, 65536)
    while batch * ctx * kv_heads * dim * _SIZE[dtype] > 3e8:
        batch, ctx = max(1, batch * 2 // 3), max(64, ctx * 3 // 4)
    budget = max(8, int(ctx * rng.choice((0.05, 0.2, 0.5, 0.9))))
    recent = min(budget // 2, rng.choice((0, 16, 128)))
    return _evict(None, batch, kv_heads, dim, (ctx // rng.choice((1, 1, 4)), ctx), budget, min(4, budget - recent), recent,
                  dtype, block, again=rng.choice((True, False)))


# ------------------------------------------------------------------------------------ sizes of a case

def _between(least, most, n):
    """n whole numbers from least to most, evenly spaced."""
    return [most if n == 1 else least + (most - least) * i // (n - 1) for i in range(n)]


def _lengths(case):
    """(new rows, tokens with the new rows) of each sequence; the longest contexts have the fewest rows."""
    rows = _between(case["rows_max"], case["rows_min"], case["batch"])
    old = _between(case["old_min"], case["old_max"], case["batch"])
    return rows, [o + r for o, r in zip(old, rows)]


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "rotate":
        rows = sum(_lengths(case)[0])
        elements = rows * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": elements * (_SIZE[case["src"]] + size) + rows * 4 * case["rotary"], "flops": 10 * elements}
    if case["op"] == "weigh":
        rows, ctx = _lengths(case)
        keys = sum(ctx) * case["kv_heads"]
        seen = sum(r * c - r * (r - 1) // 2 for r, c in zip(rows, ctx)) * case["heads"]
        return {"bytes": keys * (case["dim"] * size + 8) + sum(rows) * case["heads"] * case["dim"] * size,
                "flops": 2 * seen * case["dim"]}
    lens = _between(case["ctx_min"], case["ctx_max"], case["batch"])
    moved = sum(min(case["budget"], c - case["budget"]) * (0.5 if case["again"] else case["budget"] / c)
                for c in lens if c > case["budget"])  # about: which tokens stay depends on their weights
    kept = sum(min(c, case["budget"]) for c in lens)
    return {"bytes": case["kv_heads"] * (8 * sum(lens) + 8 * kept + moved * 4 * case["dim"] * size), "flops": 0}


# ------------------------------------------------------------------------------------ inputs

def _tables(case, ctx, gen):
    """A block table of shuffled blocks, as wide as the longest context, and the number of blocks."""
    width = max(1, -(-max(ctx) // case["block"]))
    blocks = case["batch"] * width + 3
    order = torch.randperm(blocks, generator=gen, device="cuda")
    return order[: case["batch"] * width].view(case["batch"], width).contiguous(), blocks


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _starts(rows):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 11)
    dtype = _DTYPES[case["dtype"]]
    kv_heads, dim, block, batch = case["kv_heads"], case["dim"], case["block"], case["batch"]
    s = {"case": case}
    if case["op"] == "evict":
        ctx = _between(case["ctx_min"], case["ctx_max"], batch)
        ctx = [ctx[i] for i in np.random.RandomState(int(seed) % 2**31).permutation(batch)]
    else:
        rows, ctx = _lengths(case)
    s["table"], blocks = _tables(case, ctx, gen)
    s["ctx"] = torch.tensor(ctx, dtype=torch.int64, device="cuda")
    shape = (blocks, kv_heads, block, dim)
    if case["op"] == "rotate":
        src, heads, total = _DTYPES[case["src"]], case["heads"], sum(rows)
        if case["packed"]:
            qkv = _normal(gen, (total, heads + 2 * kv_heads, dim), src)
            s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        else:
            s["q"], s["k"], s["v"] = (_normal(gen, (total, n, dim), src) for n in (heads, kv_heads, kv_heads))
        s["kc"], s["vc"] = _normal(gen, shape, dtype), _normal(gen, shape, dtype)
        s["starts"] = _starts(rows)
        s["positions"] = None
        shift = [0] * batch
        if case["moved"]:
            shift = [17 * (i % 5) + 100 for i in range(batch)]
            s["positions"] = torch.cat([torch.arange(c - r, c) + d for r, c, d in zip(rows, ctx, shift)]).cuda()
        most = max(c + d for c, d in zip(ctx, shift))
        # The table a program makes once for its model, in 64 bits, rounded once.
        freq = _BASE ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])
        angle = torch.outer(torch.arange(most, dtype=torch.float64), freq)
        s["cos"], s["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
        s["qw"] = s["kw"] = None
        if case["norm"]:
            s["qw"], s["kw"] = (1 + 0.2 * torch.randn(dim, generator=gen, device="cuda") for _ in range(2))
            s["qw"], s["kw"] = s["qw"].to(src), s["kw"].to(src)
        return s
    most = s["table"].shape[1] * block
    if case["op"] == "weigh":
        # Queries of a trained model are sharper than unit normal ones against unit normal keys.
        s["q"] = _normal(gen, (sum(rows), case["heads"], dim), dtype) * 1.5
        s["kc"] = _normal(gen, shape, dtype)
        s["starts"], s["most"] = _starts(rows), max(rows)
        s["weights"] = torch.rand((batch, kv_heads, most), generator=gen, device="cuda") * 4
        s["positions"] = torch.arange(most, dtype=torch.int32, device="cuda").repeat(batch, kv_heads, 1)
        s["out"] = torch.zeros_like(s["weights"])
        return s
    s["kc"], s["vc"] = _normal(gen, shape, dtype), _normal(gen, shape, dtype)
    # Accumulated weight is heavy-tailed: few tokens hold most of it.
    s["weights"] = torch.exp(2 * _normal(gen, (batch, kv_heads, most), torch.float32) - 2)
    s["positions"] = torch.arange(most, dtype=torch.int32, device="cuda").repeat(batch, kv_heads, 1)
    if case["again"]:
        front = torch.rand((batch, kv_heads, min(most, case["budget"])), generator=gen, device="cuda").argsort(-1)
        s["positions"] += 1000
        s["positions"][..., : front.shape[-1]] = front.int()
    s["out"] = torch.zeros_like(s["weights"]), torch.zeros_like(s["positions"])
    return s


# ------------------------------------------------------------------------------------ the operators

def run(s):
    case = s["case"]
    if own:
        return _OWN[case["op"]](s, case)
    return _PLAIN[case["op"]](s, case)


def _own_rotate(s, c):
    import kyro_amd

    kv = kyro_amd.PagedKVCache(c["block"], c["kv_heads"], c["dim"])
    out = kv.append_qkv_async(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["table"], s["ctx"], cos=s["cos"], sin=s["sin"],
                              positions=s["positions"], q_weight=s["qw"], k_weight=s["kw"],
                              norm_eps=_EPS if c["norm"] else None, interleaved=c["interleaved"], q_start_loc=s["starts"])
    return out, s["kc"], s["vc"]


def _own_weigh(s, c):
    import kyro_amd

    ev = kyro_amd.CacheEviction(c["block"], c["heads"], c["dim"], c["kv_heads"])
    ev.accumulate_async(s["q"], s["kc"], s["table"], s["ctx"], s["weights"], s["positions"], q_start_loc=s["starts"],
                        max_q_len=s["most"], out=s["out"])
    return s["out"], s["positions"]


def _own_evict(s, c):
    import kyro_amd

    ev = kyro_amd.CacheEviction(c["block"], c["kv_heads"], c["dim"], c["kv_heads"])
    ctx = ev.evict_async(s["kc"], s["vc"], s["table"], s["ctx"], s["weights"], s["positions"], budget=c["budget"],
                         sink=c["sink"], recent=c["recent"], out=s["out"])
    return s["kc"], s["vc"], s["out"][0], s["out"][1], ctx


def _row_places(s):
    """(sequence, row within it) of each packed row."""
    starts = s["starts"].long()
    row = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return seq, row - starts[seq]


def _plain_rotate(s, c):
    seq, j = _row_places(s)
    starts = s["starts"].long()
    slot = s["ctx"][seq] - (starts[seq + 1] - starts[seq]) + j
    pos = slot if s["positions"] is None else s["positions"]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    n = c["rotary"]

    def norm_rotate(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.float()
        if c["interleaved"]:
            a, b = x[..., 0:n:2], x[..., 1:n:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = x[..., : n // 2], x[..., n // 2:n]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((turned, x[..., n:]), -1)

    blk, at = s["table"][seq, slot // c["block"]], slot % c["block"]
    s["kc"][blk, :, at] = norm_rotate(s["k"], s["kw"]).to(s["kc"].dtype)
    s["vc"][blk, :, at] = s["v"].to(s["vc"].dtype)
    return norm_rotate(s["q"], s["qw"]).to(s["kc"].dtype), s["kc"], s["vc"]


def _plain_weigh(s, c):
    batch, hkv, dim, most = c["batch"], c["kv_heads"], c["dim"], s["weights"].shape[-1]
    group, rows = c["heads"] // hkv, s["most"]
    starts = s["starts"].long()
    n = starts[1:] - starts[:-1]
    tok = torch.arange(most, device="cuda")
    keys = s["kc"][s["table"]].permute(0, 2, 1, 3, 4).reshape(batch, hkv, most, dim).float()
    j = torch.arange(rows, device="cuda")
    q = s["q"][(starts[:-1, None] + j).clamp(max=s["q"].shape[0] - 1)].float()
    q = q.view(batch, rows, hkv, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, hkv, group * rows, dim)
    scores = torch.matmul(q, keys.transpose(-1, -2)).view(batch, hkv, group, rows, most) * (dim ** -0.5)
    sees = (tok <= (s["ctx"] - n)[:, None, None] + j[:, None]) & (j < n[:, None])[..., None]
    sees = sees[:, None, None]
    scores = scores.masked_fill(~sees, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0))
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1)
    new = (tok >= (s["ctx"] - n)[:, None]) & (tok < s["ctx"][:, None])
    held = (tok < s["ctx"][:, None])[:, None]
    added = p.sum((2, 3)) + s["weights"].masked_fill(new[:, None], 0)
    out = torch.where(held, added, s["out"])
    pos = torch.where(new[:, None], tok.int(), s["positions"])
    return out, pos


def _plain_evict(s, c):
    batch, hkv, most = s["weights"].shape
    budget, ctx = c["budget"], s["ctx"][:, None, None]
    slot = torch.arange(most, device="cuda")
    held = slot < ctx
    pos, w = s["positions"].long(), s["weights"]
    newest = pos.masked_fill(~held, -1).amax(-1, keepdim=True)
    safe = (pos < c["sink"]) | (pos > newest - c["recent"])
    key = w.double().masked_fill(w.isnan(), -math.inf).masked_fill(safe, math.inf).masked_fill(~held, -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(held.expand(batch, hkv, most)).scatter_(
        -1, order[..., :budget], True) & held
    lens = torch.minimum(s["ctx"], torch.full_like(s["ctx"], budget))
    src = slot.expand(batch, hkv, most).clone()
    hole = (slot < budget) & ~kept & held
    late = kept & (slot >= budget)
    b, h, to = hole.nonzero(as_tuple=True)  # both in ascending order, as many of each for every head
    src[b, h, to] = late.nonzero(as_tuple=True)[2]
    frm = src[b, h, to]
    blk, at = s["table"][b, to // c["block"]], to % c["block"]
    blk2, at2 = s["table"][b, frm // c["block"]], frm % c["block"]
    s["kc"][blk, h, at] = s["kc"][blk2, h, at2]
    s["vc"][blk, h, at] = s["vc"][blk2, h, at2]
    stays = slot < lens[:, None, None]
    return (s["kc"], s["vc"], torch.where(stays, w.gather(-1, src), s["out"][0]),
            torch.where(stays, s["positions"].gather(-1, src), s["out"][1]), lens)


_OWN = {"rotate": _own_rotate, "weigh": _own_weigh, "evict": _own_evict}
_PLAIN = {"rotate": _plain_rotate, "weigh": _plain_weigh, "evict": _plain_evict}


# ------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "weigh": _exact_weigh, "evict": _exact_evict}[case["op"]](s, case)


def _exact_rotate(s, c):
    rows, ctx = _lengths(c)
    block, half = c["block"], c["rotary"] // 2
    kc, vc, table = s["kc"].double(), s["vc"].double(), s["table"].cpu()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, length) in enumerate(zip(rows, ctx)):
        mine = slice(first, first + n)
        slots = torch.arange(length - n, length)
        at = (slots if s["positions"] is None else s["positions"][mine].cpu()).cuda()
        # e^{i angle} from the same rounded table that the operator is given
        turn = torch.complex(s["cos"][at].double(), s["sin"][at].double()).unsqueeze(1)
        done = []
        for x, w in ((s["q"][mine], s["qw"]), (s["k"][mine], s["kw"])):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS) * w.double()
            re = x[..., : c["rotary"]: 2] if c["interleaved"] else x[..., :half]
            im = x[..., 1: c["rotary"]: 2] if c["interleaved"] else x[..., half: 2 * half]
            z = torch.complex(re, im) * turn
            y = x.clone()
            if c["interleaved"]:
                y[..., : c["rotary"]: 2], y[..., 1: c["rotary"]: 2] = z.real, z.imag
            else:
                y[..., :half], y[..., half: 2 * half] = z.real, z.imag
            done.append(y)
        out[mine] = done[0]
        blocks, places = table[b, slots // block].cuda(), (slots % block).cuda()
        kc[blocks, :, places] = done[1]
        vc[blocks, :, places] = s["v"][mine].double()
        first += n
    return out, kc, vc


def _exact_weigh(s, c):
    rows, ctx = _lengths(c)
    group = c["heads"] // c["kv_heads"]
    out, pos = s["out"].double(), s["positions"].clone()
    first = 0
    for b, (n, length) in enumerate(zip(rows, ctx)):
        blocks = s["table"][b, : -(-length // c["block"])]
        for h in range(c["kv_heads"]):
            keys = s["kc"][blocks, h].reshape(-1, c["dim"])[:length].double()
            q = s["q"][first:first + n, h * group:(h + 1) * group].double().reshape(n * group, c["dim"])
            p = q @ keys.T / math.sqrt(c["dim"])
            last = length - n + torch.arange(n, device="cuda").repeat_interleave(group)
            p[torch.arange(length, device="cuda") > last[:, None]] = -math.inf
            out[b, h, :length] = torch.softmax(p, -1).sum(0)
            out[b, h, : length - n] += s["weights"][b, h, : length - n].double()
            pos[b, h, length - n:length] = torch.arange(length - n, length, device="cuda").int()
        first += n
    return out, pos


def _exact_evict(s, c):
    lens = s["ctx"].tolist()
    if sum(lens) * c["kv_heads"] > 6_000_000:
        return None
    table, kc, vc = s["table"].cpu().numpy(), s["kc"].clone(), s["vc"].clone()
    out_w, out_p = s["out"][0].cpu().numpy(), s["out"][1].cpu().numpy()
    moves = []
    for b, length in enumerate(lens):
        keep = min(length, c["budget"])
        w = s["weights"][b].cpu().numpy()
        p = s["positions"][b].cpu().numpy()
        for h in range(c["kv_heads"]):
            at = np.arange(length)
            safe = (p[h, :length] < c["sink"]) | (p[h, :length] > p[h, :length].max(initial=-1) - c["recent"])
            best = np.lexsort((at, -w[h, :length], ~safe))[:keep]
            source = np.arange(keep)
            source[np.setdiff1d(source, best)] = np.sort(best[best >= keep])
            out_w[b, h, :keep], out_p[b, h, :keep] = w[h, source], p[h, source]
            to = np.flatnonzero(source != np.arange(keep))
            moves.append(np.stack([np.full(len(to), h), table[b, to // c["block"]], to % c["block"],
                                   table[b, source[to] // c["block"]], source[to] % c["block"]]))
    h, blk, at, blk2, at2 = (torch.from_numpy(x).cuda() for x in np.concatenate(moves, 1))
    kc[blk, h, at], vc[blk, h, at] = kc[blk2, h, at2], vc[blk2, h, at2]
    return kc, vc, torch.from_numpy(out_w), torch.from_numpy(out_p), np.minimum(lens, c["budget"])
