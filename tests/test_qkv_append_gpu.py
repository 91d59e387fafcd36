"""Head norms, rotation and paged write in one launch (PagedKVCache.append_qkv) against the formulas in
64 bits, at the sizes, strides and layouts where the pass can go wrong."""
import numpy as np
import pytest
import torch

import kyro_amd

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
# Roundings of a query or key element before the store, in steps of 2^-24 of |n cos| + |n' sin|: at most 22 adds
# of the mean square (16 in a lane, 6 between lanes) and its products halved by the root, 11.5; division by D, the
# addition of eps, root and reciprocal 3; times rstd, weight (its offset and product) 3; the turn's two products
# and their sum 2. 24 covers the 19.5.
STEPS = 24


def setup(gpu, *, B=5, rows=(3, 1, 0, 9, 2), old=(0, 15, 4, 30, 100), H=8, hkv=2, D=64, bs=16, src=BF16, dst=BF16,
          packed=True, extra_rows=0, seed=0, pos=None, rot=None, norm=True, wdt=None, interleaved=False):
    g = torch.Generator().manual_seed(seed)
    rows, old = np.asarray(rows), np.asarray(old)
    ctx = rows + old
    width = int(max(1, -(-ctx.max() // bs)))
    nb = B * width + 2
    table = torch.randperm(nb, generator=g)[: B * width].view(B, width)
    total = int(rows.sum()) + extra_rows
    make = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    if packed:
        qkv = make(total, H + 2 * hkv, D).to(src).to(gpu)
        q, k, v = qkv[:, :H], qkv[:, H:H + hkv], qkv[:, H + hkv:]
    else:
        q, k, v = (make(total, n, D).to(src).to(gpu) for n in (H, hkv, hkv))
    c = dict(query=q, key=k, value=v, key_cache=make(nb, hkv, bs, D).to(dst).to(gpu),
             value_cache=make(nb, hkv, bs, D).to(dst).to(gpu), block_table=table.to(gpu),
             context_lens=torch.from_numpy(ctx).to(gpu),
             q_start_loc=torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device=gpu))
    rot = D if rot is None else rot
    if rot:
        c["cos"], c["sin"] = kyro_amd.rope_tables(1000, rot, device=gpu)
        c["interleaved"] = interleaved
    if pos is not None:
        c["positions"] = torch.randint(0, 1000, (total,), generator=g).to(gpu)
    if norm:
        c["norm_eps"] = 1e-5
        if wdt is not None:
            c["q_weight"], c["k_weight"] = (1 + 0.3 * make(D)).to(wdt).to(gpu), (1 + 0.3 * make(D)).to(wdt).to(gpu)
            c["weight_offset"] = 0.25
    return c


def expected(c):
    """(query, key cache, value cache) in 64 bits, and how far a right answer may be from each."""
    q, k, v = (c[n].double().cpu() for n in ("query", "key", "value"))
    kc, vc = c["key_cache"].double().cpu(), c["value_cache"].double().cpu()
    half_step = torch.finfo(c["key_cache"].dtype).eps / 2
    starts, ctx, table = c["q_start_loc"].tolist(), c["context_lens"].tolist(), c["block_table"].cpu()
    bs = kc.shape[2]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    ktol, vtol = torch.zeros_like(kc), torch.zeros_like(vc)
    for b in range(len(ctx)):
        n = starts[b + 1] - starts[b]
        for j in range(n):
            r, p = starts[b] + j, ctx[b] - n + j
            at = int(c["positions"][r]) if c.get("positions") is not None else p
            blk = int(table[b, p // bs])
            for x, w, store in ((q[r], "q_weight", "q"), (k[r], "k_weight", "k")):
                x = x.clone()
                if "norm_eps" in c:
                    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + float(np.float32(c["norm_eps"])))
                    if c.get(w) is not None:
                        x = x * (c[w].double().cpu() + c["weight_offset"])
                err = x.abs() * STEPS * U
                if "cos" in c:
                    cs, sn = c["cos"][at].double().cpu(), c["sin"][at].double().cpu()
                    m = 2 * len(cs)
                    i, i2 = (slice(0, m, 2), slice(1, m, 2)) if c["interleaved"] else (slice(0, m // 2), slice(m // 2, m))
                    a, d = x[:, i].clone(), x[:, i2].clone()
                    x[:, i], x[:, i2] = a * cs - d * sn, d * cs + a * sn
                    err[:, i] = STEPS * U * ((a * cs).abs() + (d * sn).abs())
                    err[:, i2] = STEPS * U * ((d * cs).abs() + (a * sn).abs())
                bound = err + half_step * (x.abs() + err) + 1e-40
                if store == "q":
                    out[r], tol[r] = x, bound
                else:
                    kc[blk, :, p % bs], ktol[blk, :, p % bs] = x, bound
            vc[blk, :, p % bs] = v[r].to(c["value_cache"].dtype).double()
    return (out, tol), (kc, ktol), (vc, vtol)


def check(c, **more):
    want = expected(c)
    covered = int(c["q_start_loc"][-1])
    kv = kyro_amd.PagedKVCache(c["key_cache"].shape[2], c["key"].shape[1], c["key"].shape[2])
    out = kv.append_qkv(**c, **more)
    assert out.dtype == c["key_cache"].dtype
    for name, got, (ref, tol) in zip(("query", "key cache", "value cache"), (out, c["key_cache"], c["value_cache"]), want):
        if name == "query":
            got, ref, tol = got[:covered], ref[:covered], tol[:covered]
        off = (got.double().cpu() - ref).abs() - tol
        assert not off.isnan().any() and (off <= 0).all(), f"{name}: {off.max():.3g} past its bound"
    return out


@pytest.mark.parametrize("src,dst", [(BF16, BF16), (F32, F32), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("D,rot,interleaved", [(128, 128, False), (64, 32, False), (80, 80, False), (96, 48, True),
                                               (72, 72, False), (40, 20, False), (256, 256, False), (256, 20, False),
                                               (8, 8, False), (16, 6, True), (112, 0, False), (24, 24, True),
                                               (72, 70, True), (200, 196, False)])
def test_against_64_bits(gpu, src, dst, D, rot, interleaved):
    check(setup(gpu, D=D, rot=rot, interleaved=interleaved, src=src, dst=dst, wdt=src, seed=D + rot))


@pytest.mark.parametrize("norm,wdt", [(False, None), (True, None), (True, F32), (True, BF16)])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("pos", [None, True])
def test_norm_strides_positions(gpu, norm, wdt, packed, pos):
    check(setup(gpu, norm=norm, wdt=wdt, packed=packed, pos=pos, bs=8, H=6, hkv=6, seed=3))


@pytest.mark.parametrize("B,H,hkv", [(1, 1, 1), (1, 32, 8), (64, 4, 1), (65, 4, 2), (200, 3, 1), (4200, 1, 1)])
def test_batches(gpu, B, H, hkv):
    """The search of a row's sequence over one probe, several, and sequences without rows between."""
    g = np.random.default_rng(B)
    rows = g.integers(0, 4, B)
    rows[-1] = 1
    check(setup(gpu, B=B, rows=rows, old=g.integers(0, 20, B), H=H, hkv=hkv, D=16, bs=16, seed=B))


def test_one_row_per_sequence_without_q_start(gpu):
    c = setup(gpu, B=7, rows=[1] * 7, old=range(10, 17))
    d = {k: v.clone() if k.endswith("cache") else v for k, v in c.items() if k != "q_start_loc"}
    out = check(c)
    again = kyro_amd.PagedKVCache(16, 2, 64).append_qkv(**d)
    assert torch.equal(out, again) and torch.equal(c["key_cache"], d["key_cache"])


def test_rows_behind_the_last_sequence_stay(gpu):
    c = setup(gpu, extra_rows=4)
    out = torch.full(c["query"].shape, 7.0, dtype=BF16, device=gpu)
    check(c, out=out)
    assert (out[-4:] == 7).all()


def test_query_rotated_in_place(gpu):
    c = setup(gpu, packed=False)
    d = {k: v.clone() if torch.is_tensor(v) else v for k, v in c.items()}
    want = check(c)
    got = kyro_amd.PagedKVCache(16, 2, 64).append_qkv(**d, out=d["query"])
    assert got.data_ptr() == d["query"].data_ptr() and torch.equal(got, want)


def test_values_keep_their_bits_and_odd_numbers_pass(gpu):
    """NaN payloads, infinities, subnormals and zeros of a value row; a head of zeros under the norm is zeros."""
    c = setup(gpu, B=1, rows=[1], old=[0], packed=False, D=16, bs=4, H=2, hkv=2)
    bits = torch.tensor([0x7FC1, 0xFFA5, 0x7F80, 0xFF80, 1, 0x8001, 0x8000, 0] * 2, dtype=torch.int32).to(torch.int16)
    c["value"][0, :] = bits.view(BF16).to(gpu)
    c["query"][0, 0] = 0
    out = kyro_amd.PagedKVCache(4, 2, 16).append_qkv(**c)
    blk = int(c["block_table"][0, 0])
    assert torch.equal(c["value_cache"][blk, 1, 0].view(torch.int16).cpu(), bits)
    assert (out[0, 0] == 0).all() and out[0, 1].isfinite().all()


def test_append_then_attend(gpu):
    """Norm, rotation, append and attention in a row equal attention over 64-bit keys of the same formulas."""
    c = setup(gpu, B=3, rows=[4, 1, 20], old=[0, 33, 5], D=128, H=8, hkv=2, src=F32, dst=F32, wdt=F32)
    out = check(c)
    got = kyro_amd.PagedAttention(16, 8, 128, 2).forward(out, c["key_cache"], c["value_cache"], c["block_table"],
                                                         c["context_lens"], q_start_loc=c["q_start_loc"])
    starts = c["q_start_loc"].tolist()
    for b, n in enumerate(c["context_lens"].tolist()):
        kd, vd = (c[x][c["block_table"][b]].transpose(0, 1).reshape(2, -1, 128)[:, :n].double() for x in ("key_cache", "value_cache"))
        r0, r1 = starts[b], starts[b + 1]
        q = out[r0:r1].double()
        for h in range(8):
            s = q[:, h] @ kd[h // 4].T / 128 ** 0.5
            s[torch.arange(n, device=gpu) > n - (r1 - r0) + torch.arange(r1 - r0, device=gpu)[:, None]] = -float("inf")
            ref = torch.softmax(s, -1) @ vd[h // 4]
            # tests' bound for f32 attention outputs
            assert (got[r0:r1, h].double() - ref).abs().max() < 1e-3


def test_bad_rows_are_reported_and_not_written(gpu):
    for what in ("position", "block", "context", "layout"):
        c = setup(gpu, pos=True, seed=9)
        if what == "position":
            c["positions"][1] = 1000
            c["positions"][3] = -1
            bad = [1, 3]
        elif what == "block":
            c["block_table"][1, 0] = c["key_cache"].shape[0]
            bad = [3]
        elif what == "context":
            c["context_lens"][3] = 8  # nine new rows
            bad = list(range(4, 13))
        else:
            c["q_start_loc"][5] = 99
            bad = [13, 14]
        old_k = c["key_cache"].clone()
        out = torch.full(c["query"].shape, 7.0, dtype=BF16, device=gpu)
        kv = kyro_amd.PagedKVCache(16, 2, 64)
        with pytest.raises(kyro_amd.KyroError, match={"position": "position", "block": "block_table", "context": "context length",
                                                      "layout": "q_start_loc"}[what]):
            kv.append_qkv(**c, out=out)
        wrote = (out != 7).flatten(1).any(1).cpu()
        assert wrote.tolist() == [r not in bad for r in range(15)], what
        changed = (c["key_cache"] != old_k).any(-1).any(1).sum().item()
        assert changed == 15 - len(bad), what
        kyro_amd.sync()  # the error was handed out once


def test_refused_tensors(gpu):
    c = setup(gpu, wdt=F32)
    kv = kyro_amd.PagedKVCache(16, 2, 64)

    def refused(error, **change):
        with pytest.raises(error):
            kv.append_qkv(**{**c, **change})

    refused(TypeError, query=c["query"].half())
    refused(TypeError, key=c["key"].float())
    refused(ValueError, key=c["key"][:, :1])
    refused(ValueError, query=c["query"].transpose(1, 2).contiguous().transpose(1, 2))
    refused(ValueError, cos=c["cos"][:, :8])
    refused(ValueError, sin=None)
    refused(ValueError, positions=torch.zeros(3, dtype=torch.int64, device=gpu))
    refused(TypeError, positions=torch.zeros(15, dtype=torch.int32, device=gpu))
    refused(ValueError, k_weight=None)
    refused(ValueError, norm_eps=None)
    refused(ValueError, q_start_loc=None)
    refused(ValueError, value=c["value"].cpu())
    refused(ValueError, out=torch.empty((15, 8, 32), dtype=BF16, device=gpu))
    refused(kyro_amd.KyroError, query=torch.empty(15 * 512 + 4, dtype=BF16, device=gpu)[4:].view(15, 8, 64))  # 8 bytes off
    refused(kyro_amd.KyroError, out=c["query"].as_strided((15, 8, 64), (512, 64, 1)))  # inside the packed rows
    check(c)


def test_graph_replays_and_streams(gpu):
    c = setup(gpu, wdt=BF16, pos=True)
    kv = kyro_amd.PagedKVCache(16, 2, 64)
    start = c["key_cache"].clone(), c["value_cache"].clone()
    out = torch.empty(c["query"].shape, dtype=BF16, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv.append_qkv_async(**c, out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kv.append_qkv_async(**c, out=out)
    torch.cuda.current_stream().wait_stream(side)
    for turn in range(3):
        c["query"].copy_(torch.randn(c["query"].shape, device=gpu))
        c["positions"].copy_(torch.randint(0, 1000, (15,), device=gpu))
        c["key_cache"].copy_(start[0]), c["value_cache"].copy_(start[1])
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        d = dict(c, key_cache=start[0].clone(), value_cache=start[1].clone())
        want = check(d)
        assert torch.equal(out, want) and torch.equal(c["key_cache"], d["key_cache"])


def test_cache_past_32_bits(gpu):
    """Slots past element 2^32 of a cache."""
    nb = 2 ** 32 // (8 * 16 * 128) + 3
    kc, vc = (torch.empty((nb, 8, 16, 128), dtype=BF16, device=gpu) for _ in range(2))
    c = setup(gpu, B=2, rows=[1, 17], old=[0, 3], H=8, hkv=8, D=128)
    small = c["key_cache"].shape[0]
    shift = nb - small
    kc[shift:], vc[shift:] = c["key_cache"], c["value_cache"]
    kc[:small], vc[:small] = c["key_cache"], c["value_cache"]
    out = kyro_amd.PagedKVCache(16, 8, 128).append_qkv(**dict(c, key_cache=kc, value_cache=vc, block_table=c["block_table"] + shift))
    keep = c["key_cache"].clone(), c["value_cache"].clone()
    want = check(c)
    assert torch.equal(out, want)
    assert torch.equal(kc[shift:], c["key_cache"]) and torch.equal(vc[shift:], c["value_cache"])
    assert torch.equal(kc[:small], keep[0]) and torch.equal(vc[:small], keep[1])
