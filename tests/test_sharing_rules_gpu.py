"""Attention over shared prefixes as callers get it, with the library's own rules for which calls take its kernel and which
groups share: the shapes of the kernel's tests on tables wide enough, against attention in 64 bits."""
import numpy as np
import pytest
import torch

import kyro_amd
from kyro_amd import KyroError, workloads as wl
from tests import helpers as h
from tests.test_shared_attention_gpu import SHAPES, check, make, reference

pytestmark = pytest.mark.gpu


def wide_enough(case):
    """Blocks of a table row with which the call's tables could name 520 MiB of K and V."""
    block = 2 * case.num_kv_heads * case.block_size * case.head_dim * (2 if case.dtype == "bf16" else 4)
    return -(-520 * 2 ** 20 // (block * case.batch))


def call(gpu, t, case, starts, blocks, **kw):
    attn = kyro_amd.PagedAttention(case.block_size, case.num_heads, case.head_dim, case.num_kv_heads)
    return attn.forward_shared(t["query"], t["key_cache"], t["value_cache"], t["block_table"], t["context_lens"],
                               h.to_device(starts, gpu), h.to_device(blocks, gpu), q_start_loc=t["q_start_loc"], **kw)


def tensors(gpu, case):
    t = h.attention_tensors(case, gpu)
    table = torch.zeros((case.batch, max(wide_enough(case), t["block_table"].shape[1])), dtype=torch.int64, device=gpu)
    table[:, : t["block_table"].shape[1]] = t["block_table"]
    return dict(t, block_table=table)


@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("bf16", 96), ("bf16", 128), ("bf16", 256), ("f32", 64), ("f32", 112), ("f32", 128)],
                         ids=lambda x: str(x))
@pytest.mark.parametrize("name", sorted(SHAPES))
def test_parity_under_the_library_s_rules(gpu, name, dtype, D):
    """Some groups share and some are not worth it; that the kernel has the call shows in the error for groups out of order."""
    case, starts, blocks = make(name, dtype, D, seed=11)
    ref = reference(case)
    t = tensors(gpu, case)
    check(call(gpu, t, case, starts, blocks), case, ref)
    with pytest.raises(KyroError, match="group_starts"):
        call(gpu, t, case, starts[::-1].copy(), blocks)
    check(call(gpu, t, case, starts, blocks, out_dtype=torch.bfloat16), case, ref)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 96)])
def test_many_sequences_of_many_groups(gpu, dtype, D):
    """More than 256 sequences (the plan for any batch), groups of 1 to 9 with 0 to 700 tokens in common."""
    rng = np.random.default_rng(D)
    sizes = [int(x) for x in rng.integers(1, 10, 70)]
    starts = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    blocks = rng.integers(0, 45, 70).astype(np.int32)
    rows = rng.integers(0, 5, starts[-1])
    ctx = [int(blocks[g]) * 16 + int(rng.integers(0, 60)) + int(rows[b])
           for g, n in enumerate(sizes) for b in range(starts[g], starts[g + 1])]
    case = wl.make_attention_case(context_lens=ctx, q_lens=[int(x) for x in rows], num_heads=4, num_kv_heads=2,
                                  head_dim=D, block_size=16, dtype=dtype, seed=D)
    for g, nb in enumerate(blocks):
        case.block_table[starts[g]:starts[g + 1], :nb] = case.block_table[starts[g], :nb]
    assert case.batch > 256
    t = tensors(gpu, case)
    check(call(gpu, t, case, starts, blocks), case, reference(case))
