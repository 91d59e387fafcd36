"""Which calls of attention over shared prefixes take its own kernel: seen from an error that only that one finds."""
import numpy as np
import pytest
import torch

import kyro_amd
from kyro_amd import KyroError
from tests import helpers as h
from tests.test_shared_attention_gpu import check, make, reference

pytestmark = pytest.mark.gpu


def call(gpu, case, starts, blocks, width=None):
    t = h.attention_tensors(case, gpu)
    table = t["block_table"]
    if width is not None:  # wider tables, whose other entries no context reaches
        table = torch.zeros((table.shape[0], width), dtype=table.dtype, device=gpu)
        table[:, : t["block_table"].shape[1]] = t["block_table"]
    attn = kyro_amd.PagedAttention(case.block_size, case.num_heads, case.head_dim, case.num_kv_heads)
    return attn.forward_shared(t["query"], t["key_cache"], t["value_cache"], table, t["context_lens"], h.to_device(starts, gpu),
                               h.to_device(blocks, gpu), q_start_loc=t["q_start_loc"])


@pytest.mark.parametrize("name,dtype,D", [("decode", "bf16", 128), ("verify", "bf16", 64), ("verify", "f32", 96)])
def test_small_calls_leave_the_groups_unread(gpu, name, dtype, D):
    case, starts, blocks = make(name, dtype, D)
    ref = reference(case)
    check(call(gpu, case, starts, blocks), case, ref)
    check(call(gpu, case, starts[::-1].copy(), blocks), case, ref)  # out of order: an error where they are read


@pytest.mark.parametrize("name,dtype,D,width", [("decode", "bf16", 128, 9500), ("verify", "f32", 96, 9000), ("prompts", "bf16", 64, None)])
def test_wide_tables_and_prompts_are_shared(gpu, name, dtype, D, width):
    """7 x 9500 blocks of 16 tokens, 2 heads of 128 in bf16: 109 MB of K and as many of V. 6 x 9000 in f32 are 166 and 166."""
    case, starts, blocks = make(name, dtype, D)
    ref = reference(case)
    check(call(gpu, case, starts, blocks, width), case, ref)
    with pytest.raises(KyroError):
        call(gpu, case, starts[::-1].copy(), blocks, width)
    check(call(gpu, case, starts, np.zeros_like(blocks), width), case, ref)  # and the error is gone
