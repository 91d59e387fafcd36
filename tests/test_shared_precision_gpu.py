"""Attention over shared prefixes in f32: sums as exact as those of attention over each sequence by itself."""
import pytest
import torch

import kyro_amd

pytestmark = pytest.mark.gpu

BS = 16
# (heads, kv heads, sequences, rows of each, blocks in common, blocks of each sequence's own)
SHAPES = {
    "decode": (16, 8, 160, 1, 20, 5),
    "verify": (14, 2, 48, 5, 24, 7),
    "prompts": (16, 4, 6, 80, 10, 20),
}


@pytest.mark.parametrize("D", [64, 80, 96, 112])
@pytest.mark.parametrize("name", sorted(SHAPES))
def test_f32_error_against_64_bits_is_the_vector_kernels(gpu, name, D):
    """The vector kernel adds up in trees. The same 32-bit operations in chains no deeper give the same error up to
    sampling: the ratio of two error norms over 2500 rows or more scatters by 0.5 / sqrt(2500) of a row's own scatter,
    which is about its size, so by 1 to 2 %, and a few operations more or fewer move it by 2. Two chains a score and
    one a tile's output instead are 1.2 to 1.4."""
    H, Hkv, B, n, common, own = SHAPES[name]
    gen = torch.Generator().manual_seed(D + B)
    blocks, ctx = common + own, (common + own) * BS - 3
    table = torch.randperm(B * blocks, generator=gen).view(B, blocks)
    table[:, :common] = table[0, :common].clone()
    kc, vc = (torch.randn((B * blocks, Hkv, BS, D), generator=gen) for _ in range(2))
    q = torch.randn((B * n, H, D), generator=gen)
    exact = torch.empty(q.shape, dtype=torch.float64)
    seen = torch.arange(ctx) <= ctx - n + torch.arange(n)[:, None]
    for b in range(B):
        k, v = (x[table[b]].transpose(0, 1).reshape(Hkv, -1, D)[:, :ctx].double() for x in (kc, vc))
        x = q[b * n:(b + 1) * n].double().view(n, Hkv, H // Hkv, D).permute(1, 2, 0, 3).reshape(Hkv, -1, D)
        s = (torch.matmul(x, k.transpose(1, 2)) / D ** 0.5).view(Hkv, H // Hkv, n, ctx).masked_fill(~seen, float("-inf"))
        p = torch.softmax(s, -1).view(Hkv, -1, ctx)
        exact[b * n:(b + 1) * n] = torch.matmul(p, v).view(Hkv, H // Hkv, n, D).permute(2, 0, 1, 3).reshape(n, H, D)
    attn = kyro_amd.PagedAttention(BS, H, D, Hkv)
    args = [x.to(gpu) for x in (q, kc, vc, table, torch.full((B,), ctx))]
    starts = torch.arange(0, B * n + 1, n, dtype=torch.int32, device=gpu)
    groups = torch.tensor([0, B], dtype=torch.int32, device=gpu), torch.tensor([common], dtype=torch.int32, device=gpu)
    err = {"shared": attn.forward_shared(*args, *groups, q_start_loc=starts, max_q_len=n),
           "vector": attn.forward(*args, q_start_loc=starts, max_q_len=n, path="vector")}
    err = {x: float((y.cpu().double() - exact).norm() / exact.norm()) for x, y in err.items()}
    assert err["shared"] <= 1.08 * err["vector"], err
