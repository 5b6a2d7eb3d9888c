"""Paged decode with so many partitions for a CTA that it describes them in several goes, of lanes that leave some warps without a share for long runs."""
import pytest
import torch

import tatara_b200 as tb

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = tb.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("kv_heads,group,dim,lens", [
    (192, 1, 256, [16] * 128 + [100] * 128), (200, 2, 256, [16, 0, 9, 1] * 40 + [300] * 40 + [33, 64] * 28), (512, 1, 128, [16] * 200 + [200] * 56),
    (400, 1, 64, [16] * 200 + [200] * 56), (1000, 1, 64, ([12] * 60 + [129, 16, 65, 40]) * 4), (300, 9, 128, [16] * 180 + [300] * 76)])
@pytest.mark.parametrize("mass", [False, True])
def test_warps_without_a_share_for_long_runs(ctx, kv_heads, group, dim, lens, mass):
    """In calls of eight lanes a CTA has few partitions, all described at once; the batch has the same bits."""
    gen = torch.Generator(device="cuda").manual_seed(kv_heads)
    page, lanes = 16, len(lens)
    columns = -(-max(lens) // page)
    used = [-(-n // page) for n in lens]
    pages = sum(used) + 1
    pools = [torch.empty((pages, kv_heads, page, dim), dtype=torch.bfloat16, device="cuda").normal_(generator=gen) for _ in range(2)]
    order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
    table = torch.full((lanes, columns), -1, dtype=torch.int32, device="cuda")
    at = 0
    for lane, k in enumerate(used):
        table[lane, :k] = order[at: at + k]
        at += k
    state = torch.tensor([[n, max(0, n - 1)] for n in lens], dtype=torch.int32, device="cuda")
    q = torch.randn((lanes, kv_heads * group, dim), generator=gen, device="cuda").to(torch.bfloat16)

    def attend(part):
        weights = torch.zeros((len(lens[part]), kv_heads, columns * page), device="cuda") if mass else None
        h = tb.paged_cache(*pools, table[part].contiguous(), mass=weights)
        out = torch.full_like(q[part], 7.0)
        need = tb.decode_paged_scratch_bytes(h, len(lens[part]), h.capacity, q.shape[1])
        ctx.attn_decode_paged(h, state[part].contiguous(), q[part], None, out, torch.empty(need, dtype=torch.uint8, device="cuda"))
        ctx.sync()
        return out, weights

    out, weights = attend(slice(0, lanes))
    for i in range(0, lanes, 8):
        part = slice(i, i + 8)
        got, its = attend(part)
        assert torch.equal(got, out[part])
        if mass:
            assert torch.equal(its, weights[part])
            live = [j for j in range(i, i + 8) if lens[j]]
            # a head's weights sum up to 1: two sums of up to 300 f32 numbers in a tree, exponentials and quotients of a few last places
            assert (weights[live].sum(dim=2) - group).abs().max() <= group * 2.0 ** -16
    # against 64 bits, a lane of each length: half a step of the result; weights off by 2^-14.9 as the product takes them, and by twice the
    # (dim + 2) 2^-24 of a score's terms, which add up to less than 30 here: 2^-9 in all
    for lane in {n: i for i, n in enumerate(lens) if n}.values():
        s = torch.arange(lens[lane], device="cuda")
        k, v = (x[table[lane, s // page].long(), :, s % page].double().transpose(0, 1) for x in pools)       # [head][slot][dim]
        w = torch.softmax(q[lane].double().view(kv_heads, group, dim) @ k.transpose(1, 2) * dim ** -0.5, dim=-1)
        want, size = (w @ v).reshape(-1, dim), (w @ v.abs()).reshape(-1, dim)
        assert ((out[lane].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -9 * size).all()
