"""The attention weights of the paged decode, where their precision shows: a few slots that outweigh the rest of a lane, values that cancel."""
import os
import sys

import pytest
import torch

import tatara_b200 as tb

sys.path.insert(0, os.path.dirname(__file__))
from paged_util import Cache, U  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = tb.Context(0)
    yield c
    c.close()


def decode(ctx, c, q, scale):
    h = tb.paged_cache(c.keys, c.values, c.table, mass=c.mass, positions=c.positions)
    out = torch.full_like(q, 7.0)
    need = tb.decode_paged_scratch_bytes(h, len(c.lens), min(h.capacity, tb.MAX_CONTEXT), q.shape[1])
    ctx.attn_decode_paged(h, c.lanes, q, None, out, torch.full((need // 4 + 1,), float("nan"), device="cuda"), scale=scale)
    ctx.sync()
    return out


def definition(c, q, scale, lost, least):
    """out, its bound, the weights added to the mass and their bound, in 64 bits, for weights that lose `lost` of themselves and at most `least`
    of the largest one before the product with V.

    Beside that: the result is rounded once (half a step, 2^-25 at least); the scores are f32 sums of dim products, each term off by at
    most (dim + 2) 2^-24 of sum |q k| scale, which the exponential turns into that relative error of a weight, in the numerator and in
    the sum; sums over n slots run over at most n / 64 + 80 additions; exp2 and the division add a few last places (2^-20)."""
    u, dim = U[q.dtype], q.shape[2]
    heads = c.keys.shape[1]
    group = q.shape[1] // heads
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    added, added_bound = (torch.zeros(c.mass.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for lane, n in enumerate(c.lanes[:, 0].tolist()):
        for head in range(heads):
            k, v = (c.rows(x, lane, head, n).double() for x in (c.keys, c.values))
            of = slice(head * group, (head + 1) * group)
            x = q[lane, of].double()
            p = torch.softmax(x @ k.T * scale, dim=-1)
            slack = 2 * (dim + 2) * 2.0 ** -24 * float((x.abs() @ k.abs().T).max()) * abs(scale) + (n / 64 + 80) * 2.0 ** -24 + 2.0 ** -20
            o = p @ v
            out[lane, of] = o
            bound[lane, of] = u * o.abs() + (lost + slack) * (p @ v.abs()) + least * v.abs().sum(dim=0) + 2.0 ** -25
            added[lane, head, :n] = p.sum(dim=0)
            added_bound[lane, head, :n] = slack * p.sum(dim=0) + 2.0 ** -126
    return out, bound, added, added_bound


@pytest.mark.parametrize("kv_heads,group,dim,lens", [(2, 8, 256, [100, 700, 17]), (1, 16, 256, [1000]), (8, 4, 128, [5003]), (2, 12, 128, [300, 64]),
                                                     (1, 1, 64, [262144]), (200, 1, 64, [20000]), (3, 16, 64, [3000, 33])])
def test_f16_slots_far_below_one_that_dominates(ctx, kv_heads, group, dim, lens):
    """One slot 17.4 above all others, with values of zero: the output is what the others hold, 2.8e-8 of the largest weight each.  The
    weights are rounded to f16 (2^-11 each, and 2^-39 of the largest, where f16 has no normal step left)."""
    c = Cache(lens, kv_heads, dim, dtype=torch.float16, page=64, seed=dim + group)
    q = torch.zeros((len(lens), kv_heads * group, dim), dtype=torch.float16, device="cuda")
    q[:, :, 3] = 1.0
    c.keys[..., 3] = torch.where(torch.isnan(c.keys[..., 3]), c.keys[..., 3], 0.0)
    for lane, n in enumerate(lens):
        slot = (7 * n) // 11
        at = (int(c.table[lane, slot // 64]), slice(None), slot % 64)
        c.keys[at + (3,)] = 17.4
        c.values[at] = 0.0
    c.values.abs_()
    want, bound, added, added_bound = definition(c, q, 1.0, 2.0 ** -11, 2.0 ** -39)
    before = c.mass.double()
    out = decode(ctx, c, q, 1.0)
    assert ((out.double() - want).abs() <= bound).all()
    assert ((c.mass.double() - before - added).abs() <= added_bound + 2.0 ** -24 * (before + added)).all()


def test_f16_scores_whose_size_leaves_no_room(ctx):
    """Scores near 5e8, where an f32 step is 32 or more: equal ones share the weight, and the factor that f16 weights carry is no part of them."""
    c = Cache([50], 1, 64, dtype=torch.float16, seed=5)
    q = torch.full((1, 4, 64), 8000.0, dtype=torch.float16, device="cuda")
    c.keys.copy_(torch.where(torch.isnan(c.keys), c.keys, 1000.0))
    before = c.mass.double()
    out = decode(ctx, c, q, 1.0)
    mean = c.rows(c.values, 0, 0, 50).double().mean(dim=0)
    assert ((out[0].double() - mean).abs() <= 2.0 ** -11 * mean.abs() + 2.0 ** -17 * c.rows(c.values, 0, 0, 50).double().abs().mean(dim=0) + 2.0 ** -25).all()
    assert ((c.mass.double() - before)[0, 0, :50] - 4 / 50).abs().max() <= 2.0 ** -20


# A weight is the sum of two numbers of the type: the second is off by half a step of what the first leaves, a step and 2^-12 of the weight at most.
LOST = {t: u * (2 * u + 2.0 ** -12) for t, u in U.items()}
LEAST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -39}      # f16: half of its smallest step, for weights up to 2^14
LAYOUTS = [(2, 8, 256, 16), (1, 16, 256, 48), (8, 4, 128, 16), (2, 11, 128, 64), (12, 1, 64, 32), (2, 16, 64, 16), (3, 5, 64, 112)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv_heads,group,dim,page", LAYOUTS)
def test_values_that_cancel(ctx, dtype, kv_heads, group, dim, page):
    """Slots 2i and 2i + 1 hold nearly the same key and opposite values: what is left of the sum is the difference of two weights."""
    lens = [2, 40, 130, 1000, 4000]
    c = Cache(lens, kv_heads, dim, dtype=dtype, page=page, seed=page + dim)
    for lane, n in enumerate(lens):
        s = torch.arange(0, n, 2, device="cuda")
        pair = [(c.table[lane, x // page].long(), slice(None), x % page) for x in (s, s + 1)]
        c.values[pair[1]] = -c.values[pair[0]]
        c.keys[pair[1]] = c.keys[pair[0]]
        c.keys[pair[1] + (5,)] *= 0.9
    q = (0.2 * torch.randn((len(lens), kv_heads * group, dim), generator=c.gen, device="cuda")).to(dtype)
    scale = dim ** -0.5
    want, bound, added, added_bound = definition(c, q, scale, LOST[dtype], LEAST[dtype])
    before = c.mass.double()
    out = decode(ctx, c, q, scale)
    assert ((out.double() - want).abs() <= bound).all()
    assert ((c.mass.double() - before - added).abs() <= added_bound + 2.0 ** -24 * (before + added)).all()


@pytest.mark.parametrize("kv_heads,group,dim,lens", [(2, 8, 256, [100, 700, 17]), (8, 4, 128, [5003]), (1, 1, 64, [262144]), (3, 16, 64, [3000, 33])])
def test_f16_slots_far_below_lose_hardly_anything(ctx, kv_heads, group, dim, lens):
    """As above, held to what two numbers of the type lose, the slots at every distance from the one that dominates."""
    c = Cache(lens, kv_heads, dim, dtype=torch.float16, page=64, seed=dim + group)
    q = torch.zeros((len(lens), kv_heads * group, dim), dtype=torch.float16, device="cuda")
    q[:, :, 3] = 1.0
    spread = 22 * torch.rand(c.keys.shape[:-1], generator=c.gen, device="cuda")
    c.keys[..., 3] = torch.where(torch.isnan(c.keys[..., 3]), float("nan"), spread).half()
    for lane, n in enumerate(lens):
        c.values[int(c.table[lane, (n // 2) // 64]), :, (n // 2) % 64] = 0.0
        c.keys[int(c.table[lane, (n // 2) // 64]), :, (n // 2) % 64, 3] = 30.0
    want, bound, _, _ = definition(c, q, 1.0, LOST[torch.float16], LEAST[torch.float16])
    assert ((decode(ctx, c, q, 1.0).double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv_heads,group,dim,page", LAYOUTS)
def test_infinite_values_stay_infinite(ctx, dtype, kv_heads, group, dim, page):
    """A value that overflowed makes its dim infinite, with its sign, wherever its slot lies, the largest weight's and a lane's only one included."""
    lens = [1, 60, 700]
    c = Cache(lens, kv_heads, dim, dtype=dtype, page=page, seed=page)
    q = (0.3 * torch.randn((len(lens), kv_heads * group, dim), generator=c.gen, device="cuda")).to(dtype)
    plain = decode(ctx, c.clone(), q, dim ** -0.5)
    for lane, n in enumerate(lens):
        for i, slot in enumerate({0, n // 2, n - 1}):
            c.values[int(c.table[lane, slot // page]), :, slot % page, 7 * i] = float("inf")
            c.values[int(c.table[lane, slot // page]), :, slot % page, 7 * i + 1] = -float("inf")
    out = decode(ctx, c, q, dim ** -0.5)
    for lane, n in enumerate(lens):
        dims = [7 * i for i in range(len({0, n // 2, n - 1}))]
        assert (out[lane][:, dims] == float("inf")).all() and (out[lane][:, [d + 1 for d in dims]] == -float("inf")).all()
        rest = [d for d in range(dim) if d not in dims and d - 1 not in dims]
        assert torch.equal(out[lane][:, rest], plain[lane][:, rest])
