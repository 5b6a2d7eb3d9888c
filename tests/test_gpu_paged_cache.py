"""Paged KV cache operators on the device, against their 64-bit definitions (tests/paged_util.py)."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import tatara_b200 as tb
from tatara_b200 import synthetic as syn

sys.path.insert(0, os.path.dirname(__file__))
from gpu_util import dev_bf16  # noqa: E402
from paged_util import Cache, decode_definition, evict_definition, same, same_cache  # noqa: E402

pytestmark = pytest.mark.gpu

RANGE = tb.STATUS_NAMES.index("ContextOutOfRange")


@pytest.fixture(scope="module")
def ctx():
    c = tb.Context(0)
    yield c
    c.close()


def handle(c, mass=True, positions=True):
    return tb.paged_cache(c.keys, c.values, c.table, mass=c.mass if mass else None, positions=c.positions if positions else None)


def query(c, q_heads, warmth=1.5):
    shape = (len(c.lens), q_heads, c.keys.shape[3])
    q = (warmth * torch.randn(shape, generator=c.gen, device="cuda")).to(c.keys.dtype)
    return q, torch.randn(shape, generator=c.gen, device="cuda").to(c.keys.dtype)


def scratch_for(h, lanes, max_keys, q_heads):
    # not-a-number: whatever is read before it was written shows
    n = tb.decode_paged_scratch_bytes(h, lanes, max_keys, q_heads)
    return torch.full((n // 4 + 1,), float("nan"), device="cuda")


def decode(ctx, c, q, gate, mass=True, max_keys=None, stream=None, **kw):
    h = handle(c, mass=mass)
    out = torch.full_like(q, 7.0)
    most = h.capacity if max_keys is None else max_keys
    ctx.attn_decode_paged(h, c.lanes, q, gate, out, scratch_for(h, len(c.lens), most, q.shape[1]), max_keys=most, stream=stream, **kw)
    ctx.sync(stream)
    return out


# ---- decode ------------------------------------------------------------------------------------------------------------

LENGTHS = [0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 500, 1025]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv_heads,group,dim,page,slot_major", [
    (2, 8, 256, 16, False), (2, 8, 256, 64, True), (1, 16, 256, 48, False), (3, 1, 256, 16, True), (2, 5, 256, 1024, False),
    (8, 4, 128, 16, True), (1, 9, 128, 32, False), (5, 8, 128, 80, True), (12, 1, 64, 32, True), (2, 16, 64, 16, False), (3, 7, 64, 112, False)])
def test_decode_and_mass_match_the_definition(ctx, dtype, kv_heads, group, dim, page, slot_major):
    c = Cache(LENGTHS, kv_heads, dim, dtype=dtype, page=page, slot_major=slot_major, seed=kv_heads * dim + group)
    q, gate = query(c, kv_heads * group)
    for g, scale in ((gate, dim ** -0.5), (None, 0.11)):
        want, bound, added, added_bound = decode_definition(c, q, g, scale)
        before = c.mass.double()
        out = decode(ctx, c, q, g, scale=scale)
        assert ((out.double() - want).abs() <= bound).all()
        assert (out[0] == 0).all()                                            # an idle lane
        # the sum with what was there is rounded once more
        off = (c.mass.double() - before - added).abs()
        assert (off <= added_bound + 2.0 ** -24 * (before + added)).all()
        without = decode(ctx, c, q, g, mass=False, scale=scale)
        assert torch.equal(out, without)


@pytest.mark.parametrize("kv_heads,group,dim,n,page", [(2, 8, 256, 9472, 64), (2, 8, 256, 9473, 16), (2, 8, 256, 70001, 48),
                                                       (1, 16, 64, 75777, 16), (8, 4, 128, 33001, 64), (300, 1, 64, 700, 32)])
def test_long_lanes_and_many_heads(ctx, kv_heads, group, dim, n, page):
    c = Cache([n, 3], kv_heads, dim, page=page, seed=n)
    q, gate = query(c, kv_heads * group, warmth=3.0)
    want, bound, added, added_bound = decode_definition(c, q, gate, dim ** -0.5)
    before = c.mass.double()
    out = decode(ctx, c, q, gate)
    assert ((out.double() - want).abs() <= bound).all()
    assert ((c.mass.double() - before - added).abs() <= added_bound + 2.0 ** -24 * (before + added)).all()


@pytest.mark.parametrize("kv_heads,group,dim,most", [(2, 8, 256, 300), (3, 16, 256, 40), (8, 4, 128, 200), (4, 11, 128, 17), (12, 1, 64, 70),
                                                     (16, 16, 64, 300), (64, 2, 64, 20)])
def test_many_short_lanes(ctx, kv_heads, group, dim, most):
    """Far more partitions than CTAs, most of them too short for every warp to have a share, of lanes in any mixture of lengths."""
    rng = np.random.default_rng(most)
    lens = [int(x) for x in rng.integers(0, most + 1, 256)]
    lens[100], lens[101] = 3 * most + 400, 1
    c = Cache(lens, kv_heads, dim, page=32, seed=most)
    q, gate = query(c, kv_heads * group)
    want, bound, added, added_bound = decode_definition(c, q, gate, dim ** -0.5)
    before = c.mass.double()
    out = decode(ctx, c, q, gate)
    assert ((out.double() - want).abs() <= bound).all()
    assert ((c.mass.double() - before - added).abs() <= added_bound + 2.0 ** -24 * (before + added)).all()


def test_more_partitions_than_a_cta_describes_at_once(ctx):
    """256 lanes of 300 heads are about 260 partitions for every CTA; the same lanes in calls of eight are at most nine."""
    rng = np.random.default_rng(8)
    lens = [int(x) for x in rng.integers(0, 17, 256)]
    lens[7], lens[200] = 16, 1
    c = Cache(lens, 300, 256, page=16, seed=8, extra_columns=0)
    q, gate = query(c, 300)
    out = decode(ctx, c, q, gate, mass=False)
    for i in range(0, 256, 8):
        part = tb.paged_cache(c.keys, c.values, c.table[i: i + 8])
        got, lanes = torch.full_like(q[i: i + 8], 7.0), c.lanes[i: i + 8].contiguous()
        ctx.attn_decode_paged(part, lanes, q[i: i + 8], gate[i: i + 8], got, scratch_for(part, 8, 16, 300))
        ctx.sync()
        assert torch.equal(got, out[i: i + 8])


def test_lanes_that_share_a_prefix(ctx):
    """Two lanes on the same first pages: decode reads them twice, the masses stay apart, an eviction that guards the prefix leaves it."""
    c = Cache([200, 150], 2, 128, page=16, seed=33)
    c.table[1, :4] = c.table[0, :4]                                   # 64 common slots
    q, gate = query(c, 8)
    want, bound, added, added_bound = decode_definition(c, q, gate, 128 ** -0.5)
    before = c.mass.double()
    out = decode(ctx, c, q, gate)
    assert ((out.double() - want).abs() <= bound).all()
    assert ((c.mass.double() - before - added).abs() <= added_bound + 2.0 ** -24 * (before + added)).all()
    # each lane against a definition of its own cache: no page below the guarded slots is written
    prefix = [x[c.table[0, :4].long()].clone() for x in (c.keys, c.values)]
    expected = evict_definition(c, 100, 64, 12)
    run_evict(ctx, c, 100, 64, 12)
    assert same_cache(c, expected)
    assert all(same(x[c.table[0, :4].long()], y) for x, y in zip((c.keys, c.values), prefix))


def test_the_longest_context(ctx):
    c = Cache([262144], 2, 256, page=64, seed=9, extra_columns=0)
    q, gate = query(c, 16)
    want, bound, added, added_bound = decode_definition(c, q, gate, 0.0625)
    before = c.mass.double()
    out = decode(ctx, c, q, gate)
    assert ((out.double() - want).abs() <= bound).all()
    assert ((c.mass.double() - before - added).abs() <= added_bound + 2.0 ** -24 * (before + added)).all()


@pytest.mark.parametrize("dim,kv_heads,group", [(256, 2, 8), (256, 7, 6), (128, 4, 12), (128, 16, 6), (64, 3, 5)])
def test_a_lane_has_the_same_bits_alone_in_a_batch_and_in_other_pages(ctx, dim, kv_heads, group):
    lens = [700, 0, 1300, 90, 12000, 257]
    c = Cache(lens, kv_heads, dim, seed=4)
    q, gate = query(c, kv_heads * group)
    start = c.mass.clone()
    out = decode(ctx, c, q, gate)
    batch_mass = c.mass.clone()
    for i, n in enumerate(lens):
        alone = Cache([n], kv_heads, dim, page=32, slot_major=True, seed=50 + i)
        for pool, source in ((alone.keys, c.keys), (alone.values, c.values)):
            for head in range(kv_heads if n else 0):
                s = torch.arange(n, device="cuda")
                pool[alone.table[0, s // 32].long(), head, s % 32] = c.rows(source, i, head, n)
        alone.mass[:, :, :n] = start[i, :, :n]
        got = decode(ctx, alone, q[i: i + 1], gate[i: i + 1], max_keys=max(1, n))
        assert torch.equal(got[0], out[i])
        assert same(alone.mass[0, :, :n], batch_mass[i, :, :n])


@pytest.mark.parametrize("slot_major,dim", [(False, 256), (True, 128), (True, 64)])
def test_rows_asked_ahead_change_no_bit(ctx, slot_major, dim):
    """Long partitions ask their first rows into L2 before the wait; tokens whose lane and rows change right before each call."""
    n, kept = 60000, ctx.get_policy(tb.POLICY_DECODE_L2_PREFETCH_KEYS)
    c = Cache([n + 40], 2, dim, page=64, slot_major=slot_major, seed=dim)
    c.lanes[0, 0] = n
    q, gate = query(c, 8)
    rows = [torch.randn((40, 1, 2, dim), device="cuda").to(torch.bfloat16) for _ in range(2)]
    results = []
    for ahead in (0, 512):
        ctx.set_policy(tb.POLICY_DECODE_L2_PREFETCH_KEYS, ahead)
        own = c.clone()
        h = handle(own)
        scratch, outs = scratch_for(h, 1, h.capacity, 8), torch.zeros((40, *q.shape), dtype=q.dtype, device="cuda")
        torch.cuda.synchronize()
        for i in range(40):
            ctx.paged_lanes_step(own.lanes)
            ctx.paged_append(h, own.lanes, rows[0][i], rows[1][i])
            ctx.attn_decode_paged(h, own.lanes, q, gate, outs[i], scratch)
        ctx.sync()
        results.append((outs, own))
    ctx.set_policy(tb.POLICY_DECODE_L2_PREFETCH_KEYS, kept)
    assert torch.equal(results[0][0], results[1][0]) and same_cache(results[0][1], results[1][1])
    assert torch.isfinite(results[0][0]).all()


def test_matches_the_contiguous_decode(ctx):
    """The same cache as a stripe of the contiguous operator: two results within both operators' roundings."""
    n = 3001
    c = Cache([n], 2, 256, seed=6)
    q, gate = query(c, 16)
    k, v = (torch.stack([c.rows(x, 0, h, n) for h in range(2)]).contiguous() for x in (c.keys, c.values))
    other = torch.zeros_like(q)
    scratch = torch.empty(tb.decode_scratch_bytes(n) // 4, device="cuda")
    ctx.attn_decode(q, gate, k, v, n - 1, n, other, scratch)
    out = decode(ctx, c, q, gate)
    _, bound, _, _ = decode_definition(c, q, gate, 0.0625)
    assert ((out.double() - other.double()).abs() <= 2 * bound).all()


def test_strided_rows_of_queries_and_outputs(ctx):
    c = Cache([100, 40], 2, 128, seed=8)
    wide = torch.randn((3, 2, 1100), device="cuda").to(torch.bfloat16)
    q, gate, out = (wide[i][:, 10: 10 + 8 * 128].unflatten(1, (8, 128)) for i in range(3))
    edge = wide.clone()
    h = handle(c, mass=False)
    want, bound, _, _ = decode_definition(c, q, gate, 128 ** -0.5)
    ctx.attn_decode_paged(h, c.lanes, q, gate, out, scratch_for(h, 2, 128, 8), max_keys=128)
    ctx.sync()
    assert ((out.double() - want).abs() <= bound).all()
    assert same(wide[2][:, :10], edge[2][:, :10]) and same(wide[2][:, 1034:], edge[2][:, 1034:]) and same(wide[:2], edge[:2])


@pytest.mark.parametrize("kv_heads", [1, 3])
def test_pools_inside_one_allocation(ctx, kv_heads):
    """K and V side by side in one tensor, pages with a gap behind them: every stride its own."""
    lens, dim, page = [70, 33, 129], 128, 32
    c = Cache(lens, kv_heads, dim, page=page, seed=21)
    pages = c.keys.shape[0]
    both = torch.full((pages, 2, kv_heads + 1, page, dim + 8), float("nan"), dtype=torch.bfloat16, device="cuda")
    keys, values = both[:, 0, :kv_heads, :, :dim], both[:, 1, :kv_heads, :, :dim]
    keys.copy_(c.keys), values.copy_(c.values)
    h = tb.paged_cache(keys, values, c.table, mass=c.mass, positions=c.positions)
    q, gate = query(c, 4 * kv_heads)
    plain = c.clone()
    out = torch.zeros_like(q)
    ctx.attn_decode_paged(h, c.lanes, q, gate, out, scratch_for(h, 3, 129, 4 * kv_heads), max_keys=129)
    assert torch.equal(out, decode(ctx, plain, q, gate, max_keys=129))
    new = [torch.randn((3, kv_heads, dim), device="cuda").to(torch.bfloat16) for _ in range(2)]
    ctx.paged_append(h, c.lanes, *new)
    ctx.paged_append(handle(plain), plain.lanes, *new)
    ctx.paged_evict(h, c.lanes, 40, torch.empty(tb.paged_evict_scratch_bytes(h, 3, 160, 40), dtype=torch.uint8, device="cuda"), sink=2, recent=9, max_keys=160)
    run_evict(ctx, plain, 40, 2, 9)
    ctx.sync()
    assert same(keys, plain.keys) and same(values, plain.values) and same(c.mass, plain.mass) and same(c.positions, plain.positions)
    assert torch.isnan(both[:, :, kv_heads:]).all() and torch.isnan(both[..., dim:]).all()


def test_extreme_scores(ctx):
    """One key that takes all the weight, keys of the type's largest values, an infinite score: what the definition gives."""
    c = Cache([40, 40, 40], 1, 64, dtype=torch.float16, seed=12)
    q = torch.ones((3, 1, 64), dtype=torch.float16, device="cuda")
    p, r = int(c.table[0, 2]), 39 % 16
    c.keys[p, 0, r] = 60000.0                                         # lane 0: score 480000 against a few
    for s in range(40):                                               # lane 1: every score the type's lowest times 64
        c.keys[int(c.table[1, s // 16]), 0, s % 16] = -65504.0
    c.keys[int(c.table[2, 0]), 0, 0] = float("-inf")                  # lane 2: one key without weight
    out = decode(ctx, c, q, None)
    assert same(out[0, 0], c.values[p, 0, r])
    u = 2.0 ** -11
    for lane, slots in ((1, range(40)), (2, range(1, 40))):
        k, v = (torch.stack([pool[int(c.table[lane, s // 16]), 0, s % 16] for s in slots]).double() for pool in (c.keys, c.values))
        w = torch.softmax(q[lane].double() @ k.T / 8.0, dim=-1)
        assert ((out[lane].double() - w @ v).abs() <= u * (w @ v).abs() + (u + 2.0 ** -11) * (w @ v.abs()) + 2.0 ** -20).all()
    assert float(c.mass[2, 0, 0]) < 1.0                               # nothing was added there


def test_not_a_number_is_not_hidden(ctx):
    c = Cache([40, 40], 2, 64, seed=13)
    c.keys[int(c.table[0, 1]), 0, 3, 5] = float("nan")
    q, _ = query(c, 4)
    out = decode(ctx, c, q, None)
    assert torch.isnan(out[0, :2]).all() and torch.isfinite(out[0, 2:]).all() and torch.isfinite(out[1]).all()


def test_refused_lanes_and_absent_pages(ctx):
    c = Cache([100, 300, 60], 2, 128, seed=14)
    q, gate = query(c, 8)
    want, bound, _, _ = decode_definition(c, q, gate, 128 ** -0.5)
    h = handle(c)
    before = c.mass.clone()
    out = torch.full_like(q, 7.0)
    ctx.attn_decode_paged(h, c.lanes, q, gate, out, scratch_for(h, 3, 128, 8), max_keys=128)     # lane 1 holds more
    with pytest.raises(tb.TataraError) as e:
        ctx.sync()
    assert e.value.status == RANGE
    assert (out[1] == 7.0).all() and same(c.mass[1], before[1])
    assert ((out.double() - want).abs() <= bound)[[0, 2]].all()
    # a page that the pool does not have: its slots count as absent
    c.table[0, 2] = c.keys.shape[0] + 5
    c.table[2, :] = -1
    got = torch.full_like(q, 7.0)
    before = c.mass.clone()
    ctx.attn_decode_paged(h, c.lanes, q, gate, got, scratch_for(h, 3, 300, 8), max_keys=300)
    with pytest.raises(tb.TataraError):
        ctx.sync()
    ctx.sync()
    there = torch.tensor([s for s in range(100) if s // 16 != 2], device="cuda")
    for head in range(2):
        k, v = (x[c.table[0, there // 16].long(), head, there % 16].double() for x in (c.keys, c.values))
        w = torch.softmax(q[0, 4 * head: 4 * head + 4].double() @ k.T * 128 ** -0.5, dim=-1)
        o = (w @ v) * torch.sigmoid(gate[0, 4 * head: 4 * head + 4].double())
        assert ((got[0, 4 * head: 4 * head + 4].double() - o).abs() <= 2.0 ** -7 * (w @ v.abs()) + 2.0 ** -20).all()
    assert ((got.double() - want).abs() <= bound)[1].all() and (got[2] == 0).all()
    assert same(c.mass[0, :, 32:48], before[0, :, 32:48]) and same(c.mass[2], before[2])


# ---- append ------------------------------------------------------------------------------------------------------------


def append_definition(c, starts, keys, values):
    after = c.clone()
    for lane, (n, position) in enumerate(c.lanes.tolist()):
        count = starts[lane + 1] - starts[lane]
        for r in range(count):
            slot = n - count + r
            page = int(c.table[lane, slot // c.page])
            after.keys[page, :, slot % c.page] = keys[starts[lane] + r]
            after.values[page, :, slot % c.page] = values[starts[lane] + r]
            after.mass[lane, :, slot] = 0.0
            after.positions[lane, :, slot] = position - count + 1 + r
    return after


@pytest.mark.parametrize("kv_heads,dim,page,slot_major,dtype", [(2, 256, 16, False, torch.bfloat16), (3, 128, 48, True, torch.float16),
                                                                (1, 64, 32, True, torch.bfloat16), (9, 64, 16, False, torch.float16)])
@pytest.mark.parametrize("layout", ["rows", "planes", "padded"])
def test_append(ctx, kv_heads, dim, page, slot_major, dtype, layout):
    lens, counts = [1, 40, 64, 100, 333], [1, 0, 33, 100, 17]
    starts = [0] + np.cumsum(counts).tolist()
    c = Cache(lens, kv_heads, dim, dtype=dtype, page=page, slot_major=slot_major, seed=dim + kv_heads)
    c.lanes[3, 1] = 5000                                              # a lane that evicted before
    rows = starts[-1] + (29 if layout == "padded" else 0)             # rows behind the last lane's are padding
    make = lambda: torch.randn((kv_heads, rows + 8, dim) if layout == "planes" else (rows, kv_heads, dim + 8), device="cuda").to(dtype)
    k, v = make(), make()
    k, v = (x[:, :rows].transpose(0, 1) if layout == "planes" else x[:, :, :dim] for x in (k, v))
    want = append_definition(c, starts, k, v)
    ctx.paged_append(handle(c), c.lanes, k, v, row_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    ctx.sync()
    assert same_cache(c, want)
    # one row per lane, into a cache without planes
    k1, v1 = k[:5], v[:5]
    want = append_definition(c, list(range(6)), k1, v1)
    want.mass, want.positions = c.mass.clone(), c.positions.clone()
    ctx.paged_append(handle(c, mass=False, positions=False), c.lanes, k1, v1)
    ctx.sync()
    assert same_cache(c, want)


def test_append_leaves_out_what_has_no_slot(ctx):
    c = Cache([10, 0, 20, 30], 2, 64, seed=3)
    full = c.table.shape[1] * c.page
    c.lanes[2, 0] = full + 1                                          # beyond the page table
    c.table[3, 1] = 1 << 20                                           # a page that does not exist: slots 16 .. 29
    k, v = (torch.randn((60, 2, 64), device="cuda").to(torch.bfloat16) for _ in range(2))
    starts = [0, 12, 15, 20, 45]                                      # lane 0: two rows too many; lane 1 is idle
    want = c.clone()
    for lane, slot, row in [(0, s, s + 2) for s in range(10)] + [(3, s, 15 + s) for s in range(5, 16)]:
        row = 20 + slot - 5 if lane == 3 else row
        page = int(c.table[lane, slot // 16])
        want.keys[page, :, slot % 16], want.values[page, :, slot % 16] = k[row], v[row]
        want.mass[lane, :, slot], want.positions[lane, :, slot] = 0.0, slot
    ctx.paged_append(handle(c), c.lanes, k, v, row_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    with pytest.raises(tb.TataraError) as e:
        ctx.sync()
    assert e.value.status == RANGE
    assert same_cache(c, want)


def test_append_of_rows_that_are_not_there(ctx):
    c = Cache([40, 40], 1, 64, seed=4)
    k, v = (torch.randn((50, 1, 64), device="cuda").to(torch.bfloat16) for _ in range(2))
    want = append_definition(c, [0, 40, 80], torch.cat([k, k]), torch.cat([v, v]))
    for slot in range(10, 40):                                        # rows 50 .. 79 of lane 1 are missing
        page, row = int(c.table[1, slot // 16]), slot % 16
        want.keys[page, :, row], want.values[page, :, row] = c.keys[page, :, row], c.values[page, :, row]
        want.mass[1, :, slot], want.positions[1, :, slot] = c.mass[1, :, slot], c.positions[1, :, slot]
    ctx.paged_append(handle(c), c.lanes, k, v, row_starts=torch.tensor([0, 40, 80], dtype=torch.int32, device="cuda"))
    with pytest.raises(tb.TataraError) as e:
        ctx.sync()
    assert e.value.status == RANGE
    assert same_cache(c, want)


def test_offsets_beyond_32_bits(ctx):
    """Pools of 2.3 G elements, the lane's pages at their far end: append, decode, eviction."""
    page, heads, dim, pages = 16, 2, 256, 280000
    pools = [torch.zeros((pages, heads, page, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    n = 100
    table = torch.arange(pages - 8, pages, dtype=torch.int32, device="cuda").flip(0).reshape(1, 8).contiguous()
    mass, positions = torch.zeros((1, heads, 128), device="cuda"), torch.zeros((1, heads, 128), dtype=torch.int32, device="cuda")
    lanes = torch.tensor([[n, n - 1]], dtype=torch.int32, device="cuda")
    h = tb.paged_cache(pools[0], pools[1], table, mass=mass, positions=positions)
    k, v = (torch.randn((n, heads, dim), device="cuda").to(torch.bfloat16) for _ in range(2))
    ctx.paged_append(h, lanes, k, v, row_starts=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    small = Cache([n], heads, dim, seed=1)
    s = torch.arange(n, device="cuda")
    for pool, big, rows in ((small.keys, pools[0], k), (small.values, pools[1], v)):
        assert same(big[table[0, s // 16].long(), :, s % 16], rows)
        pool[small.table[0, s // 16].long(), :, s % 16] = rows
    q, gate = query(small, 16)
    out = torch.zeros_like(q)
    ctx.attn_decode_paged(h, lanes, q, gate, out, scratch_for(h, 1, 128, 16))
    small.mass.zero_()
    assert torch.equal(out, decode(ctx, small, q, gate))
    assert same(mass[:, :, :n], small.mass[:, :, :n])
    want = evict_definition(small, 60, 4, 10)
    ctx.paged_evict(h, lanes, 60, torch.empty(tb.paged_evict_scratch_bytes(h, 1, 128, 60), dtype=torch.uint8, device="cuda"), sink=4, recent=10)
    ctx.sync()
    s = s[:60]
    assert same(pools[0][table[0, s // 16].long(), :, s % 16], want.keys[want.table[0, s // 16].long(), :, s % 16])
    assert same(pools[1][table[0, s // 16].long(), :, s % 16], want.values[want.table[0, s // 16].long(), :, s % 16])


# ---- q/k norm + rope + append --------------------------------------------------------------------------------------------


def rope_definition(c, projection, qw, kw):
    """q, its bound, k, its bound: [lane][head][256], 64 bits.  One rounding of the result; the f32 steps before it (a sum of 256
    squares, root, quotient, two products, sine and cosine, the rotation) are off by less than 2^-17 of the pair's size."""
    x = projection.double()
    angle = c.lanes[:, 1].double()[:, None] / torch.tensor(syn.rope_divisors(), device="cuda").double()
    sine, cosine = angle.sin()[:, None], angle.cos()[:, None]

    def turn(rows, weight):
        y = weight.double() * rows / torch.sqrt((rows ** 2).mean(-1, keepdim=True) + 1e-6)
        lo, hi = y[..., :32], y[..., 32:64]
        out = torch.cat([lo * cosine - hi * sine, hi * cosine + lo * sine, y[..., 64:]], -1)
        size = torch.cat([lo.abs() + hi.abs(), lo.abs() + hi.abs(), y[..., 64:].abs()], -1)
        return out, 2.0 ** -8 * out.abs() + 2.0 ** -17 * size

    rows = x.shape[0]
    pairs = x[:, :8192].reshape(rows, 16, 2, 256)
    return *turn(pairs[:, :, 0], qw), *turn(x[:, 8192:8704].reshape(rows, 2, 256), kw)


@pytest.mark.parametrize("lanes,page", [(1, 16), (7, 48), (256, 32)])
def test_rope_paged(ctx, lanes, page):
    rng = np.random.default_rng(lanes)
    lens = [int(x) for x in rng.integers(1, 200, lanes)]
    c = Cache(lens, 2, 256, page=page, seed=lanes)
    for i in range(0, lanes, 3):
        c.lanes[i, 1] = int(rng.integers(lens[i], 262144))            # evicted before: far positions
    if lanes > 2:
        c.lanes[2, 0] = 0
    qw, kw = (dev_bf16(w) for w in syn.attn_weights(rng, unit=False))
    projection = dev_bf16(syn.attn_projection(rng, lanes))
    wide = torch.full((2, lanes, 4200), 3.0, dtype=torch.bfloat16, device="cuda")
    q, gate = (wide[i][:, :4096].unflatten(1, (16, 256)) for i in range(2))
    want_q, q_bound, want_k, k_bound = rope_definition(c, projection, qw, kw)
    want = c.clone()
    live = [i for i in range(lanes) if not (lanes > 2 and i == 2)]
    ctx.attn_qk_rope_paged(handle(c), c.lanes, projection, qw, kw, q, gate)
    ctx.sync()
    assert ((q.double() - want_q).abs() <= q_bound)[live].all()
    assert same(gate[live], projection[:, :8192].reshape(lanes, 16, 2, 256)[live, :, 1])
    if lanes > 2:
        assert (q[2] == 3.0).all() and (gate[2] == 3.0).all()
    assert (wide[:, :, 4096:] == 3.0).all()
    for i in live:
        n = lens[i]
        at = (int(c.table[i, (n - 1) // page]), slice(None), (n - 1) % page)
        assert ((c.keys[at].double() - want_k[i]).abs() <= k_bound[i]).all()
        assert same(c.values[at], projection[i, 8704:].reshape(2, 256))
        want.keys[at], want.values[at] = c.keys[at], c.values[at]
        want.mass[i, :, n - 1], want.positions[i, :, n - 1] = 0.0, c.lanes[i, 1]
    assert same_cache(c, want)                                        # nothing else was touched


def test_rope_paged_agrees_with_the_contiguous_append(ctx):
    """attn_qk_rope_batch rounds the normalised row twice to bf16 before the rotation and takes its angle in f32: at small positions that
    is three roundings of half a step against one, each of a value no larger than the pair's."""
    rng = np.random.default_rng(5)
    lanes = 6
    c = Cache([i + 1 for i in range(lanes)], 2, 256, seed=2)
    qw, kw = (dev_bf16(w) for w in syn.attn_weights(rng, unit=False))
    projection = dev_bf16(syn.attn_projection(rng, lanes))
    q, gate, q2, gate2 = (torch.zeros((lanes, 16, 256), dtype=torch.bfloat16, device="cuda") for _ in range(4))
    pools = [torch.zeros((lanes, 2, 16, 256), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ctx.attn_qk_rope_batch(projection, qw, kw, q2, gate2, *pools, 16, tb.Context.attn_lanes([(i * 8192, i) for i in range(lanes)]))
    ctx.attn_qk_rope_paged(handle(c), c.lanes, projection, qw, kw, q, gate)
    ctx.sync()
    assert torch.equal(gate, gate2)
    size = q.float().abs()
    size[..., :64] = (size[..., :32] ** 2 + size[..., 32:64] ** 2).sqrt().repeat(1, 1, 2)
    assert ((q.float() - q2.float()).abs() <= 5 * 2.0 ** -8 * size + 2.0 ** -18).all()


def test_rope_paged_latches_what_has_no_slot(ctx):
    c = Cache([10, 20, 30], 2, 256, seed=3)
    c.lanes[0, 0] = c.table.shape[1] * 16 + 1
    c.table[1, 1] = -2
    rng = np.random.default_rng(1)
    qw, kw = (dev_bf16(w) for w in syn.attn_weights(rng))
    projection = dev_bf16(syn.attn_projection(rng, 3))
    q, gate = (torch.zeros((3, 16, 256), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    want = c.clone()
    ctx.attn_qk_rope_paged(handle(c), c.lanes, projection, qw, kw, q, gate)
    with pytest.raises(tb.TataraError) as e:
        ctx.sync()
    assert e.value.status == RANGE
    at = (int(c.table[2, 1]), slice(None), 29 % 16)
    want.keys[at], want.values[at] = c.keys[at], c.values[at]
    want.mass[2, :, 29], want.positions[2, :, 29] = 0.0, 29
    assert same_cache(c, want) and (q[0] == 0).all()


# ---- eviction ------------------------------------------------------------------------------------------------------------


def run_evict(ctx, c, keep, sink=0, recent=0, max_keys=None, positions=True):
    h = handle(c, positions=positions)
    most = h.capacity if max_keys is None else max_keys
    scratch = torch.full((tb.paged_evict_scratch_bytes(h, len(c.lens), most, keep),), 0xAB, dtype=torch.uint8, device="cuda")
    ctx.paged_evict(h, c.lanes, keep, scratch, sink=sink, recent=recent, max_keys=most)
    ctx.sync()


def fill_mass(c, kind):
    m = c.mass
    if kind == "spread":
        m.copy_(torch.exp(6 * torch.randn(m.shape, generator=c.gen, device="cuda")))
    elif kind == "ties":
        m.copy_(torch.randint(0, 3, m.shape, generator=c.gen, device="cuda").float())
    elif kind == "equal":
        m.fill_(0.25)
    elif kind == "odd":                                               # what no honest sum holds, but memory may
        m.copy_(torch.randn(m.shape, generator=c.gen, device="cuda"))
        for i, x in enumerate((float("nan"), float("inf"), -float("inf"), -0.0, 0.0, 1e-45, -1e-45, -float("nan"))):
            m[:, :, i::23] = x


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("lens,keep,sink,recent", [
    ([2, 1, 3, 9], 1, 0, 0), ([100, 40, 41, 0, 39], 40, 0, 0), ([100, 64, 65, 200], 64, 4, 20), ([300], 299, 10, 30), ([300], 31, 31, 0),
    ([300], 31, 0, 31), ([777, 500, 1200, 33], 256, 16, 240)])
def test_evict_matches_the_definition(ctx, kind, lens, keep, sink, recent):
    c = Cache(lens, 3, 64, page=32, slot_major=keep % 2 == 0, dtype=torch.float16, seed=keep)
    fill_mass(c, kind)
    want = evict_definition(c, keep, sink, recent)
    run_evict(ctx, c, keep, sink, recent)
    assert same_cache(c, want)


@pytest.mark.parametrize("kv_heads,dim,n,keep,sink,recent,kind", [
    (2, 256, 4200, 4096, 4, 100, "spread"), (2, 128, 20000, 5000, 64, 1000, "ties"), (1, 64, 52001, 1000, 0, 0, "spread"),
    (1, 64, 262144, 100000, 128, 4096, "ties"), (40, 64, 5000, 2500, 3, 7, "odd"), (160, 64, 300, 100, 1, 5, "spread")])
def test_evict_of_long_lanes_and_many_heads(ctx, kv_heads, dim, n, keep, sink, recent, kind):
    """A CTA for a head with 2 to 16 keys a thread, and lanes that many CTAs share."""
    c = Cache([n], kv_heads, dim, page=64, seed=n, extra_columns=0)
    fill_mass(c, kind)
    # slots in no order of position, as after earlier evictions
    c.positions[0, :, :n] = torch.stack([torch.randperm(n, generator=c.gen, device="cuda") for _ in range(kv_heads)]).to(torch.int32)
    want = evict_definition(c, keep, sink, recent)
    run_evict(ctx, c, keep, sink, recent)
    assert same_cache(c, want)


@pytest.mark.parametrize("kv_heads,lens,keep,sink,recent,kind", [
    (16, [40000, 700, 16385, 30001], 700, 3, 40, "spread"), (13, [17000, 20480, 20481, 9], 16384, 5, 2000, "ties"), (2, [16385, 36865, 0], 4096, 0, 0, "equal"),
    (3, [70000, 50, 33000], 30000, 9, 100, "odd")])
def test_evict_of_ragged_long_lanes(ctx, kv_heads, lens, keep, sink, recent, kind):
    """Lanes of many CTAs next to lanes of one and lanes that stay, in few large and many small shares; a lane beyond max_keys is left alone."""
    c = Cache(lens, kv_heads, 64, page=64, seed=keep, extra_columns=0)
    fill_mass(c, kind)
    for lane, n in enumerate(lens):
        c.positions[lane, :, :n] = torch.stack([torch.randperm(n, generator=c.gen, device="cuda") for _ in range(kv_heads)]).to(torch.int32)
    want = evict_definition(c, keep, sink, recent)
    before = c.clone()
    run_evict(ctx, c, keep, sink, recent)
    assert same_cache(c, want)
    h = handle(before)
    untouched = before.clone()
    most = max(x for x in lens if x < max(lens))
    scratch = torch.full((tb.paged_evict_scratch_bytes(h, len(lens), most, keep),), 0x5A, dtype=torch.uint8, device="cuda")
    ctx.paged_evict(h, before.lanes, keep, scratch, sink=sink, recent=recent, max_keys=most)
    with pytest.raises(tb.TataraError) as e:
        ctx.sync()
    assert e.value.status == RANGE
    long = lens.index(max(lens))
    mine = untouched.table[long].long()
    assert same(before.keys[mine], untouched.keys[mine]) and same(before.mass[long], untouched.mass[long])
    rest = [i for i in range(len(lens)) if i != long]
    assert all(same(before.mass[i], want.mass[i]) and same(before.keys[want.table[i].long()], want.keys[want.table[i].long()]) for i in rest)


def test_evict_more_guarded_than_kept(ctx):
    c = Cache([200], 2, 64, seed=5)
    c.positions[:, :, :200] = 199                                     # every token says it is the newest
    want = evict_definition(c, 50, 5, 10)
    run_evict(ctx, c, 50, 5, 10)
    assert same_cache(c, want) and same(want.keys, Cache([200], 2, 64, seed=5).keys)    # the lower slots stay: nothing moves


def test_evict_without_positions_and_a_lane_beyond_max_keys(ctx):
    c = Cache([200, 120], 2, 64, seed=6)
    want = evict_definition(c, 50, 5, 0)
    want.positions = c.positions.clone()
    for x in ("keys", "values"):
        getattr(want, x)[c.table[0].long()] = getattr(c, x)[c.table[0].long()]
    want.mass[0] = c.mass[0]
    h = handle(c, positions=False)
    scratch = torch.empty(tb.paged_evict_scratch_bytes(h, 2, 150, 50), dtype=torch.uint8, device="cuda")
    ctx.paged_evict(h, c.lanes, 50, scratch, sink=5, max_keys=150)    # lane 0 holds 200
    with pytest.raises(tb.TataraError) as e:
        ctx.sync()
    assert e.value.status == RANGE
    assert same_cache(c, want)


def test_evict_leaves_absent_pages_alone(ctx):
    c = Cache([100], 1, 64, seed=7)
    c.mass[0, 0, :50] = torch.arange(50, device="cuda").float()       # slots 0 .. 14 go, 85 .. 99 come
    c.mass[0, 0, 50:100] = torch.arange(50, device="cuda").float() - 20
    whole = c.clone()
    c.table[0, 0] = 1 << 30                                           # the holes have no page
    want = evict_definition(whole, 50, 0, 0)
    p = int(whole.table[0, 0])
    h = handle(c)
    ctx.paged_evict(h, c.lanes, 50, torch.empty(tb.paged_evict_scratch_bytes(h, 1, 100, 50), dtype=torch.uint8, device="cuda"), max_keys=100)
    with pytest.raises(tb.TataraError):
        ctx.sync()
    other = [i for i in range(c.keys.shape[0]) if i != p]
    assert same(c.keys[other], want.keys[other]) and same(c.keys[p], whole.keys[p])


# ---- together -------------------------------------------------------------------------------------------------------------


def test_lanes_step(ctx):
    lanes = torch.tensor([[5, 9], [0, 0], [100, 300], [64, 63]], dtype=torch.int32, device="cuda")
    ctx.paged_lanes_step(lanes)
    assert lanes.tolist() == [[6, 10], [0, 0], [101, 301], [65, 64]]
    ctx.paged_lanes_step(lanes, keep=64, advance=0)
    assert lanes.tolist() == [[6, 10], [0, 0], [64, 301], [64, 64]]
    ctx.paged_lanes_step(lanes, keep=64, advance=2)
    assert lanes.tolist() == [[8, 12], [0, 0], [66, 303], [66, 66]]


def serve(ctx, c, projections, qw, kw, keep, every, graph):
    """Tokens through rope + append, decode with mass, the lane step, and every few tokens an eviction; outputs of every token."""
    lanes, h = len(c.lens), handle(c)
    most = h.capacity
    scratch = scratch_for(h, lanes, most, 16)
    evict_scratch = torch.empty(tb.paged_evict_scratch_bytes(h, lanes, most, keep), dtype=torch.uint8, device="cuda")
    x = torch.zeros_like(projections[0])
    q, gate, out = (torch.zeros((lanes, 16, 256), dtype=torch.bfloat16, device="cuda") for _ in range(3))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def token(trim):
        ctx.paged_lanes_step(c.lanes, stream=stream)
        ctx.attn_qk_rope_paged(h, c.lanes, x, qw, kw, q, gate, stream=stream)
        ctx.attn_decode_paged(h, c.lanes, q, gate, out, scratch, stream=stream)
        if trim:
            ctx.paged_evict(h, c.lanes, keep, evict_scratch, sink=4, recent=16, stream=stream)
            ctx.paged_lanes_step(c.lanes, keep=keep, advance=0, stream=stream)

    graphs = {}
    if graph:
        for trim in (False, True):
            graphs[trim] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graphs[trim], stream=stream):
                token(trim)
    outs = []
    for i, row in enumerate(projections):
        trim = (i + 1) % every == 0
        with torch.cuda.stream(stream):
            x.copy_(row)
            if graph:
                graphs[trim].replay()
            else:
                token(trim)
            outs.append(out.clone())
    ctx.sync(stream)
    return outs


@pytest.mark.parametrize("graph", [False, True])
def test_a_served_batch_follows_its_definition(ctx, graph):
    """Prompts appended from a contiguous cache, then 40 tokens with an eviction every 7: each token's output against the 64-bit attention
    over the tokens that the definition still holds."""
    prompts, keep, every, tokens = [90, 5, 130], 100, 7, 40
    rng = np.random.default_rng(17)
    qw, kw = (dev_bf16(w) for w in syn.attn_weights(rng, unit=False))
    c = Cache([n + tokens for n in prompts], 2, 256, seed=31)
    c.lanes.copy_(torch.tensor([[n, n - 1] for n in prompts], dtype=torch.int32))
    c.keys[c.table.long().flatten()] = float("nan")
    c.values[c.table.long().flatten()] = float("nan")
    stripes = [torch.randn((2, sum(prompts) + 3, 256), generator=c.gen, device="cuda").to(torch.bfloat16) for _ in range(2)]
    k, v = (s[:, : sum(prompts)].transpose(0, 1) for s in stripes)
    starts = torch.tensor(np.concatenate([[0], np.cumsum(prompts)]), dtype=torch.int32, device="cuda")
    ctx.paged_append(handle(c), c.lanes, k, v, row_starts=starts)
    ctx.sync()
    model = c.clone()
    projections = [dev_bf16(syn.attn_projection(rng, 3)) for _ in range(tokens)]
    outs = serve(ctx, c, projections, qw, kw, keep, every, graph)
    # the definition, token by token; K, q and the masses that rank are taken from the kernels' own types
    h = handle(model)
    q, gate = (torch.zeros((3, 16, 256), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for i, row in enumerate(projections):
        model.lanes += 1
        ctx.attn_qk_rope_paged(h, model.lanes, row, qw, kw, q, gate)
        want, bound, added, _ = decode_definition(model, q, gate, 0.0625)
        assert ((outs[i].double() - want).abs() <= bound).all(), f"token {i}"
        decode(ctx, model, q, gate)                                   # the masses as the kernel rounds them
        if (i + 1) % every == 0:
            model = evict_definition(model, keep, 4, 16)
            model.lanes[:, 0].clamp_(max=keep)
            h = handle(model)
    for lane, n in enumerate(model.lanes[:, 0].tolist()):
        assert c.lanes[lane].tolist() == model.lanes[lane].tolist()
        assert same(c.mass[lane, :, :n], model.mass[lane, :, :n]) and same(c.positions[lane, :, :n], model.positions[lane, :, :n])
        for head in range(2):
            assert same(c.rows(c.keys, lane, head, n), model.rows(model.keys, lane, head, n))
            assert same(c.rows(c.values, lane, head, n), model.rows(model.values, lane, head, n))


def test_the_first_calls_of_a_process_inside_a_capture():
    """Nothing has to be set up by an earlier call: a fresh process captures the operators at once and replays them."""
    code = """
import sys, torch
sys.path.insert(0, %r), sys.path.insert(0, %r)
import tatara_b200 as tb
from paged_util import Cache, decode_definition
ctx = tb.Context(0)
c = Cache([200, 3000], 2, 256, seed=3)
h = tb.paged_cache(c.keys, c.values, c.table, mass=c.mass, positions=c.positions)
q, out = torch.randn((2, 16, 256), device="cuda").to(torch.bfloat16), torch.zeros((2, 16, 256), dtype=torch.bfloat16, device="cuda")
want, bound, _, _ = decode_definition(c, q, None, 0.0625)
scratch = torch.empty(tb.decode_paged_scratch_bytes(h, 2, h.capacity, 16), dtype=torch.uint8, device="cuda")
trim = torch.empty(tb.paged_evict_scratch_bytes(h, 2, h.capacity, 150), dtype=torch.uint8, device="cuda")
torch.cuda.synchronize()
graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
with torch.cuda.graph(graph, stream=stream):
    ctx.attn_decode_paged(h, c.lanes, q, None, out, scratch, stream=stream)
    ctx.paged_evict(h, c.lanes, 150, trim, sink=4, recent=20, stream=stream)
    ctx.paged_lanes_step(c.lanes, keep=150, advance=0, stream=stream)
assert (out == 0).all()
graph.replay()
torch.cuda.synchronize()
assert ((out.double() - want).abs() <= bound).all() and c.lanes[:, 0].tolist() == [150, 150]
ctx.sync()
print("captured")
""" % (os.path.dirname(os.path.dirname(os.path.abspath(__file__))), os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


def test_two_streams_at_once_and_a_stream_that_is_not_current(ctx):
    caches = [Cache([900, 40], 2, 256, seed=70 + i) for i in range(2)]
    asked = [query(c, 16) for c in caches]
    want = [decode(ctx, c.clone(), *a) for c, a in zip(caches, asked)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    handles = [handle(c, mass=False) for c in caches]
    scratches = [scratch_for(h, 2, h.capacity, 16) for h in handles]
    outs = [torch.zeros_like(a[0]) for a in asked]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            ctx.attn_decode_paged(handles[i], caches[i].lanes, *asked[i], outs[i], scratches[i], stream=streams[i])
    torch.cuda.synchronize()
    for got, expected in zip(outs, want):
        assert torch.equal(got, expected)


def test_an_eviction_beside_a_decode_on_another_stream(ctx):
    """A long lane is trimmed on one stream while another batch decodes on a second one; each finds what it finds alone."""
    trimmed, batch = Cache([40000, 20000], 2, 64, page=64, seed=80), Cache([3000, 700, 1], 2, 256, seed=81)
    fill_mass(trimmed, "spread")
    want = evict_definition(trimmed, 9000, 4, 500)
    q, gate = query(batch, 16)
    expected = decode(ctx, batch.clone(), q, gate, mass=False)
    h, hb = handle(trimmed), handle(batch, mass=False)
    trim = torch.empty(tb.paged_evict_scratch_bytes(h, 2, h.capacity, 9000), dtype=torch.uint8, device="cuda")
    scratch, outs = scratch_for(hb, 3, hb.capacity, 16), torch.zeros((30, *q.shape), dtype=q.dtype, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(30):
        ctx.attn_decode_paged(hb, batch.lanes, q, gate, outs[i], scratch, stream=streams[0])
        if i == 10:
            ctx.paged_evict(h, trimmed.lanes, 9000, trim, sink=4, recent=500, stream=streams[1])
    torch.cuda.synchronize()
    ctx.sync()
    assert same_cache(trimmed, want) and all(torch.equal(o, expected) for o in outs)


def test_python_refusals(ctx):
    c = Cache([10, 20], 2, 256, seed=1)
    h = handle(c)
    q, gate = query(c, 16)
    out, scratch = torch.zeros_like(q), scratch_for(h, 2, 20, 16)
    launches = ctx.launches
    for bad in (lambda: ctx.attn_decode_paged(h, c.lanes.long(), q, gate, out, scratch),
                lambda: ctx.attn_decode_paged(h, c.lanes, q.half(), gate, out, scratch),
                lambda: ctx.attn_decode_paged(h, c.lanes, q[:1], gate, out, scratch),
                lambda: ctx.attn_decode_paged(h, c.lanes, q, gate[:, :, ::2], out, scratch),
                lambda: ctx.attn_decode_paged(h, c.lanes, q.transpose(1, 2), gate, out, scratch),
                lambda: ctx.paged_append(h, c.lanes, q[:, :2], gate[:, :2, :128]),
                lambda: ctx.paged_append(h, c.lanes, q[:, :3], gate[:, :3]),
                lambda: ctx.paged_append(h, c.lanes, q[:, :2], gate[:, :2], row_starts=c.lanes),
                lambda: ctx.attn_qk_rope_paged(h, c.lanes, q, q, q, q, gate),
                lambda: ctx.attn_decode_paged(h, c.lanes, q, gate, out, scratch.cpu()),
                lambda: ctx.attn_decode_paged(h, c.lanes.cpu(), q, gate, out, scratch),
                lambda: ctx.attn_decode_paged(h, c.lanes, q.cpu(), gate, out, scratch),
                lambda: ctx.paged_evict(h, c.lanes, 10, scratch.cpu()),
                lambda: ctx.paged_append(h, c.lanes, q[:, :2].cpu(), gate[:, :2].cpu())):
        with pytest.raises(ValueError):
            bad()
    assert ctx.launches == launches
