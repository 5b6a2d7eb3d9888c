"""Paged operators at the edges of what a call promises: eviction bounds that no lane can exceed, rotation at far positions."""
import os
import sys

import numpy as np
import pytest
import torch

import tatara_b200 as tb
from tatara_b200 import synthetic as syn

sys.path.insert(0, os.path.dirname(__file__))
from gpu_util import dev_bf16  # noqa: E402
from paged_util import Cache, same_cache  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = tb.Context(0)
    yield c
    c.close()


def evict(ctx, c, keep, max_keys):
    h = tb.paged_cache(c.keys, c.values, c.table, mass=c.mass, positions=c.positions)
    scratch = torch.full((tb.paged_evict_scratch_bytes(h, len(c.lens), max_keys, keep) + 16,), 0xAB, dtype=torch.uint8, device="cuda")
    ctx.paged_evict(h, c.lanes, keep, scratch, sink=2, recent=5, max_keys=max_keys)


@pytest.mark.parametrize("keep", [150, 151, 300])
def test_an_eviction_that_no_lane_can_need_looks_at_none(ctx, keep):
    """keep >= max_keys: nothing is enqueued, not even for a lane that holds more than it may; with keep below, that lane is reported."""
    c = Cache([200, 120], 2, 64, seed=6)
    want, launches = c.clone(), ctx.launches
    evict(ctx, c, keep, 150)
    ctx.sync()
    assert ctx.launches == launches and same_cache(c, want)
    evict(ctx, c, 149, 150)
    with pytest.raises(tb.TataraError) as e:
        ctx.sync()
    assert e.value.status == tb.STATUS_NAMES.index("ContextOutOfRange")
    assert same_cache(c, want)


def test_rope_paged_and_the_contiguous_append_at_far_positions(ctx):
    """attn_qk_rope_batch takes its angle, position / divisor, in f32: half a step of it, 2^-24 of the angle, turns the pair by as much more or
    less; up to 2^-7 rad at the longest context.  Beside that its two roundings of the normalised row and one of the result against one:
    five half steps of the pair's size at most."""
    rng = np.random.default_rng(11)
    where = [0, 1, 1000, 65537, 131071, 200003, 262000, 262143]
    lanes = len(where)
    c = Cache([i + 1 for i in range(lanes)], 2, 256, seed=2)
    c.lanes[:, 1] = torch.tensor(where, dtype=torch.int32)
    qw, kw = (dev_bf16(w) for w in syn.attn_weights(rng, unit=False))
    projection = dev_bf16(syn.attn_projection(rng, lanes))
    q, gate, q2, gate2 = (torch.zeros((lanes, 16, 256), dtype=torch.bfloat16, device="cuda") for _ in range(4))
    planes = [torch.zeros((2, 262144, 256), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ctx.attn_qk_rope_batch(projection, qw, kw, q2, gate2, *planes, 262144, tb.Context.attn_lanes([(0, x) for x in where]))
    ctx.attn_qk_rope_paged(tb.paged_cache(c.keys, c.values, c.table), c.lanes, projection, qw, kw, q, gate)
    ctx.sync()
    at = [(int(c.table[i, i // 16]), i % 16) for i in range(lanes)]
    k, v = (torch.stack([pool[page, :, row] for page, row in at]) for pool in (c.keys, c.values))
    k2, v2 = (plane[:, where].transpose(0, 1) for plane in planes)
    assert torch.equal(gate, gate2) and torch.equal(v, v2)
    angle = torch.tensor(where, device="cuda").double()[:, None] / torch.tensor(syn.rope_divisors(), device="cuda").double()
    turned = torch.zeros((lanes, 1, 256), dtype=torch.float64, device="cuda")
    turned[:, 0, :64] = (angle * 2.0 ** -24).repeat(1, 2)
    for a, b in ((q, q2), (k, k2)):
        size = a.double().abs()
        size[..., :64] = (size[..., :32] ** 2 + size[..., 32:64] ** 2).sqrt().repeat(1, 1, 2)
        assert ((a.double() - b.double()).abs() <= (5 * 2.0 ** -8 + 1.01 * turned) * size + 2.0 ** -18).all()
