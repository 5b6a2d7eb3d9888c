"""Paged operators at the edges of what a call promises: eviction bounds that no lane can exceed."""
import os
import sys

import pytest
import torch

import tatara_b200 as tb

sys.path.insert(0, os.path.dirname(__file__))
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
