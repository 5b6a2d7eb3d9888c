"""The paged cache operators without a device: the checks that come before anything is enqueued, the scratch sizes, and the
Python descriptors.  A zero-filled block stands for the context: a refused call only writes its error text."""
import ctypes
import os
import sys

import pytest
import torch

import tatara_b200 as tb

sys.path.insert(0, os.path.dirname(__file__))
from paged_util import Cache, evict_definition, same_cache  # noqa: E402

OK, BUFFER, RANGE, GROUP, EXTENT, SCRATCH = 0, 1, 2, 4, 5, 7
A = 0x10000   # an aligned address; no refused call reads it


@pytest.fixture()
def ctx():
    return ctypes.create_string_buffer(4096)


def cache(**change):
    c = tb.PagedCache(A, A, 2 * 16 * 256, 16 * 256, 256, A, A, A, 8, 100, 50, 16, 2, 256, 0, 0)
    for name, value in change.items():
        setattr(c, name, value)
    return c


def append(ctx, c, lanes=A, n=4, keys=A, values=A, row=512, head=256, starts=None, rows=4):
    return tb.lib().tatara_paged_append(ctx, None, ctypes.byref(c), lanes, n, keys, values, row, head, starts, rows)


def rope(ctx, c, lanes=A, n=4, projection=A, q=A, stride=9216, query=4096):
    return tb.lib().tatara_attn_qk_rope_paged(ctx, None, ctypes.byref(c), lanes, n, projection, A, A, q, A, stride, query)


def decode(ctx, c, lanes=A, n=4, max_keys=1000, q=A, gate=A, q_heads=16, stride=4096, scale=0.0625, out=A, scratch=A, nbytes=1 << 40):
    return tb.lib().tatara_attn_decode_paged(ctx, None, ctypes.byref(c), lanes, n, max_keys, q, gate, q_heads, stride, scale, out, scratch, nbytes)


def evict(ctx, c, lanes=A, n=4, max_keys=1000, keep=500, sink=4, recent=100, scratch=A, nbytes=1 << 40):
    return tb.lib().tatara_paged_evict(ctx, None, ctypes.byref(c), lanes, n, max_keys, keep, sink, recent, scratch, nbytes)


CALLS = [append, rope, decode, evict]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("change,status", [
    ({"keys": None}, BUFFER), ({"values": None}, BUFFER), ({"page_table": None}, BUFFER), ({"keys": A + 8}, BUFFER),
    ({"values": A + 2}, BUFFER), ({"page_table": A + 2}, BUFFER), ({"mass": A + 1}, BUFFER), ({"positions": A + 2}, BUFFER),
    ({"dtype": 2}, EXTENT), ({"head_dim": 96}, EXTENT), ({"head_dim": 0}, EXTENT), ({"kv_heads": 0}, EXTENT),
    ({"kv_heads": 1025}, EXTENT), ({"page_slots": 0}, EXTENT), ({"page_slots": 8}, EXTENT), ({"page_slots": 24}, EXTENT),
    ({"page_slots": 1040}, EXTENT), ({"table_pages": 0}, EXTENT), ({"n_pages": 0}, EXTENT), ({"table_lanes": 0}, EXTENT),
    ({"table_pages": 1 << 28}, EXTENT), ({"page_stride": 4}, EXTENT), ({"head_stride": 0}, EXTENT), ({"slot_stride": 252}, EXTENT),
    ({"slot_stride": 128}, EXTENT), ({"table_lanes": 3}, GROUP)])
def test_a_cache_that_cannot_be_is_refused(ctx, call, change, status):
    assert call(ctx, cache(**change)) == status
    assert tb.lib().tatara_last_error_string(ctx)


@pytest.mark.parametrize("call", CALLS)
def test_lane_tables_are_checked(ctx, call):
    assert call(ctx, cache(), lanes=None) == BUFFER
    assert call(ctx, cache(), lanes=A + 4) == BUFFER
    assert call(ctx, cache(), n=0) == GROUP
    assert call(ctx, cache(table_lanes=1000), n=257) == GROUP
    assert call(None, cache()) == BUFFER


def test_append_refusals(ctx):
    c = cache()
    assert append(ctx, c, keys=None) == BUFFER and append(ctx, c, values=A + 8) == BUFFER
    assert append(ctx, c, starts=A + 2) == BUFFER
    assert append(ctx, c, row=252) == EXTENT and append(ctx, c, row=508) == EXTENT and append(ctx, c, head=12) == EXTENT
    assert append(ctx, c, rows=0) == EXTENT and append(ctx, c, rows=5) == EXTENT      # one row per lane without row_starts
    assert append(ctx, c, starts=A, rows=(1 << 28) + 1) == EXTENT


def test_rope_refusals(ctx):
    assert rope(ctx, cache(), projection=None) == BUFFER and rope(ctx, cache(), projection=A + 8) == BUFFER
    assert rope(ctx, cache(), q=A + 2) == BUFFER
    assert rope(ctx, cache(dtype=1)) == EXTENT and rope(ctx, cache(kv_heads=4)) == EXTENT and rope(ctx, cache(head_dim=128)) == EXTENT
    assert rope(ctx, cache(), stride=9208) == EXTENT and rope(ctx, cache(), query=4092) == EXTENT and rope(ctx, cache(), stride=9218) == EXTENT


def test_decode_refusals(ctx):
    c = cache()
    for bad in ({"q": None}, {"out": None}, {"scratch": None}, {"q": A + 2}, {"gate": A + 1}, {"out": A + 1}, {"scratch": A + 8}):
        assert decode(ctx, c, **bad) == BUFFER, bad
    for bad in ({"q_heads": 0}, {"q_heads": 15}, {"q_heads": 34, "stride": 1 << 20}, {"stride": 4094}, {"stride": 4097},
                {"scale": float("nan")}, {"scale": float("inf")}):
        assert decode(ctx, c, **bad) == EXTENT, bad
    assert decode(ctx, c, max_keys=0) == RANGE and decode(ctx, c, max_keys=1601) == RANGE
    assert decode(ctx, cache(table_pages=40000), max_keys=262145) == RANGE
    need = tb.decode_paged_scratch_bytes(c, 4, 1000, 16)
    assert decode(ctx, c, nbytes=need - 1) == SCRATCH


def test_evict_refusals(ctx):
    c = cache()
    assert evict(ctx, cache(mass=None)) == BUFFER and evict(ctx, cache(positions=None)) == BUFFER
    assert evict(ctx, c, scratch=None) == BUFFER and evict(ctx, c, scratch=A + 4) == BUFFER
    assert evict(ctx, c, keep=0, sink=0, recent=0) == EXTENT and evict(ctx, c, keep=103) == EXTENT
    assert evict(ctx, c, sink=0xFFFFFFFF, recent=2) == EXTENT
    assert evict(ctx, c, max_keys=0) == RANGE and evict(ctx, c, max_keys=1601) == RANGE
    assert evict(ctx, c, nbytes=tb.paged_evict_scratch_bytes(c, 4, 1000, 500) - 1) == SCRATCH
    assert evict(ctx, c, keep=1000) == OK      # no lane can hold more: nothing is launched


def test_lanes_step_refusals(ctx):
    step = tb.lib().tatara_paged_lanes_step
    assert step(None, None, A, 1, 1, 1) == BUFFER and step(ctx, None, None, 1, 1, 1) == BUFFER and step(ctx, None, A + 4, 1, 1, 1) == BUFFER
    assert step(ctx, None, A, 0, 1, 1) == GROUP and step(ctx, None, A, 257, 1, 1) == GROUP
    assert step(ctx, None, A, 1, 0, 1) == EXTENT and step(ctx, None, A, 1, 1, 262145) == EXTENT


def test_scratch_covers_every_shorter_lane_and_grows_with_the_mass():
    for kv_heads, dim, q_heads in ((2, 256, 16), (1, 64, 16), (8, 128, 32), (1024, 64, 1024)):
        c = cache(kv_heads=kv_heads, head_dim=dim, mass=None)
        sizes = [tb.decode_paged_scratch_bytes(c, 3, n, q_heads) for n in (1, 127, 128, 129, 1000, 9472, 9473, 100000, 262144)]
        assert sizes == sorted(sizes) and sizes[0] > 0
        held = cache(kv_heads=kv_heads, head_dim=dim)
        assert tb.decode_paged_scratch_bytes(held, 3, 1000, q_heads) >= sizes[4] + 3 * 1000 * q_heads * 4
    assert tb.decode_paged_scratch_bytes(cache(), 3, 262145, 16) == 0
    assert tb.paged_evict_scratch_bytes(cache(), 3, 1000, 100) >= 6 * 100 * 8
    assert tb.paged_evict_scratch_bytes(cache(), 3, 1000, 900) >= 6 * 100 * 8


def test_descriptor_checks():
    c = Cache([5, 40], 2, 64, device="cpu")
    got = tb.paged_cache(c.keys, c.values, c.table, mass=c.mass, positions=c.positions)
    assert (got.n_pages, got.kv_heads, got.page_slots, got.head_dim) == tuple(c.keys.shape)
    assert got.capacity == c.table.shape[1] * 16 and got.table_lanes == 2 and got.dtype == 0
    s = Cache([5, 40], 2, 64, slot_major=True, dtype=torch.float16, device="cpu")
    got = tb.paged_cache(s.keys, s.values, s.table)
    assert (got.head_stride, got.slot_stride, got.dtype, got.mass) == (64, 128, 1, None)
    for bad in (lambda: tb.paged_cache(c.keys, c.values[:3], c.table),
                lambda: tb.paged_cache(c.keys, c.values.half(), c.table),
                lambda: tb.paged_cache(c.keys.float(), c.values.float(), c.table),
                lambda: tb.paged_cache(c.keys.transpose(2, 3), c.values.transpose(2, 3), c.table),
                lambda: tb.paged_cache(c.keys, c.values, c.table.long()),
                lambda: tb.paged_cache(c.keys, c.values, c.table, mass=c.mass[:, :, :16]),
                lambda: tb.paged_cache(c.keys, c.values, c.table, mass=c.mass.double()),
                lambda: tb.paged_cache(c.keys, c.values, c.table, positions=c.positions.long())):
        with pytest.raises(ValueError):
            bad()


def test_eviction_definition_on_a_small_cache():
    """The definition itself, by hand: slots 0 and 1 are guarded, 7 is the newest, equals go to the lower slot."""
    c = Cache([8], 1, 64, device="cpu")
    c.mass[0, 0, :8] = torch.tensor([0.0, 0.0, 5.0, 1.0, 1.0, 9.0, 1.0, 0.0])
    after = evict_definition(c, keep=5, sink=2, recent=1)     # stay: 0, 1, 7, 5, 2
    assert after.positions[0, 0, :8].tolist() == [0, 1, 2, 5, 7, 5, 6, 7]
    assert after.mass[0, 0, :8].tolist() == [0.0, 0.0, 5.0, 9.0, 0.0, 9.0, 1.0, 0.0]
    assert same_cache(evict_definition(c, keep=8, sink=0, recent=0), c)
