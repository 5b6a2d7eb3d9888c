// Eviction from a paged KV cache by accumulated attention weight.
//
// Per (lane, kv head) of n > keep slots: rank key = 0xFFFFFFFF for guarded slots, else the mass mapped to an unsigned integer of the
// same order; the keep largest stay, equals by the lower slot.  A slot below `keep` that is given up is a hole, a slot from
// `keep` on that stays is a donor; there are as many of one as of the other and the j-th hole takes the j-th donor's row.  Attention
// does not ask for an order of the slots, so nothing else moves: 8 x head_dim bytes for each pair against the whole kept part
// for a cache that is kept in order.
//
// The keep-th key is found by a radix search (digits of 11, 11 and 10 bits), then both lists are written in the order of the slots, then
// paged_move_kernel copies the rows.  Lanes of up to 16384 slots are searched by one CTA a head in one launch, up to 16 keys in the registers
// of each thread.  Longer ones are shared out over many CTAs that never wait for one another: a launch for each digit, with the heads'
// histograms added up in memory between them.  Bound: HBM (the rows) for a large cut, the latency of the search's steps for
// a small one.
#include "paged.cuh"

namespace tb {

constexpr uint32_t kSelThreads = 1024, kSelWarps = kSelThreads / 32, kSelBins = 2048, kSelMaxKeys = 16;
constexpr uint32_t kMoveThreads = 256, kMoveBatch = 2;

struct PagedEvictParams {
    PagedView cache;
    const tatara_paged_lane* lanes;
    uint32_t* counts;    // [row]: pairs of a (lane, kv head)
    uint32_t* holes;     // [row][room]
    uint32_t* donors;    // [row][room]
    // of lanes that several CTAs search
    uint32_t* hist;      // [row][3][kSelBins]
    uint2* found;        // [row][4]: after d digits, the threshold's digits and how many keys with them are still to be found
    uint4* blocks;       // [row][row_blocks]: a CTA's counts
    uint32_t* keys;      // [row][key_stride]
    uint32_t row_blocks, key_stride;
    uint32_t n_lanes, max_keys, keep, sink, recent;
    uint32_t room;       // no row has more pairs
    uint32_t move_blocks, warp_pairs;   // blocks of the second kernel for each row, pairs of a warp (at most 32)
};

struct SelectShared {                // beside the histograms
    uint4 warp_counts[kSelWarps];
    uint32_t warp_sum[kSelWarps];
    uint32_t bin, above;             // the digit that holds the threshold, keys beyond it
};

// An unsigned integer in the order of the floats: negative ones reversed, not-a-number first, the guarded slots' value left free.
__device__ __forceinline__ uint32_t rank_key(float mass) {
    if (mass != mass) return 0u;
    const uint32_t u = __float_as_uint(mass + 0.0f);     // -0 counts as 0
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t warp_inclusive(uint32_t v) {
#pragma unroll
    for (uint32_t off = 1; off < 32; off <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, off);
        if ((threadIdx.x & 31u) >= off) v += u;
    }
    return v;
}

// A thread's keys: of slots first + 32 j, j < each <= kKeys, as far as they are below n.  A warp owns a run of 32 * each slots, lane by lane,
// so ballots count in the order of the slots.
template <uint32_t kKeys>
struct SlotKeys {
    uint32_t key[kKeys];
    uint32_t unit, first, n, each;
};

// The keys of a lane's slots out of mass and positions.
template <uint32_t kKeys>
__device__ __forceinline__ void rank_slots(const PagedEvictParams& p, uint64_t plane, uint32_t position, SlotKeys<kKeys>& s) {
    float mass[kKeys];
    uint32_t where[kKeys];
#pragma unroll
    for (uint32_t j = 0; j < kKeys; ++j) {
        const uint32_t slot = s.first + 32u * j;
        if (j >= s.each) break;
        mass[j] = slot < s.n ? __ldcg(p.cache.mass + plane + slot) : 0.0f;
    }
    if (p.recent != 0u) {
#pragma unroll
        for (uint32_t j = 0; j < kKeys; ++j) {
            const uint32_t slot = s.first + 32u * j;
            if (j >= s.each) break;
            where[j] = slot < s.n ? __ldcg(p.cache.positions + plane + slot) : 0u;
        }
    }
    const uint32_t newest = p.recent > position ? 0u : position - p.recent + 1u;   // positions from here on are guarded
#pragma unroll
    for (uint32_t j = 0; j < kKeys; ++j) {
        if (j >= s.each) break;
        const bool guarded = s.first + 32u * j < p.sink || (p.recent != 0u && where[j] >= newest);
        s.key[j] = guarded ? 0xFFFFFFFFu : rank_key(mass[j]);
    }
}

__device__ __forceinline__ uint32_t digit_bins(uint32_t digit) { return digit == 2u ? 1024u : 2048u; }

// Counts digit `digit` of the keys whose earlier digits are `prefix`.
template <uint32_t kKeys>
__device__ __forceinline__ void add_digit(uint32_t* hist, const SlotKeys<kKeys>& s, uint32_t digit, uint32_t prefix) {
    const uint32_t shift = digit == 0u ? 21u : digit == 1u ? 10u : 0u, above = digit == 1u ? 21u : 10u, mask = digit_bins(digit) - 1u;
    const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
    for (uint32_t j = 0; j < kKeys; ++j) {
        if (j >= s.each) break;
        const bool in = s.first + 32u * j < s.n && (digit == 0u || s.key[j] >> above == prefix);
        const uint32_t bin = (s.key[j] >> shift) & mask;
        // (a run of guarded, untouched or equal slots falls into one bin: one addition for all of them)
        const bool full = __all_sync(0xffffffffu, in);
        const uint32_t its = __shfl_sync(0xffffffffu, bin, 0);
        if (full && __all_sync(0xffffffffu, bin == its)) {
            if (lane == 0u) atomicAdd(&hist[bin], 32u);
        } else if (in) {
            atomicAdd(&hist[bin], 1u);
        }
    }
}

// The next digit of the threshold: the bin, counted from the top, that holds the `want`-th key.  Moves prefix and want on.  By all threads; ends
// with a barrier.
__device__ __forceinline__ void find_digit(const uint32_t* hist, bool in_memory, uint32_t digit, SelectShared& sh, uint32_t& prefix, uint32_t& want) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, bins = digit_bins(digit);
    // thread t takes bins 2t and 2t + 1, counted from the top
    const uint32_t top = bins - 2u - threadIdx.x * 2u;
    const bool holds = threadIdx.x * 2u < bins;
    uint2 v = make_uint2(0u, 0u);
    if (holds) v = in_memory ? __ldcg(reinterpret_cast<const uint2*>(hist + top)) : *reinterpret_cast<const uint2*>(hist + top);
    const uint32_t incl = warp_inclusive(v.x + v.y);
    if (lane == 31u) sh.warp_sum[warp] = incl;
    __syncthreads();
    const uint32_t sums = warp_inclusive(sh.warp_sum[lane]);
    const uint32_t before = __shfl_sync(0xffffffffu, sums, warp == 0u ? 0u : warp - 1u);
    const uint32_t above = (warp == 0u ? 0u : before) + incl - v.x - v.y;
    if (holds && above < want && want <= above + v.x + v.y) {
        const bool upper = want <= above + v.y;
        sh.bin = top + (upper ? 1u : 0u);
        sh.above = upper ? above : above + v.y;
    }
    __syncthreads();
    prefix = digit == 0u ? sh.bin : (prefix << (digit == 1u ? 11 : 10)) | sh.bin;
    want -= sh.above;
}

// Keys above `prefix` stay, and of those equal to it the first `want` by slot.  Four counts, of the keys above and of those equal below slot `keep`
// (x, y) and from it on (z, w), give each warp its place in both lists.
template <uint32_t kKeys>
__device__ __forceinline__ uint4 count_slots(const PagedEvictParams& p, const SlotKeys<kKeys>& s, uint32_t prefix) {
    uint32_t low = 0u, high = 0u;   // those above | those equal << 16
#pragma unroll
    for (uint32_t j = 0; j < kKeys; ++j) {
        const uint32_t slot = s.first + 32u * j;
        if (j >= s.each) break;
        const uint32_t one = slot >= s.n || s.key[j] < prefix ? 0u : s.key[j] == prefix ? 0x10000u : 1u;
        low += slot < p.keep ? one : 0u;
        high += slot < p.keep ? 0u : one;
    }
    low = __reduce_add_sync(0xffffffffu, low);
    high = __reduce_add_sync(0xffffffffu, high);
    return make_uint4(low & 0xFFFFu, low >> 16, high & 0xFFFFu, high >> 16);
}
// The counts of the warps before this one, and of the whole CTA.
__device__ __forceinline__ uint4 counts_before(SelectShared& sh, const uint4& mine, uint4& all) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    if (lane == 0u) sh.warp_counts[warp] = mine;
    __syncthreads();
    const uint4 of = sh.warp_counts[lane];
    const uint4 sum = make_uint4(warp_inclusive(of.x), warp_inclusive(of.y), warp_inclusive(of.z), warp_inclusive(of.w));
    all = make_uint4(__shfl_sync(0xffffffffu, sum.x, 31), __shfl_sync(0xffffffffu, sum.y, 31), __shfl_sync(0xffffffffu, sum.z, 31),
                     __shfl_sync(0xffffffffu, sum.w, 31));
    const uint32_t prior = warp == 0u ? 0u : warp - 1u;
    const uint4 b = make_uint4(__shfl_sync(0xffffffffu, sum.x, prior), __shfl_sync(0xffffffffu, sum.y, prior), __shfl_sync(0xffffffffu, sum.z, prior),
                               __shfl_sync(0xffffffffu, sum.w, prior));
    return warp == 0u ? make_uint4(0u, 0u, 0u, 0u) : b;
}

// The warp's part of both lists.  b: the counts of all warps before it; c: its own.
template <uint32_t kKeys>
__device__ __forceinline__ void write_lists(const PagedEvictParams& p, uint32_t row, const SlotKeys<kKeys>& s, uint32_t prefix, uint32_t want, const uint4& b,
                                            const uint4& c) {
    const uint32_t lane = threadIdx.x & 31u;
    // ties below `keep` come before those from it on, so the first `want` of all are min(want, y) below and the rest above
    uint32_t tie_rank = b.y + b.w;
    uint32_t hole_at = min(p.keep, s.unit) - b.x - min(want, b.y), donor_at = b.z + min(want, b.y + b.w) - min(want, b.y);
    uint32_t* hole_list = p.holes + uint64_t(row) * p.room;
    uint32_t* donor_list = p.donors + uint64_t(row) * p.room;
    const uint32_t below = (1u << lane) - 1u;
    const bool all_ties = tie_rank + c.y + c.w <= want, split = !all_ties && tie_rank < want;   // what of the warp's ties stays: all, some, none
    if (!split && s.unit + 32u * s.each <= p.keep) {
        // the warp's slots all lie below `keep`: holes only
#pragma unroll
        for (uint32_t j = 0; j < kKeys; ++j) {
            if (j >= s.each) break;
            const bool hole = s.key[j] < prefix || (!all_ties && s.key[j] == prefix);
            const uint32_t hb = __ballot_sync(0xffffffffu, hole), h = hole_at + __popc(hb & below);
            if (hole && h < p.room) hole_list[h] = s.first + 32u * j;
            hole_at += __popc(hb);
        }
    } else if (!split && s.unit >= p.keep) {
        // or from it on: donors only
#pragma unroll
        for (uint32_t j = 0; j < kKeys; ++j) {
            if (j >= s.each) break;
            const bool donor = s.first + 32u * j < s.n && (s.key[j] > prefix || (all_ties && s.key[j] == prefix));
            const uint32_t db = __ballot_sync(0xffffffffu, donor), d = donor_at + __popc(db & below);
            if (donor && d < p.room) donor_list[d] = s.first + 32u * j;
            donor_at += __popc(db);
        }
    } else {
#pragma unroll 1
        for (uint32_t j = 0; j < s.each; ++j) {
            uint32_t mine = s.key[0];
#pragma unroll
            for (uint32_t i = 1; i < kKeys; ++i) mine = i == j ? s.key[i] : mine;
            const uint32_t slot = s.first + 32u * j;
            const bool tie = slot < s.n && mine == prefix;
            const uint32_t tied = __ballot_sync(0xffffffffu, tie);
            const bool kept = slot < s.n && (mine > prefix || (tie && tie_rank + __popc(tied & below) < want));
            tie_rank += __popc(tied);
            const bool hole = slot < p.keep && !kept, donor = slot >= p.keep && kept;       // (slots below `keep` all exist: n > keep)
            const uint32_t hb = __ballot_sync(0xffffffffu, hole), db = __ballot_sync(0xffffffffu, donor);
            const uint32_t h = hole_at + __popc(hb & below), d = donor_at + __popc(db & below);
            if (hole && h < p.room) hole_list[h] = slot;
            if (donor && d < p.room) donor_list[d] = slot;
            hole_at += __popc(hb);
            donor_at += __popc(db);
        }
    }
}

// ---- lanes of up to 16384 slots: one CTA a head --------------------------------------------
// Measured: 7 us for two heads of 4196 slots, 15 for 16384, 18 for 192 heads of up to 16000.
template <uint32_t kKeys>
__global__ void __launch_bounds__(kSelThreads, 1)
paged_select_kernel(const __grid_constant__ PagedEvictParams p) {
    __shared__ SelectShared sh;
    __shared__ __align__(8) uint32_t hist[3][kSelBins];
    const uint32_t row = blockIdx.x, lane_row = row / p.cache.kv_heads, head = row - lane_row * p.cache.kv_heads;
    for (uint32_t i = threadIdx.x; i < 3u * kSelBins; i += kSelThreads) (&hist[0][0])[i] = 0u;
    wait_for_predecessor();
    release_dependents();
    const uint2 l = __ldcg(reinterpret_cast<const uint2*>(p.lanes + lane_row));   // keys, position
    if (l.x > p.max_keys || l.x <= p.keep) {
        if (l.x > p.max_keys && threadIdx.x == 0) latch_out_of_range(p.cache, lane_row);
        if (threadIdx.x == 0) p.counts[row] = 0u;
        return;
    }
    SlotKeys<kKeys> s;
    s.n = l.x;
    s.each = (s.n + kSelThreads - 1u) / kSelThreads;       // as many as the lane's slots need
    s.unit = (threadIdx.x >> 5) * 32u * s.each;
    s.first = s.unit + (threadIdx.x & 31u);
    rank_slots(p, plane_row(p.cache, lane_row, head), l.y, s);
    __syncthreads();
    uint32_t prefix = 0u, want = p.keep;
#pragma unroll
    for (uint32_t digit = 0; digit < 3u; ++digit) {
        add_digit(hist[digit], s, digit, prefix);
        __syncthreads();
        find_digit(hist[digit], false, digit, sh, prefix, want);
    }
    uint4 all;
    const uint4 c = count_slots(p, s, prefix), b = counts_before(sh, c, all);
    if (threadIdx.x == 0u) p.counts[row] = p.keep - all.x - min(want, all.y);
    write_lists(p, row, s, prefix, want, b, c);
}

// ---- longer lanes: row_blocks CTAs a head, 1024 kKeys slots each -----------------------------
// Six short launches, each staged while its predecessor finishes: the histograms are cleared; the keys are made, kept and their first
// digit counted; a digit is found and the next one counted, twice; the last digit is found and each CTA's counts are written down; the lists are
// written.  Measured: 22 us for two heads of 262144 slots on 128 SMs, 18 for 40000, the launches included; sharing a head within one
// cluster of 16 CTAs took 26 and had to have 16 SMs free at the same time.
struct WideBlock {
    uint32_t row, block;
    uint2 lane;       // keys, position
    bool works;       // the lane is to be trimmed and this CTA holds some of its slots
};
template <uint32_t kKeys>
__device__ __forceinline__ WideBlock wide_block(const PagedEvictParams& p, SlotKeys<kKeys>& s) {
    WideBlock w;
    w.row = blockIdx.x / p.row_blocks;
    w.block = blockIdx.x - w.row * p.row_blocks;
    w.lane = __ldcg(reinterpret_cast<const uint2*>(p.lanes + w.row / p.cache.kv_heads));
    s.n = w.lane.x;
    s.each = kKeys;
    s.unit = (w.block * kSelWarps + (threadIdx.x >> 5)) * 32u * kKeys;
    s.first = s.unit + (threadIdx.x & 31u);
    w.works = s.n <= p.max_keys && s.n > p.keep && w.block * kSelThreads * kKeys < s.n;
    return w;
}
template <uint32_t kKeys>
__device__ __forceinline__ void read_keys(const PagedEvictParams& p, uint32_t row, SlotKeys<kKeys>& s) {
#pragma unroll
    for (uint32_t j = 0; j < kKeys; ++j) {
        const uint32_t slot = s.first + 32u * j;
        s.key[j] = slot < s.n ? __ldcg(p.keys + uint64_t(row) * p.key_stride + slot) : 0u;
    }
}
__device__ __forceinline__ void clear_hist(uint32_t* hist) {
    for (uint32_t i = threadIdx.x; i < kSelBins; i += kSelThreads) hist[i] = 0u;
}
__device__ __forceinline__ void add_up(uint32_t* to, const uint32_t* hist) {
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kSelBins; i += kSelThreads)
        if (hist[i] != 0u) atomicAdd(to + i, hist[i]);     // whole numbers: any order gives the same sum
}

__global__ void __launch_bounds__(kSelThreads)
paged_search_clear_kernel(const __grid_constant__ PagedEvictParams p) {
    wait_for_predecessor();
    release_dependents();
    for (uint32_t i = threadIdx.x; i < 3u * kSelBins; i += kSelThreads) p.hist[uint64_t(blockIdx.x) * 3u * kSelBins + i] = 0u;
}

template <uint32_t kKeys>
__global__ void __launch_bounds__(kSelThreads, 1)
paged_search_keys_kernel(const __grid_constant__ PagedEvictParams p) {
    __shared__ uint32_t hist[kSelBins];
    clear_hist(hist);
    wait_for_predecessor();
    release_dependents();
    SlotKeys<kKeys> s;
    const WideBlock w = wide_block(p, s);
    const uint32_t lane_row = w.row / p.cache.kv_heads, head = w.row - lane_row * p.cache.kv_heads;
    if (w.block == 0u && threadIdx.x == 0u) {
        if (s.n > p.max_keys) latch_out_of_range(p.cache, lane_row);
        if (!w.works) p.counts[w.row] = 0u;
    }
    if (!w.works) return;
    rank_slots(p, plane_row(p.cache, lane_row, head), w.lane.y, s);
#pragma unroll
    for (uint32_t j = 0; j < kKeys; ++j) {
        const uint32_t slot = s.first + 32u * j;
        if (slot < s.n) p.keys[uint64_t(w.row) * p.key_stride + slot] = s.key[j];
    }
    __syncthreads();
    add_digit(hist, s, 0u, 0u);
    add_up(p.hist + uint64_t(w.row) * 3u * kSelBins, hist);
}

// Finds digit `digit` and counts the next one, or, after the last, the CTA's slots.
template <uint32_t kKeys>
__global__ void __launch_bounds__(kSelThreads, 1)
paged_search_digit_kernel(const __grid_constant__ PagedEvictParams p, const uint32_t digit) {
    __shared__ SelectShared sh;
    __shared__ uint32_t next[kSelBins];
    clear_hist(next);
    wait_for_predecessor();
    release_dependents();
    SlotKeys<kKeys> s;
    const WideBlock w = wide_block(p, s);
    if (!w.works) return;
    read_keys(p, w.row, s);
    uint2 so_far = make_uint2(0u, p.keep);
    if (digit != 0u) so_far = __ldcg(p.found + w.row * 4u + digit);
    uint32_t* hist = p.hist + (uint64_t(w.row) * 3u + digit) * kSelBins;
    find_digit(hist, true, digit, sh, so_far.x, so_far.y);
    if (w.block == 0u && threadIdx.x == 0u) p.found[w.row * 4u + digit + 1u] = so_far;
    if (digit != 2u) {
        add_digit(next, s, digit + 1u, so_far.x);
        add_up(hist + kSelBins, next);
    } else {
        uint4 all;
        (void)counts_before(sh, count_slots(p, s, so_far.x), all);
        if (threadIdx.x == 0u) p.blocks[uint64_t(w.row) * p.row_blocks + w.block] = all;
    }
}

template <uint32_t kKeys>
__global__ void __launch_bounds__(kSelThreads, 1)
paged_search_lists_kernel(const __grid_constant__ PagedEvictParams p) {
    __shared__ SelectShared sh;
    wait_for_predecessor();
    release_dependents();
    SlotKeys<kKeys> s;
    const WideBlock w = wide_block(p, s);
    if (!w.works) return;
    read_keys(p, w.row, s);
    const uint2 found = __ldcg(p.found + w.row * 4u + 3u);
    // the counts of the CTAs before this one, and those below `keep` of all
    const uint32_t lane = threadIdx.x & 31u, used = (s.n + kSelThreads * kKeys - 1u) / (kSelThreads * kKeys);
    uint4 prior = make_uint4(0u, 0u, 0u, 0u);
    uint2 total = make_uint2(0u, 0u);
    for (uint32_t i = lane; i < used; i += 32u) {
        const uint4 of = __ldcg(p.blocks + uint64_t(w.row) * p.row_blocks + i);
        total.x += of.x;
        total.y += of.y;
        if (i < w.block) prior = make_uint4(prior.x + of.x, prior.y + of.y, prior.z + of.z, prior.w + of.w);
    }
    prior = make_uint4(__reduce_add_sync(0xffffffffu, prior.x), __reduce_add_sync(0xffffffffu, prior.y), __reduce_add_sync(0xffffffffu, prior.z),
                       __reduce_add_sync(0xffffffffu, prior.w));
    total = make_uint2(__reduce_add_sync(0xffffffffu, total.x), __reduce_add_sync(0xffffffffu, total.y));
    if (w.block == 0u && threadIdx.x == 0u) p.counts[w.row] = p.keep - total.x - min(found.y, total.y);
    uint4 all;
    const uint4 c = count_slots(p, s, found.x), b = counts_before(sh, c, all);
    write_lists(p, w.row, s, found.x, found.y, make_uint4(b.x + prior.x, b.y + prior.y, b.z + prior.z, b.w + prior.w), c);
}

// A warp takes p.warp_pairs pairs: each lane looks up one pair's slots and pages, then kChunks lanes together copy a pair's rows, with
// the loads of kMoveBatch steps on their way before the first store.  Bound by HBM: rows of 512 bytes move at 5.7 TB/s read and written
// (36 us from 262144 slots to 65536), of 256 bytes at 5.1; eight steps at a time are slower (79 against 70 us in all), fewer
// pairs to a look-up too (73).
template <uint32_t kChunks>   // 16-byte chunks of a row
__global__ void __launch_bounds__(kMoveThreads)
paged_move_kernel(const __grid_constant__ PagedEvictParams p) {
    constexpr uint32_t kTogether = 32u / kChunks;   // pairs of a step
    const uint32_t row = blockIdx.x / p.move_blocks, block = blockIdx.x - row * p.move_blocks;
    const uint32_t lane_row = row / p.cache.kv_heads, head = row - lane_row * p.cache.kv_heads, lane = threadIdx.x & 31u;
    wait_for_predecessor();
    const uint32_t pairs = __ldcg(p.counts + row), first = (block * (kMoveThreads / 32u) + (threadIdx.x >> 5)) * p.warp_pairs;
    if (first >= pairs) return;
    const uint32_t mine = min(p.warp_pairs, pairs - first);
    uint64_t src = 0, dst = 0;
    uint32_t ok = 0u;
    if (lane < mine) {
        const uint64_t at = uint64_t(row) * p.room + first + lane;
        const uint32_t to = __ldcg(p.holes + at), from = __ldcg(p.donors + at);
        const bool there = slot_offset(p.cache, lane_row, head, from, src);
        if (slot_offset(p.cache, lane_row, head, to, dst) && there) {
            ok = 1u;
            const uint64_t plane = plane_row(p.cache, lane_row, head);
            p.cache.mass[plane + to] = __ldcg(p.cache.mass + plane + from);
            if (p.cache.positions != nullptr) p.cache.positions[plane + to] = __ldcg(p.cache.positions + plane + from);
        }
    }
    const uint32_t sub = lane / kChunks, offset = (lane % kChunks) * 16u;
    for (uint32_t j0 = 0; j0 < mine; j0 += kMoveBatch * kTogether) {
        uint4 k[kMoveBatch], v[kMoveBatch];
        uint64_t to[kMoveBatch];
        bool live[kMoveBatch];
#pragma unroll
        for (uint32_t i = 0; i < kMoveBatch; ++i) {
            const uint32_t j = j0 + i * kTogether + sub;
            const uint64_t from = __shfl_sync(0xffffffffu, src, j & 31u) + offset;
            to[i] = __shfl_sync(0xffffffffu, dst, j & 31u) + offset;
            live[i] = (__shfl_sync(0xffffffffu, ok, j & 31u) & (j < mine ? 1u : 0u)) != 0u;
            if (live[i]) {
                k[i] = __ldcs(reinterpret_cast<const uint4*>(p.cache.keys + from));
                v[i] = __ldcs(reinterpret_cast<const uint4*>(p.cache.values + from));
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kMoveBatch; ++i) {
            if (live[i]) {
                __stcs(reinterpret_cast<uint4*>(p.cache.keys + to[i]), k[i]);
                __stcs(reinterpret_cast<uint4*>(p.cache.values + to[i]), v[i]);
            }
        }
    }
}

static uint32_t evict_room(uint32_t max_keys, uint32_t keep) { return max_keys <= keep ? 0u : keep < max_keys - keep ? keep : max_keys - keep; }

// Where the parts of the scratch lie, in bytes.
struct PagedEvictLayout {
    uint32_t room, row_blocks, thread_keys;   // row_blocks 0: one CTA a head
    uint64_t lists, hist, found, blocks, keys, bytes;
};
static PagedEvictLayout evict_layout(uint64_t rows, uint32_t max_keys, uint32_t keep) {
    const auto whole = [](uint64_t n) { return (n + 255u) / 256u * 256u; };
    PagedEvictLayout l{};
    l.room = evict_room(max_keys, keep);
    l.lists = whole(rows * 4u);
    l.bytes = l.hist = whole(l.lists + rows * l.room * 8u);
    if (l.room == 0u || max_keys <= kSelThreads * kSelMaxKeys) return l;
    // few slots a CTA while that takes no more than twice the SMs, else few CTAs
    l.thread_keys = rows * ((max_keys + 4095u) / 4096u) <= 2u * kSmCount ? 4u : kSelMaxKeys;
    l.row_blocks = (max_keys + kSelThreads * l.thread_keys - 1u) / (kSelThreads * l.thread_keys);
    l.found = whole(l.hist + rows * 3u * kSelBins * 4u);
    l.blocks = whole(l.found + rows * 4u * 8u);
    l.keys = whole(l.blocks + rows * l.row_blocks * 16u);
    l.bytes = l.keys + rows * max_keys * 4u;
    return l;
}

} // namespace tb

using namespace tb;

extern "C" uint64_t tatara_paged_evict_scratch_bytes(const tatara_paged_cache* cache, uint32_t n_lanes, uint32_t max_keys,
                                                     uint32_t keep) {
    if (cache == nullptr || max_keys > TATARA_MAX_CONTEXT) return 0;
    return evict_layout(uint64_t(n_lanes) * cache->kv_heads, max_keys, keep).bytes;
}

extern "C" tatara_status tatara_paged_evict(tatara_ctx* ctx, void* stream, const tatara_paged_cache* cache,
                                            const tatara_paged_lane* lanes_device, uint32_t n_lanes, uint32_t max_keys,
                                            uint32_t keep, uint32_t sink, uint32_t recent, void* scratch,
                                            uint64_t scratch_bytes) {
    if (ctx == nullptr) return TATARA_INVALID_BUFFER;
    const tatara_status st = check_paged(ctx, cache, lanes_device, n_lanes);
    if (st != TATARA_OK) return st;
    if (cache->mass == nullptr || (recent != 0u && cache->positions == nullptr) || scratch == nullptr || !aligned(scratch, 16))
        return fail(ctx, TATARA_INVALID_BUFFER, "paged_evict: needs mass, positions for recent > 0, and scratch");
    if (keep == 0 || uint64_t(sink) + recent > keep)
        return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged_evict: keep of at least sink + recent slots");
    if (max_keys == 0 || max_keys > cache->table_pages * cache->page_slots || max_keys > TATARA_MAX_CONTEXT)
        return fail(ctx, TATARA_CONTEXT_OUT_OF_RANGE, "paged_evict: max_keys beyond the page table or the longest context");
    const uint64_t rows = uint64_t(n_lanes) * cache->kv_heads;
    const PagedEvictLayout layout = evict_layout(rows, max_keys, keep);
    if (scratch_bytes < layout.bytes) return fail(ctx, TATARA_SCRATCH_TOO_SMALL, "paged_evict: scratch");
    if (layout.room == 0u) return TATARA_OK;   // no lane of max_keys slots holds more than keep; none is looked at
    PagedEvictParams p{};
    p.cache = paged_view(ctx, *cache);
    p.lanes = lanes_device;
    p.n_lanes = n_lanes;
    p.max_keys = max_keys;
    p.keep = keep;
    p.sink = sink;
    p.recent = recent;
    auto* base = static_cast<uint8_t*>(scratch);
    p.room = layout.room;
    p.counts = static_cast<uint32_t*>(scratch);
    p.holes = reinterpret_cast<uint32_t*>(base + layout.lists);
    p.donors = p.holes + rows * p.room;
    p.hist = reinterpret_cast<uint32_t*>(base + layout.hist);
    p.found = reinterpret_cast<uint2*>(base + layout.found);
    p.blocks = reinterpret_cast<uint4*>(base + layout.blocks);
    p.keys = reinterpret_cast<uint32_t*>(base + layout.keys);
    p.row_blocks = layout.row_blocks;
    p.key_stride = max_keys;
    // A few pairs go to many warps, many pairs 32 to a warp: one look-up for all lanes.
    const uint64_t spread = rows * p.room / (uint64_t(ctx->sm_count) * 32u);
    p.warp_pairs = spread < 4u ? 4u : spread > 32u ? 32u : uint32_t(spread);
    const uint32_t block_pairs = kMoveThreads / 32u * p.warp_pairs;
    p.move_blocks = (p.room + block_pairs - 1u) / block_pairs;
    if (rows * p.move_blocks > 0x7FFFFFFFull) return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged_evict: grid");
    const DeviceGuard guard(ctx);
    const auto s = static_cast<cudaStream_t>(stream);
    tatara_status launched;
    if (layout.row_blocks == 0u) {
        const uint32_t keys = (max_keys + kSelThreads - 1u) / kSelThreads;   // of a thread, at most
        auto select = keys <= 2u ? paged_select_kernel<2> : keys <= 4u ? paged_select_kernel<4> : keys <= 8u ? paged_select_kernel<8> : paged_select_kernel<16>;
        (void)launch_staged(select, dim3(uint32_t(rows)), kSelThreads, 0u, s, p);
        launched = check_launch(ctx, "paged_evict");
    } else {
        const bool few = layout.thread_keys == 4u;
        const dim3 grid(uint32_t(rows * layout.row_blocks));
        (void)launch_staged(paged_search_clear_kernel, dim3(uint32_t(rows)), kSelThreads, 0u, s, p);
        launched = check_launch(ctx, "paged_evict: clear");
        if (launched == TATARA_OK) {
            (void)launch_staged(few ? paged_search_keys_kernel<4> : paged_search_keys_kernel<kSelMaxKeys>, grid, kSelThreads, 0u, s, p);
            launched = check_launch(ctx, "paged_evict: keys");
        }
        for (uint32_t digit = 0; digit < 3u && launched == TATARA_OK; ++digit) {
            (void)launch_staged(few ? paged_search_digit_kernel<4> : paged_search_digit_kernel<kSelMaxKeys>, grid, kSelThreads, 0u, s, p, digit);
            launched = check_launch(ctx, "paged_evict: digit");
        }
        if (launched == TATARA_OK) {
            (void)launch_staged(few ? paged_search_lists_kernel<4> : paged_search_lists_kernel<kSelMaxKeys>, grid, kSelThreads, 0u, s, p);
            launched = check_launch(ctx, "paged_evict: lists");
        }
    }
    if (launched != TATARA_OK) return launched;
    auto move = cache->head_dim == 64u ? paged_move_kernel<8> : cache->head_dim == 128u ? paged_move_kernel<16> : paged_move_kernel<32>;
    (void)launch_staged(move, dim3(uint32_t(rows * p.move_blocks)), kMoveThreads, 0u, s, p);
    return check_launch(ctx, "paged_evict: move");
}
