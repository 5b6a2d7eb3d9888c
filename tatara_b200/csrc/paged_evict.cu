// Eviction from a paged KV cache by accumulated attention weight.
//
// Per (lane, kv head) of n > keep slots: rank key = 0xFFFFFFFF for guarded slots, else the mass mapped to an unsigned integer of the
// same order; the keep largest stay, equals by the lower slot.  A slot below `keep` that is given up is a hole, a slot from
// `keep` on that stays is a donor; there are as many of one as of the other and the j-th hole takes the j-th donor's row.  Attention
// does not ask for an order of the slots, so nothing else moves: 8 x head_dim bytes for each pair against the whole kept part
// for a cache that is kept in order.
//
// Two launches.  paged_select_kernel finds the keep-th key by a radix search (11 + 11 + 10 bits) and writes the two lists: up
// to 16 keys sit in the registers of each thread, so mass and positions are read once, and up to 16 CTAs of a cluster share a head
// and add their histograms over distributed shared memory.  paged_move_kernel copies the rows.  Bound: HBM (the rows) for a
// large cut, the latency of the search's steps for a small one.
#include "paged.cuh"

#include <cooperative_groups.h>

namespace tb {

namespace cg = cooperative_groups;

constexpr uint32_t kSelThreads = 1024, kSelWarps = kSelThreads / 32, kSelBins = 2048, kSelMaxCluster = 16, kSelMaxKeys = 16;
static_assert(kSelThreads * kSelMaxKeys * kSelMaxCluster >= TATARA_MAX_CONTEXT, "one cluster holds the longest lane");
constexpr uint32_t kMoveThreads = 256, kMoveBatch = 2;

struct PagedEvictParams {
    PagedView cache;
    const tatara_paged_lane* lanes;
    uint32_t* counts;    // [row]: pairs of a (lane, kv head)
    uint32_t* holes;     // [row][room]
    uint32_t* donors;    // [row][room]
    uint32_t n_lanes, max_keys, keep, sink, recent;
    uint32_t room;       // no row has more pairs
    uint32_t cluster;
    uint32_t move_blocks, warp_pairs;   // blocks of the second kernel for each row, pairs of a warp (at most 32)
};

struct SelectShared {
    uint32_t hist[3][kSelBins];
    uint4 warp_counts[kSelWarps];
    uint4 counts;                    // of this CTA, read by the others of the cluster
    uint32_t slice[kSelBins];        // this CTA's share of the cluster's bins, summed up from the top; read by the others
    uint32_t slice_total[kSelMaxCluster];   // of every CTA, written by each
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

// Measured: 7 us for two heads of 4196 slots, 23 us for two of 262144 (32 SMs; a digit's step 4.5 us, of which 2.6 are spent between the
// CTAs), 19 us for 192 heads of up to 16000.
// kKeys: the most keys of a thread; `each` of them are used, as many as the lane's slots need.  A warp owns a run of 32 * each slots,
// lane by lane, so ballots count in the order of the slots.
template <uint32_t kKeys>
__global__ void __launch_bounds__(kSelThreads, 1)
paged_select_kernel(const __grid_constant__ PagedEvictParams p) {
    __shared__ __align__(16) SelectShared s;
    cg::cluster_group cluster = cg::this_cluster();
    const auto meet = [&] {            // the CTAs that share a head
        if (p.cluster == 1u) __syncthreads(); else cluster.sync();
    };
    const uint32_t rank = blockIdx.x % p.cluster, row = blockIdx.x / p.cluster;
    const uint32_t lane_row = row / p.cache.kv_heads, head = row - lane_row * p.cache.kv_heads;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    for (uint32_t i = threadIdx.x; i < 3u * kSelBins; i += kSelThreads) (&s.hist[0][0])[i] = 0u;
    wait_for_predecessor();
    release_dependents();
    const uint2 l = __ldcg(reinterpret_cast<const uint2*>(p.lanes + lane_row));   // keys, position
    const uint32_t n = l.x;
    if (n > p.max_keys || n <= p.keep) {                                          // (the same for every CTA of the cluster)
        if (n > p.max_keys && rank == 0u && threadIdx.x == 0) latch_out_of_range(p.cache, lane_row);
        if (rank == 0u && threadIdx.x == 0) p.counts[row] = 0u;
        return;
    }
    const uint32_t each = (n + p.cluster * kSelThreads - 1u) / (p.cluster * kSelThreads);
    const uint32_t unit = (rank * kSelWarps + warp) * 32u * each, first = unit + lane;            // the thread's slots: first + 32 j
    const uint64_t plane = plane_row(p.cache, lane_row, head);

    // ---- keys into registers; a slot that is not there gets no key
    uint32_t key[kKeys];
    {
        float mass[kKeys];
        uint32_t where[kKeys];
#pragma unroll
        for (uint32_t j = 0; j < kKeys; ++j) {
            const uint32_t slot = first + 32u * j;
            if (j >= each) break;
            mass[j] = slot < n ? __ldcg(p.cache.mass + plane + slot) : 0.0f;
        }
        if (p.recent != 0u) {
#pragma unroll
            for (uint32_t j = 0; j < kKeys; ++j) {
                const uint32_t slot = first + 32u * j;
                if (j >= each) break;
                where[j] = slot < n ? __ldcg(p.cache.positions + plane + slot) : 0u;
            }
        }
        const uint32_t newest = p.recent > l.y ? 0u : l.y - p.recent + 1u;   // positions from here on are guarded
#pragma unroll
        for (uint32_t j = 0; j < kKeys; ++j) {
            if (j >= each) break;
            const bool guarded = first + 32u * j < p.sink || (p.recent != 0u && where[j] >= newest);
            key[j] = guarded ? 0xFFFFFFFFu : rank_key(mass[j]);
        }
    }
    __syncthreads();

    // ---- radix search: the digits of the keep-th largest key, the largest digit first
    uint32_t prefix = 0u, want = p.keep;     // `want` keys are still to be found among those with this prefix
#pragma unroll
    for (uint32_t digit = 0; digit < 3u; ++digit) {
        const uint32_t shift = digit == 0u ? 21u : digit == 1u ? 10u : 0u, bins = digit == 2u ? 1024u : 2048u;
#pragma unroll
        for (uint32_t j = 0; j < kKeys; ++j) {
            if (j >= each) break;
            const bool in = first + 32u * j < n && (digit == 0u || key[j] >> (digit == 1u ? 21u : 10u) == prefix);
            const uint32_t bin = (key[j] >> shift) & (bins - 1u);
            // (a run of guarded, untouched or equal slots falls into one bin: one addition for all of them)
            const bool full = __all_sync(0xffffffffu, in);
            const uint32_t its = __shfl_sync(0xffffffffu, bin, 0);
            if (full && __all_sync(0xffffffffu, bin == its)) {
                if (lane == 0u) atomicAdd(&s.hist[digit][bin], 32u);
            } else if (in) {
                atomicAdd(&s.hist[digit][bin], 1u);
            }
        }
        meet();
        if (p.cluster == 1u) {
            // thread t takes bins 2t and 2t + 1, counted from the top
            const uint32_t top = bins - 2u - threadIdx.x * 2u;
            const bool holds = threadIdx.x * 2u < bins;
            uint2 v = make_uint2(0u, 0u);
            if (holds) v = *reinterpret_cast<const uint2*>(&s.hist[digit][top]);
            const uint32_t incl = warp_inclusive(v.x + v.y);
            if (lane == 31u) s.warp_sum[warp] = incl;
            __syncthreads();
            const uint32_t sums = warp_inclusive(s.warp_sum[lane]);
            const uint32_t before = __shfl_sync(0xffffffffu, sums, warp == 0u ? 0u : warp - 1u);
            const uint32_t above = (warp == 0u ? 0u : before) + incl - v.x - v.y;
            if (holds && above < want && want <= above + v.x + v.y) {
                const bool upper = want <= above + v.y;
                s.bin = top + (upper ? 1u : 0u);
                s.above = upper ? above : above + v.y;
            }
        } else {
            // Each CTA adds up one slice of the bins over the cluster (the slice of rank 0 is the topmost), sums it up from the top and
            // tells the others its total: a few hundred bytes cross between SMs in place of every histogram to every CTA.
            const uint32_t width = bins / p.cluster, slice_top = bins - 1u - rank * width;
            uint32_t mine = 0u;
            if (threadIdx.x < width)
                for (uint32_t r = 0; r < p.cluster; ++r) mine += *cluster.map_shared_rank(&s.hist[digit][slice_top - threadIdx.x], r);
            const uint32_t incl = warp_inclusive(mine);
            if (lane == 31u) s.warp_sum[warp] = incl;
            __syncthreads();
            const uint32_t sums = warp_inclusive(s.warp_sum[lane]);
            const uint32_t before = __shfl_sync(0xffffffffu, sums, warp == 0u ? 0u : warp - 1u);
            if (threadIdx.x < width) s.slice[threadIdx.x] = (warp == 0u ? 0u : before) + incl;
            const uint32_t all = __shfl_sync(0xffffffffu, sums, 31);
            if (threadIdx.x < p.cluster) *cluster.map_shared_rank(&s.slice_total[rank], threadIdx.x) = all;
            cluster.sync();
            const uint32_t of_rank = warp_inclusive(lane < p.cluster ? s.slice_total[lane] : 0u);
            const uint32_t owner = __ffs(__ballot_sync(0xffffffffu, want <= of_rank)) - 1u;       // (the last rank's sum is at least `want`)
            const uint32_t over = __shfl_sync(0xffffffffu, of_rank, owner == 0u ? 0u : owner - 1u);
            const uint32_t above = owner == 0u ? 0u : over;
            if (threadIdx.x < width) {
                const uint32_t to = above + *cluster.map_shared_rank(&s.slice[threadIdx.x], owner);
                const uint32_t from = threadIdx.x == 0u ? above : above + *cluster.map_shared_rank(&s.slice[threadIdx.x - 1u], owner);
                if (from < want && want <= to) {
                    s.bin = bins - 1u - owner * width - threadIdx.x;
                    s.above = from;
                }
            }
        }
        __syncthreads();
        prefix = digit == 0u ? s.bin : (prefix << (digit == 1u ? 11 : 10)) | s.bin;
        want -= s.above;
    }

    // ---- keys above `prefix` stay, and of those equal to it the first `want` by slot.  Four counts of every warp, below slot `keep` (x, y)
    // and from it on (z, w), those above and those equal, give each warp its place in both lists.
    uint32_t low_counts = 0u, high_counts = 0u;   // those above | those equal << 16
#pragma unroll
    for (uint32_t j = 0; j < kKeys; ++j) {
        const uint32_t slot = first + 32u * j;
        if (j >= each) break;
        const uint32_t one = slot >= n || key[j] < prefix ? 0u : key[j] == prefix ? 0x10000u : 1u;
        low_counts += slot < p.keep ? one : 0u;
        high_counts += slot < p.keep ? 0u : one;
    }
    low_counts = __reduce_add_sync(0xffffffffu, low_counts);
    high_counts = __reduce_add_sync(0xffffffffu, high_counts);
    const uint4 c = make_uint4(low_counts & 0xFFFFu, low_counts >> 16, high_counts & 0xFFFFu, high_counts >> 16);
    if (lane == 0u) s.warp_counts[warp] = c;
    __syncthreads();
    const uint4 of = s.warp_counts[lane];
    const uint4 sum = make_uint4(warp_inclusive(of.x), warp_inclusive(of.y), warp_inclusive(of.z), warp_inclusive(of.w));
    if (threadIdx.x == 31u) s.counts = sum;
    const uint32_t prior = warp == 0u ? 0u : warp - 1u;
    uint4 b = make_uint4(__shfl_sync(0xffffffffu, sum.x, prior), __shfl_sync(0xffffffffu, sum.y, prior), __shfl_sync(0xffffffffu, sum.z, prior),
                         __shfl_sync(0xffffffffu, sum.w, prior));
    if (warp == 0u) b = make_uint4(0u, 0u, 0u, 0u);
    meet();
    const uint4 other = lane < p.cluster ? *cluster.map_shared_rank(&s.counts, lane) : make_uint4(0u, 0u, 0u, 0u);
    const bool prior_rank = lane < rank;
    b.x += __reduce_add_sync(0xffffffffu, prior_rank ? other.x : 0u);
    b.y += __reduce_add_sync(0xffffffffu, prior_rank ? other.y : 0u);
    b.z += __reduce_add_sync(0xffffffffu, prior_rank ? other.z : 0u);
    b.w += __reduce_add_sync(0xffffffffu, prior_rank ? other.w : 0u);
    if (rank == 0u && warp == 0u) {
        const uint32_t over = __reduce_add_sync(0xffffffffu, other.x), ties = __reduce_add_sync(0xffffffffu, other.y);
        if (lane == 0u) p.counts[row] = p.keep - over - min(want, ties);
    }
    // ties below `keep` come before those from it on, so the first `want` of all are min(want, y) below and the rest above
    uint32_t tie_rank = b.y + b.w;
    uint32_t hole_at = min(p.keep, unit) - b.x - min(want, b.y), donor_at = b.z + min(want, b.y + b.w) - min(want, b.y);
    uint32_t* hole_list = p.holes + uint64_t(row) * p.room;
    uint32_t* donor_list = p.donors + uint64_t(row) * p.room;
    const uint32_t below = (1u << lane) - 1u;
    const bool all_ties = tie_rank + c.y + c.w <= want, split = !all_ties && tie_rank < want;   // what of the warp's ties stays: all, some, none
    if (!split && unit + 32u * each <= p.keep) {
        // the warp's slots all lie below `keep`: holes only
#pragma unroll
        for (uint32_t j = 0; j < kKeys; ++j) {
            if (j >= each) break;
            const bool hole = key[j] < prefix || (!all_ties && key[j] == prefix);
            const uint32_t hb = __ballot_sync(0xffffffffu, hole), h = hole_at + __popc(hb & below);
            if (hole && h < p.room) hole_list[h] = first + 32u * j;
            hole_at += __popc(hb);
        }
    } else if (!split && unit >= p.keep) {
        // or from it on: donors only
#pragma unroll
        for (uint32_t j = 0; j < kKeys; ++j) {
            if (j >= each) break;
            const bool donor = first + 32u * j < n && (key[j] > prefix || (all_ties && key[j] == prefix));
            const uint32_t db = __ballot_sync(0xffffffffu, donor), d = donor_at + __popc(db & below);
            if (donor && d < p.room) donor_list[d] = first + 32u * j;
            donor_at += __popc(db);
        }
    } else {
#pragma unroll 1
        for (uint32_t j = 0; j < each; ++j) {
            uint32_t mine = key[0];
#pragma unroll
            for (uint32_t i = 1; i < kKeys; ++i) mine = i == j ? key[i] : mine;
            const uint32_t slot = first + 32u * j;
            const bool tie = slot < n && mine == prefix;
            const uint32_t tied = __ballot_sync(0xffffffffu, tie);
            const bool kept = slot < n && (mine > prefix || (tie && tie_rank + __popc(tied & below) < want));
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
    if (p.cluster != 1u) cluster.sync();   // nobody leaves while its counters are read
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

} // namespace tb

using namespace tb;

extern "C" uint64_t tatara_paged_evict_scratch_bytes(const tatara_paged_cache* cache, uint32_t n_lanes, uint32_t max_keys,
                                                     uint32_t keep) {
    if (cache == nullptr) return 0;
    const uint64_t rows = uint64_t(n_lanes) * cache->kv_heads;
    return (rows * 4u + 255u) / 256u * 256u + rows * evict_room(max_keys, keep) * 8u;
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
    if (scratch_bytes < tatara_paged_evict_scratch_bytes(cache, n_lanes, max_keys, keep))
        return fail(ctx, TATARA_SCRATCH_TOO_SMALL, "paged_evict: scratch");
    PagedEvictParams p{};
    p.cache = paged_view(ctx, *cache);
    p.lanes = lanes_device;
    p.n_lanes = n_lanes;
    p.max_keys = max_keys;
    p.keep = keep;
    p.sink = sink;
    p.recent = recent;
    p.room = evict_room(max_keys, keep);
    if (p.room == 0u) return TATARA_OK;   // no lane can hold more than keep
    p.counts = static_cast<uint32_t*>(scratch);
    p.holes = p.counts + (rows * 4u + 255u) / 256u * 64u;
    p.donors = p.holes + rows * p.room;
    // As few CTAs as hold a head's keys 16 to a thread: below 16384 slots none has to wait for another.
    p.cluster = 1u;
    while (p.cluster * kSelThreads * kSelMaxKeys < max_keys) p.cluster *= 2u;
    const uint32_t keys = (max_keys + p.cluster * kSelThreads - 1u) / (p.cluster * kSelThreads);   // of a thread, at most
    auto select = keys <= 2u ? paged_select_kernel<2> : keys <= 4u ? paged_select_kernel<4> : keys <= 8u ? paged_select_kernel<8> : paged_select_kernel<16>;
    // A few pairs go to many warps, many pairs 32 to a warp: one look-up for all lanes.
    const uint64_t spread = rows * p.room / (uint64_t(ctx->sm_count) * 32u);
    p.warp_pairs = spread < 4u ? 4u : spread > 32u ? 32u : uint32_t(spread);
    const uint32_t block_pairs = kMoveThreads / 32u * p.warp_pairs;
    p.move_blocks = (p.room + block_pairs - 1u) / block_pairs;
    if (rows * p.move_blocks > 0x7FFFFFFFull) return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged_evict: grid");
    const DeviceGuard guard(ctx);
    static bool configured[64] = {false};
    if (!configured[ctx->device & 63]) {
        if (cudaFuncSetAttribute(paged_select_kernel<16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
            return check_launch(ctx, "paged_evict: cluster attribute");
        configured[ctx->device & 63] = true;
    }
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(uint32_t(rows * p.cluster));
    cfg.blockDim = dim3(kSelThreads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    (void)cudaLaunchKernelEx(&cfg, select, p);
    const tatara_status launched = check_launch(ctx, "paged_evict");
    if (launched != TATARA_OK) return launched;
    auto move = cache->head_dim == 64u ? paged_move_kernel<8> : cache->head_dim == 128u ? paged_move_kernel<16> : paged_move_kernel<32>;
    (void)launch_staged(move, dim3(uint32_t(rows * p.move_blocks)), kMoveThreads, 0u, static_cast<cudaStream_t>(stream), p);
    return check_launch(ctx, "paged_evict: move");
}
