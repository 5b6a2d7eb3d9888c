// Eviction from a paged KV cache by accumulated attention weight.
//
// Per (lane, kv head) of n > keep slots: rank key = 0xFFFFFFFF for guarded slots, else the mass mapped to an unsigned integer of the
// same order; the keep largest stay, equals by the lower slot.  A slot below `keep` that is given up is a hole, a slot from
// `keep` on that stays is a donor; there are as many of one as of the other and the j-th hole takes the j-th donor's row.  Attention
// does not ask for an order of the slots, so nothing else moves: 8 x head_dim bytes for each pair against the whole kept part
// for a cache that is kept in order.
//
// Two launches.  paged_select_kernel finds the keep-th key by a radix search (11 + 11 + 10 bits) and writes the two lists;
// one cluster of CTAs holds the keys of a head in shared memory, so that mass and positions are read once and the histograms are added
// over distributed shared memory.  paged_move_kernel copies the rows.  Bound: HBM (the rows) for a large cut,
// latency of the search for a small one.
#include "paged.cuh"

#include <cooperative_groups.h>

namespace tb {

namespace cg = cooperative_groups;

constexpr uint32_t kSelThreads = 512, kSelWarps = kSelThreads / 32, kSelBins = 2048, kSelMaxCluster = 8;
constexpr uint32_t kSelMaxChunk = 49152;                 // keys of one CTA: 192 KiB beside the three histograms
constexpr uint32_t kMoveThreads = 256;

struct PagedEvictParams {
    PagedView cache;
    const tatara_paged_lane* lanes;
    uint32_t* counts;    // [row]: pairs of a (lane, kv head)
    uint32_t* holes;     // [row][room]
    uint32_t* donors;    // [row][room]
    uint32_t n_lanes, max_keys, keep, sink, recent;
    uint32_t room;       // no row has more pairs
    uint32_t cluster, chunk;
    uint32_t move_blocks, move_pairs;   // blocks of the second kernel for each row, pairs of a block
};

struct SelectShared {
    uint32_t hist[3][kSelBins];
    uint32_t ties, holes, donors;                        // of this CTA, read by the others of the cluster
    uint32_t warp_a[kSelWarps], warp_b[kSelWarps];
    uint32_t bin, above;                                 // the digit that holds the threshold, keys beyond it
};

// An unsigned integer in the order of the floats: negative ones reversed, not-a-number first, the guarded slots' value left free.
__device__ __forceinline__ uint32_t rank_key(float mass) {
    if (mass != mass) return 0u;
    const uint32_t u = __float_as_uint(mass + 0.0f);     // -0 counts as 0
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t block_exclusive(uint32_t mine, uint32_t* warp_sum, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint32_t incl = mine;
#pragma unroll
    for (uint32_t off = 1; off < 32; off <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
    }
    __syncthreads();
    if (lane == 31u) warp_sum[warp] = incl;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSelWarps; ++w) {
        if (w < warp) before += warp_sum[w];
        total += warp_sum[w];
    }
    return before + incl - mine;
}

__global__ void __launch_bounds__(kSelThreads, 1)
paged_select_kernel(const __grid_constant__ PagedEvictParams p) {
    extern __shared__ __align__(16) uint8_t sel_smem[];
    SelectShared& s = *reinterpret_cast<SelectShared*>(sel_smem);
    uint32_t* keys = reinterpret_cast<uint32_t*>(sel_smem + sizeof(SelectShared));
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = blockIdx.x % p.cluster, row = blockIdx.x / p.cluster;
    const uint32_t lane_row = row / p.cache.kv_heads, head = row - lane_row * p.cache.kv_heads;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    for (uint32_t i = threadIdx.x; i < 3u * kSelBins; i += kSelThreads) (&s.hist[0][0])[i] = 0u;
    if (threadIdx.x == 0) s.ties = s.holes = s.donors = 0u;
    wait_for_predecessor();
    release_dependents();
    const uint2 l = __ldcg(reinterpret_cast<const uint2*>(p.lanes + lane_row));   // keys, position
    const uint32_t n = l.x;
    if (n > p.max_keys || n <= p.keep) {                                          // (the same for every CTA of the cluster)
        if (n > p.max_keys && rank == 0u && threadIdx.x == 0) latch_out_of_range(p.cache, lane_row);
        if (rank == 0u && threadIdx.x == 0) p.counts[row] = 0u;
        return;
    }
    __syncthreads();
    const uint32_t base = rank * p.chunk, mine = base >= n ? 0u : min(p.chunk, n - base);
    const uint64_t plane = plane_row(p.cache, lane_row, head) + base;

    // ---- keys into shared memory, with the first digit's histogram
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < mine; i += kSelThreads) {
        const float mass = __ldcg(p.cache.mass + plane + i);
        bool guarded = base + i < p.sink;
        if (p.recent != 0u) guarded = guarded || uint64_t(__ldcg(p.cache.positions + plane + i)) + p.recent > l.y;
        const uint32_t key = guarded ? 0xFFFFFFFFu : rank_key(mass);
        keys[i] = key;
        atomicAdd(&s.hist[0][key >> 21], 1u);
    }

    // ---- radix search: the digits of the keep-th largest key, the largest digit first
    uint32_t prefix = 0u, want = p.keep;     // `want` keys are still to be found among those with this prefix
#pragma unroll
    for (uint32_t digit = 0; digit < 3u; ++digit) {
        const uint32_t shift = digit == 0u ? 21u : digit == 1u ? 10u : 0u, bins = digit == 2u ? 1024u : 2048u;
        if (digit != 0u) {
            const uint32_t upper = digit == 1u ? 21u : 10u;
            for (uint32_t i = threadIdx.x; i < mine; i += kSelThreads) {
                const uint32_t key = keys[i];
                if (key >> upper == prefix) atomicAdd(&s.hist[digit][(key >> shift) & (bins - 1u)], 1u);
            }
        }
        cluster.sync();
        // thread t adds up the cluster's bins 4t .. 4t+3, counted from the top
        uint32_t c[4] = {0u, 0u, 0u, 0u};
        const uint32_t top = bins - 4u - threadIdx.x * 4u;
        const bool holds = threadIdx.x * 4u < bins;
        if (holds) {
            for (uint32_t r = 0; r < p.cluster; ++r) {
                const uint4 v = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&s.hist[digit][top], r));
                c[0] += v.w; c[1] += v.z; c[2] += v.y; c[3] += v.x;
            }
        }
        uint32_t total;
        uint32_t above = block_exclusive(c[0] + c[1] + c[2] + c[3], s.warp_a, total);
        if (holds) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                if (above < want && want <= above + c[j]) {
                    s.bin = bins - 1u - (threadIdx.x * 4u + j);
                    s.above = above;
                }
                above += c[j];
            }
        }
        __syncthreads();
        prefix = digit == 0u ? s.bin : (prefix << (digit == 1u ? 11 : 10)) | s.bin;
        want -= s.above;
        __syncthreads();
    }
    // keys above `prefix` stay; of those equal to it the first `want`, by slot

    // ---- which stay: each warp owns a run of the chunk, in slot order
    const uint32_t run = (p.chunk / kSelWarps + 31u) / 32u * 32u, run0 = min(mine, warp * run), run1 = min(mine, run0 + run);
    uint32_t ties = 0u;
    for (uint32_t i = run0 + lane; i < run1; i += 32u) ties += keys[i] == prefix ? 1u : 0u;
    ties = __reduce_add_sync(0xffffffffu, ties);
    uint32_t total, tie_rank = block_exclusive(lane == 0u ? ties : 0u, s.warp_a, total);
    tie_rank = __shfl_sync(0xffffffffu, tie_rank, 0);
    if (threadIdx.x == 0) s.ties = total;
    cluster.sync();
    for (uint32_t r = 0; r < rank; ++r) tie_rank += *cluster.map_shared_rank(&s.ties, r);
    uint32_t holes = 0u, donors = 0u;
    for (uint32_t i0 = run0; i0 < run1; i0 += 32u) {
        const uint32_t i = i0 + lane;
        const uint32_t key = i < run1 ? keys[i] : 0u;
        const bool tie = i < run1 && key == prefix;
        const uint32_t tied = __ballot_sync(0xffffffffu, tie);
        const bool kept = i < run1 && (key > prefix || (tie && tie_rank + __popc(tied & ((1u << lane) - 1u)) < want));
        tie_rank += __popc(tied);
        const bool low = base + i < p.keep;
        if (i < run1) keys[i] = low ? (kept ? 0u : 1u) : (kept ? 2u : 0u);   // 1: hole, 2: donor
        holes += __popc(__ballot_sync(0xffffffffu, i < run1 && low && !kept));
        donors += __popc(__ballot_sync(0xffffffffu, i < run1 && !low && kept));
    }
    uint32_t hole_total, donor_total;
    uint32_t hole_at = block_exclusive(lane == 0u ? holes : 0u, s.warp_a, hole_total);
    uint32_t donor_at = block_exclusive(lane == 0u ? donors : 0u, s.warp_b, donor_total);
    hole_at = __shfl_sync(0xffffffffu, hole_at, 0);
    donor_at = __shfl_sync(0xffffffffu, donor_at, 0);
    if (threadIdx.x == 0) {
        s.holes = hole_total;
        s.donors = donor_total;
    }
    cluster.sync();
    uint32_t hole_sum = 0u;
    for (uint32_t r = 0; r < p.cluster; ++r) {
        const uint32_t h = *cluster.map_shared_rank(&s.holes, r);
        if (r < rank) {
            hole_at += h;
            donor_at += *cluster.map_shared_rank(&s.donors, r);
        }
        hole_sum += h;
    }
    if (rank == 0u && threadIdx.x == 0) p.counts[row] = hole_sum;
    uint32_t* hole_list = p.holes + uint64_t(row) * p.room;
    uint32_t* donor_list = p.donors + uint64_t(row) * p.room;
    for (uint32_t i0 = run0; i0 < run1; i0 += 32u) {
        const uint32_t i = i0 + lane, mark = i < run1 ? keys[i] : 0u, below = (1u << lane) - 1u;
        const uint32_t hb = __ballot_sync(0xffffffffu, mark == 1u), db = __ballot_sync(0xffffffffu, mark == 2u);
        const uint32_t h = hole_at + __popc(hb & below), d = donor_at + __popc(db & below);
        if (mark == 1u && h < p.room) hole_list[h] = base + i;
        if (mark == 2u && d < p.room) donor_list[d] = base + i;
        hole_at += __popc(hb);
        donor_at += __popc(db);
    }
    cluster.sync();   // nobody leaves while its counters are read
}

template <uint32_t kChunks>   // 16-byte chunks of a row
__global__ void __launch_bounds__(kMoveThreads)
paged_move_kernel(const __grid_constant__ PagedEvictParams p) {
    const uint32_t row = blockIdx.x / p.move_blocks, block = blockIdx.x - row * p.move_blocks;
    const uint32_t lane_row = row / p.cache.kv_heads, head = row - lane_row * p.cache.kv_heads;
    wait_for_predecessor();
    const uint32_t pairs = __ldcg(p.counts + row), first = block * p.move_pairs, last = min(pairs, first + p.move_pairs);
    const uint64_t plane = plane_row(p.cache, lane_row, head);
    const uint32_t chunk = threadIdx.x % kChunks;
    for (uint32_t j = first + threadIdx.x / kChunks; j < last; j += kMoveThreads / kChunks) {
        const uint32_t to = __ldcg(p.holes + uint64_t(row) * p.room + j), from = __ldcg(p.donors + uint64_t(row) * p.room + j);
        uint64_t src, dst;
        if (!slot_offset(p.cache, lane_row, head, from, src) || !slot_offset(p.cache, lane_row, head, to, dst)) continue;
        const uint4 k = __ldcs(reinterpret_cast<const uint4*>(p.cache.keys + src + chunk * 16u));
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p.cache.values + src + chunk * 16u));
        *reinterpret_cast<uint4*>(p.cache.keys + dst + chunk * 16u) = k;
        *reinterpret_cast<uint4*>(p.cache.values + dst + chunk * 16u) = v;
        if (chunk == 0u) {
            p.cache.mass[plane + to] = __ldcg(p.cache.mass + plane + from);
            if (p.cache.positions != nullptr) p.cache.positions[plane + to] = __ldcg(p.cache.positions + plane + from);
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
    // CTAs of a cluster: as few as hold the keys, more while SMs are idle and there is something to share.
    p.cluster = 1u;
    while (p.cluster < kSelMaxCluster &&
           ((max_keys + p.cluster - 1u) / p.cluster > kSelMaxChunk ||
            (rows * p.cluster * 2u <= uint64_t(ctx->sm_count) && max_keys / p.cluster > 2048u)))
        p.cluster *= 2u;
    p.chunk = ((max_keys + p.cluster - 1u) / p.cluster + 511u) / 512u * 512u;
    p.move_pairs = 4u * kMoveThreads / (cache->head_dim / 8u);
    p.move_blocks = (p.room + p.move_pairs - 1u) / p.move_pairs;
    if (rows * p.move_blocks > 0x7FFFFFFFull) return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged_evict: grid");
    const DeviceGuard guard(ctx);
    static bool configured[64] = {false};
    if (!configured[ctx->device & 63]) {
        if (cudaFuncSetAttribute(paged_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 sizeof(SelectShared) + kSelMaxChunk * 4u) != cudaSuccess)
            return check_launch(ctx, "paged_evict: shared memory attribute");
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
    cfg.dynamicSmemBytes = sizeof(SelectShared) + p.chunk * 4u;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    (void)cudaLaunchKernelEx(&cfg, paged_select_kernel, p);
    const tatara_status launched = check_launch(ctx, "paged_evict");
    if (launched != TATARA_OK) return launched;
    auto move = cache->head_dim == 64u ? paged_move_kernel<8> : cache->head_dim == 128u ? paged_move_kernel<16> : paged_move_kernel<32>;
    (void)launch_staged(move, dim3(uint32_t(rows * p.move_blocks)), kMoveThreads, 0u, static_cast<cudaStream_t>(stream), p);
    return check_launch(ctx, "paged_evict: move");
}
