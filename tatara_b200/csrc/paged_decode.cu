// Decode attention of one new token per lane over a paged KV cache, split over the cache's length and joined.
//
//   out[h] = sum_s p[h][s] v[s],  p[h][s] = softmax over s < keys of scale q[h].k[s]
//
// One pass over K and V with a running maximum and sum.  A lane's slots are cut into partitions; a work item
// (lane, kv head, partition) leaves, for every query head of the group, the un-normalised sum of its values, the
// maximum m of its scores (times log2 e) and the sum l of 2^(s - m) (f16: both sums times 2^14).  The join weighs the partitions with 2^(m - M),
// divides and applies the gate; where the cache carries a mass it adds 2^(s - M) / L of every slot, summed over the
// group, to it -- the scores were put aside in f32 by the first kernel, 4 bytes a head beside the 4 x head_dim of K and V.
//
// Bound: HBM.  A slot of a kv head is 4 x head_dim bytes and 4 x head_dim x group flops, 8 flops a byte for a group of 8, two orders
// below the tensor cores' balance, so mma.sync fragments out of shared memory carry the products and everything is
// arranged around the stream of K and V rows: every warp owns a ring of cp.async slices (16 slots of K and V) that runs ahead
// across items, and a slice never leaves its page, so one page-table entry (held by a lane, 32 slices at a time) serves it.
//
// The partition of a lane depends on its own slot count and the cache's geometry alone, each record is made in a fixed order and the join
// walks the records in order: a lane's bits are the same alone and in any batch.
#include "paged.cuh"

#include <cmath>

namespace tb {

constexpr uint32_t kPdWarps = 4, kPdThreads = kPdWarps * 32;
constexpr float kPdLog2e = 1.4426950408889634f;
constexpr uint32_t kJoinThreads = 256, kJoinWarps = kJoinThreads / 32, kJoinDims = 64;
constexpr uint32_t kJoinPhases = 8;           // the join adds partitions f, f + 8, ... in phase f, then the phases in order

// CTAs of the first kernel that share an SM: their rings fill its shared memory, their accumulators its registers.  Several, so
// that one streams while another joins its warps, fetches a query or looks up a page.  Four need 128 registers a thread, which head_dim 128
// does not fit in: 64 lanes of 1024 slots 56 us with four, 51 with three; one of 4096 9.6 and 8.8.
__host__ __device__ constexpr uint32_t pd_ctas(uint32_t head_dim) { return head_dim == 256u ? 2u : head_dim == 128u ? 3u : 4u; }
// The cut of a lane of n slots: partitions of at least pd_min_part slots, and no more items than one CTA for each SM (head_dim 256) or two
// take in one go.  Fewer and longer ones serve a batch better (fewer records), more of them would only help a lane alone.
__host__ __device__ inline uint32_t pd_per_wave(uint32_t kv_heads, uint32_t head_dim) {
    const uint32_t p = kSmCount * (head_dim == 256u ? 1u : 2u) / kv_heads;
    return p == 0u ? 1u : p;
}
// Slots of the shortest partition: its records (head_dim x group floats) stay below a sixteenth of its rows.
__host__ __device__ inline uint32_t pd_min_part(uint32_t group) { return group <= 8u ? 128u : 256u; }
struct PagedCut {
    uint32_t per_wave, least;
    __host__ __device__ uint32_t part_slots(uint32_t n) const {
        if (n <= per_wave * least) return least;
        return ((n + per_wave - 1u) / per_wave + kPagedSlice - 1u) / kPagedSlice * kPagedSlice;
    }
    __host__ __device__ uint32_t parts(uint32_t n) const {
        const uint32_t s = part_slots(n);
        return (n + s - 1u) / s;
    }
};

struct PagedDecodeParams {
    PagedView cache;
    const tatara_paged_lane* lanes;
    const uint8_t* q;
    const uint8_t* gate;
    uint8_t* out;
    float* sums;       // [lane][q head][part][head_dim]
    float2* stats;     // [lane][q head][part]: maximum (log2 units), sum of weights (2^kTopLog2 at the maximum)
    float* scores;     // [lane][kv head][max_keys rounded up to 16][group rounded up to 8], log2 units; null without a mass
    uint64_t query_stride;
    uint32_t n_lanes, max_keys, q_heads, group;
    PagedCut cut;
    uint32_t parts;        // parts of the longest lane: the stride of sums and stats
    uint32_t score_slots;  // max_keys rounded up to 16
    uint32_t units;        // places of a warp's ring
    uint32_t ahead_slots;  // most slots of a partition asked into L2 before the predecessor is waited for
    uint32_t page_slices, page_magic;   // slices of a page; floor(2^32 / page_slices) + 1
    float scale_log2e;
};

// kTopLog2: the weight of a warp's largest score, in log2 units.  f16 has 2^-14 as its smallest normal number and 2^-24 as its smallest step:
// with 2^14 for the largest, a weight is normal down to 2^-28 of it and what is lost stays below 2^-39 of it each, 2^-21 over the longest
// lane, where weights up to 1 would lose 2^-25 each.  Sums and their records all carry the factor, which the quotient takes out again.
template <typename T> struct Half;
template <> struct Half<__nv_bfloat16> {
    static constexpr float kTopLog2 = 0.0f;
    static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    static __device__ __forceinline__ uint32_t pack_down(float lo, float hi) {
        uint32_t v;
        asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
        return v;
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
    static __device__ __forceinline__ float load(const uint8_t* p) { return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p)); }
    static __device__ __forceinline__ void store(uint8_t* p, float v) { *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(v); }
};
template <> struct Half<__half> {
    static constexpr float kTopLog2 = 14.0f;
    static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    static __device__ __forceinline__ uint32_t pack_down(float lo, float hi) {
        uint32_t v;
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
        return v;
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
    static __device__ __forceinline__ float load(const uint8_t* p) { return __half2float(*reinterpret_cast<const __half*>(p)); }
    static __device__ __forceinline__ void store(uint8_t* p, float v) { *reinterpret_cast<__half*>(p) = __float2half_rn(v); }
};

// The work of every lane, counted by each CTA for itself: item_start[i] (n_lanes + 1 entries, count(slots) for each kv head) and
// the lanes' slot counts, 0 for a lane that is idle or refused.  Called by all threads.
template <uint32_t kThreads, typename Count>
__device__ __forceinline__ void scan_items(const PagedDecodeParams& p, uint32_t* item_start, uint32_t* lane_keys, uint32_t* warp_total, bool latch,
                                           Count count_of) {
    constexpr uint32_t kOwn = (TATARA_MAX_LANES + kThreads - 1u) / kThreads, kWarps = kThreads / 32u;
    const uint32_t first = threadIdx.x * kOwn, warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    uint32_t mine = 0, count[kOwn];
#pragma unroll
    for (uint32_t j = 0; j < kOwn; ++j) {
        const uint32_t i = first + j;
        uint32_t n = 0;
        if (i < p.n_lanes) {
            n = __ldcg(&p.lanes[i].keys);
            if (n > p.max_keys) {
                if (latch) latch_out_of_range(p.cache, i);
                n = 0;
            }
            lane_keys[i] = n;
        }
        count[j] = n == 0u ? 0u : count_of(n) * p.cache.kv_heads;
        mine += count[j];
    }
    uint32_t incl = mine;
#pragma unroll
    for (uint32_t off = 1; off < 32; off <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
    }
    if (lane == 31u) warp_total[warp] = incl;
    __syncthreads();
    uint32_t at = incl - mine;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w)
        if (w < warp) at += warp_total[w];
#pragma unroll
    for (uint32_t j = 0; j < kOwn; ++j) {
        if (first + j <= p.n_lanes) item_start[first + j] = at;
        at += count[j];
    }
    if (threadIdx.x == kThreads - 1u && kOwn * kThreads == p.n_lanes) item_start[p.n_lanes] = at;
    __syncthreads();
}

struct PagedItem {
    uint32_t lane, kv, part, begin, slots;   // slots of the partition, from slot `begin` of the lane
};
// Size(slots) is the length of a lane's pieces.
template <typename Size>
__device__ __forceinline__ PagedItem item_at(const PagedDecodeParams& p, const uint32_t* item_start, const uint32_t* lane_keys, uint32_t item, Size size_of) {
    uint32_t lo = 0, hi = p.n_lanes;   // last lane with item_start <= item (lanes without items share their successor's)
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) >> 1;
        if (item_start[mid] <= item) lo = mid; else hi = mid;
    }
    const uint32_t local = item - item_start[lo], n = lane_keys[lo], size = size_of(n);
    PagedItem it;
    it.lane = lo;
    it.part = local / p.cache.kv_heads;
    it.kv = local - it.part * p.cache.kv_heads;
    it.begin = it.part * size;
    it.slots = min(size, n - it.begin);
    return it;
}

constexpr uint32_t kPdItems = 128, kPdLookahead = 32;   // descriptors a CTA holds of its items; how far a warp reads ahead of its arithmetic

template <int D>
struct PdGeometry {
    // A unit is the K or the V rows of a step: one slice, or two where rows are short (what a step costs beside its rows weighs more there).
    static constexpr uint32_t kSlices = D == 64 ? 2 : 1, kStep = kSlices * kPagedSlice;
    static constexpr uint32_t kRow = D * 2, kChunks = D / 8, kUnit = kStep * kRow;
    static constexpr uint32_t kMaxUnits = 6;
    static constexpr uint32_t query(bool wide) { return wide ? 16u * kRow : 0u; }   // sixteen heads do not fit in registers beside their sums
    static constexpr uint32_t smem(uint32_t units, bool wide) { return query(wide) + kPdWarps * units * kUnit + kPdItems * 16 + kPdWarps * 8 * 8 + (2 * TATARA_MAX_LANES + 16) * 4; }
    // Places of a warp's ring when `ctas` share an SM: 64 KiB in flight an SM carry the full rate (6 TB/s), and more shared memory slows the
    // stream down, most likely because it comes out of L1, which the copies pass.  One lane of 262144 slots: 88 us at 96 to 128 KiB of rings
    // an SM, 93 - 99 at 160 to 192; 32 lanes of 16384: 189 us at 128 KiB, 205 at 192.
    static constexpr uint32_t units(uint32_t ctas) {
        const uint32_t u = 1u + 64u * 1024u / (ctas * kPdWarps * kUnit);
        return u < 2u ? 2u : u > kMaxUnits ? kMaxUnits : u;
    }
    static_assert(8 * D * 4 <= kUnit, "a warp's eight rows of the merge lie in one unit of its ring");
};

// 2^x; below 2^-126 zero
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The weight of a score that lies `below` (not above 0) from the maximum.  The factor goes to the difference, which is 0 at the maximum whatever
// its size; a large score would round it away.
template <typename T>
__device__ __forceinline__ float weight_of(float below) {
    if constexpr (Half<T>::kTopLog2 != 0.0f) below += Half<T>::kTopLog2;
    return exp2_fast(below);
}

// A weight for the second product, as the sum of two numbers of the cache's type: what lies below it and what that leaves, rounded.  One number would
// be off by half a step (bf16 2^-8, f16 2^-11 of the weight), two are by half a step of the rest: 2^-14.9 and 2^-20.6.  The second product's
// matrix instructions double: 84.0 -> 84.5 us for one lane of 262144 slots, 29.7 -> 30.4 for 96 short lanes of head_dim 64, 57.5 -> 59.0 for 16 lanes
// of 8192 with 16 query heads a kv head of 256.  The first is cut from a
// little less than the weight, so that the rest is above 0 too (f16: down to 2^-27 of the largest weight) and an infinite value stays one.
template <typename T>
__device__ __forceinline__ void two_terms(float p0, float p1, uint32_t& most, uint32_t& rest) {
    constexpr float kLess = 1.0f - 1.0f / 4096.0f;
    most = Half<T>::pack_down(p0 * kLess, p1 * kLess);
    const float2 m = Half<T>::unpack(most);
    rest = Half<T>::pack(p0 - m.x, p1 - m.y);
}

// kTiles: tiles of eight query heads, 1 or 2.  Measured with the join, 2 kv heads of 256, 16 query heads, bf16: one lane of 262144 slots 84 us
// (6.4 TB/s of K and V, bound by HBM), of 4096 8.9 us (latency), 32 lanes of 16384 185 us (5.8 TB/s); 16 lanes of 8192, 8 kv heads of
// 128 91 us (5.9 TB/s), of 64 52 us (5.2 TB/s, bound by the instructions of a step).  Short lanes of head_dim 64 are bound by what a
// partition costs beside its one step of each warp -- the join of the warps, its barriers, the record, the next query: 96 lanes of 40 to 1500,
// 12 kv heads, 30 us (4.0 TB/s).
template <typename T, int D, int kTiles>
__global__ void __launch_bounds__(kPdThreads, pd_ctas(D))
paged_decode_kernel(const __grid_constant__ PagedDecodeParams p) {
    using G = PdGeometry<D>;
    constexpr uint32_t kSteps = D / 16, kR = G::kSlices, kStep = G::kStep;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    uint8_t* query = smem + kPdWarps * p.units * G::kUnit;
    uint4* items = reinterpret_cast<uint4*>(query + G::query(kTiles == 2));    // {lane | kv << 16, part, begin, slots}
    float2* merge_ml = reinterpret_cast<float2*>(items + kPdItems);
    uint32_t* item_start = reinterpret_cast<uint32_t*>(merge_ml + kPdWarps * 8);
    uint32_t* lane_keys = item_start + TATARA_MAX_LANES + 1;
    uint32_t* warp_word = lane_keys + TATARA_MAX_LANES;
    const uint32_t ring = smem_u32(smem + warp * p.units * G::kUnit);
    const uint64_t policy = l2_evict_first_policy();
    // Before the predecessor is waited for, the first rows of this CTA's partition are asked into L2, so that HBM streams across the boundary
    // of the kernels.  The lane and the page table may be changing meanwhile; whatever they say, only rows inside the pools are asked for,
    // nothing lands in registers or shared memory, and both are read again after the wait.  Only where a CTA has one partition:
    // a batch keeps HBM busy by itself.
    if constexpr (kTiles == 1) {
        if (p.ahead_slots != 0u) {
            scan_items<kPdThreads>(p, item_start, lane_keys, warp_word, false, [&](uint32_t n) { return p.cut.parts(n); });
            if (blockIdx.x < item_start[p.n_lanes]) {
                const PagedItem it = item_at(p, item_start, lane_keys, blockIdx.x, [&](uint32_t n) { return p.cut.part_slots(n); });
                // a quarter of the partition at most: more competes in L2 with what is still streaming
                const uint32_t slices = min(p.ahead_slots, (it.slots + 3u) / 4u + kPagedSlice - 1u) / kPagedSlice;
                for (uint32_t s = threadIdx.x; s < slices; s += kPdThreads) {
                    const uint32_t slice = it.begin / kPagedSlice + s;
                    const uint32_t column = p.page_slices == 1u ? slice : __umulhi(slice, p.page_magic);
                    const uint32_t page = __ldcg(p.cache.page_table + uint64_t(it.lane) * p.cache.table_pages + column);
                    if (page >= p.cache.n_pages) continue;
                    const uint32_t rows = min(kPagedSlice, it.slots - s * kPagedSlice);
                    const uint64_t offset = page * p.cache.page_bytes + it.kv * p.cache.head_bytes + (slice - column * p.page_slices) * kPagedSlice * p.cache.slot_bytes;
                    if (p.cache.slot_bytes == G::kRow) {
                        l2_prefetch_bulk(p.cache.keys + offset, rows * G::kRow);
                        l2_prefetch_bulk(p.cache.values + offset, rows * G::kRow);
                    } else {
                        for (uint32_t r = 0; r < rows; ++r) {
                            l2_prefetch_bulk(p.cache.keys + offset + r * p.cache.slot_bytes, G::kRow);
                            l2_prefetch_bulk(p.cache.values + offset + r * p.cache.slot_bytes, G::kRow);
                        }
                    }
                }
            }
            __syncthreads();
        }
    }
    wait_for_predecessor();
    release_dependents();
    scan_items<kPdThreads>(p, item_start, lane_keys, warp_word, blockIdx.x == 0, [&](uint32_t n) { return p.cut.parts(n); });
    const uint32_t total = item_start[p.n_lanes];
    // this CTA's items are blockIdx.x, blockIdx.x + gridDim.x, ...; a thread describes one
    const uint32_t count = total > blockIdx.x ? (total - 1u - blockIdx.x) / gridDim.x + 1u : 0u;
    auto describe = [&](uint32_t k) {
        if (k >= count) return;
        const PagedItem it = item_at(p, item_start, lane_keys, blockIdx.x + k * gridDim.x, [&](uint32_t n) { return p.cut.part_slots(n); });
        items[k % kPdItems] = make_uint4(it.lane | it.kv << 16, it.part, it.begin, it.slots);
    };
    describe(threadIdx.x);
    __syncthreads();
    // ---- the warp's stream of units, ahead of the arithmetic and across items: K and V of its slices in turn.
    // Lane j looks after slice j % kR of the warp's steps kTurns * (turn / kTurns) + j / kR of an item: it fetches the slice's page, for the
    // next item an item early, and works out where the slice's rows lie; a step takes its slices' places from those lanes.
    constexpr uint32_t kTurns = 32u / kR;
    auto column_of = [&](uint32_t slice) { return p.page_slices == 1u ? slice : __umulhi(slice, p.page_magic); };   // of the lane's slice
    auto fetch_pages = [&](const uint4& it, uint32_t from) {
        const uint32_t slice = (warp + (from + lane / kR) * kPdWarps) * kR + lane % kR;
        return slice * kPagedSlice < it.w
                   ? __ldcg(p.cache.page_table + uint64_t(it.x & 0xFFFFu) * p.cache.table_pages + column_of(it.z / kPagedSlice + slice)) : 0u;
    };
    uint64_t places = 0;
    uint32_t missing = 0;          // bit j: lane j's page does not exist
    auto settle = [&](const uint4& it, uint32_t from, uint32_t page) {
        const uint32_t slice = (warp + (from + lane / kR) * kPdWarps) * kR + lane % kR, whole = it.z / kPagedSlice + slice;
        places = page * p.cache.page_bytes + (it.x >> 16) * p.cache.head_bytes + (whole - column_of(whole) * p.page_slices) * kPagedSlice * p.cache.slot_bytes;
        const bool none = slice * kPagedSlice < it.w && page >= p.cache.n_pages;
        missing = __ballot_sync(0xffffffffu, none);
        if (none) {
            places = 0;
            latch_out_of_range(p.cache, it.x & 0xFFFFu);
        }
    };
    uint32_t at = 0, turn = 0, issued = 0, consumed = 0, done_items = 0, next_pages = 0;
    uint32_t absent = 0;           // bits kR s ..: the pages of the K unit in ring place s that do not exist
    uint4 pi = make_uint4(0u, 0u, 0u, 0u);
    if (count != 0u) {
        pi = items[0];
        settle(pi, 0u, fetch_pages(pi, 0u));
        if (count > 1u) next_pages = fetch_pages(items[1], 0u);
    }
    uint32_t place_in = 0, place_out = 0;   // issued and consumed, modulo the ring's places
    uint32_t unit_place = 0;                // place of the K unit of the step under way
    bool second = false;
    uint64_t unit_offset[kR] = {};
    uint32_t unit_rows = 0;        // of the unit; slices of absent pages hold none
    bool unit_whole = false;
    const uint32_t chunk = lane % G::kChunks, row0 = lane / G::kChunks;
    const uint64_t row_step = (32u / G::kChunks) * p.cache.slot_bytes;
    // Asks for the next unit, if there is one and it may be asked for.
    auto issue = [&]() {
        if (!second) {
            // the next slice of this warp: of the current item, or of the next item that has one for it
            while (at < count && (warp + turn * kPdWarps) * kStep >= pi.w) {
                if (at + 1u >= count) { at = count; break; }
                if (at + 2u > done_items + kPdLookahead) return;
                ++at;
                turn = 0;
                pi = items[at % kPdItems];
                settle(pi, 0u, next_pages);
                if (at + 1u < count) next_pages = fetch_pages(items[(at + 1u) % kPdItems], 0u);
            }
        }
        if (at >= count) return;
        const uint32_t place = place_in;
        if (!second) {
            unit_place = place;
            if (turn != 0u && turn % kTurns == 0u) settle(pi, turn, fetch_pages(pi, turn));
            const uint32_t from = turn % kTurns * kR, gone = (missing >> from) & ((1u << kR) - 1u);
            unit_rows = min(kStep, pi.w - (warp + turn * kPdWarps) * kStep);
            unit_whole = unit_rows == kStep && gone == 0u;
            absent = (absent & ~(((1u << kR) - 1u) << (place * kR))) | gone << (place * kR);
#pragma unroll
            for (uint32_t i = 0; i < kR; ++i) unit_offset[i] = __shfl_sync(0xffffffffu, places, from + i);
            ++turn;
        }
        const uint8_t* pool = (second ? p.cache.values : p.cache.keys) + chunk * 16u + row0 * p.cache.slot_bytes;
        const uint32_t dst0 = ring + place * G::kUnit;
#pragma unroll
        for (uint32_t i = 0; i < kR; ++i) {
            const uint8_t* src = pool + unit_offset[i];
            const uint32_t dst1 = dst0 + i * kPagedSlice * G::kRow;
            if (unit_whole && p.cache.slot_bytes == G::kRow) {
#pragma unroll
                for (uint32_t r = 0; r < kPagedSlice; r += 32u / G::kChunks) {
                    const uint32_t row = r + row0;
                    cp_async_16(dst1 + row * G::kRow + ((chunk ^ (row & 7u)) << 4), src + r * G::kRow, 16u, policy);
                }
            } else if (unit_whole) {
#pragma unroll
                for (uint32_t r = 0; r < kPagedSlice; r += 32u / G::kChunks) {
                    const uint32_t row = r + row0;
                    cp_async_16(dst1 + row * G::kRow + ((chunk ^ (row & 7u)) << 4), src, 16u, policy);
                    src += row_step;
                }
            } else {
#pragma unroll 1
                for (uint32_t r = 0; r < kPagedSlice; r += 32u / G::kChunks) {
                    const uint32_t row = r + row0;
                    // rows behind the partition and absent pages read nothing: zeros
                    const bool live = i * kPagedSlice + row < unit_rows && ((absent >> (unit_place * kR + i)) & 1u) == 0u;
                    cp_async_16(dst1 + row * G::kRow + ((chunk ^ (row & 7u)) << 4), live ? src : pool, live ? 16u : 0u, policy);
                    src += row_step;
                }
            }
        }
        second = !second;
        cp_async_commit();
        ++issued;
        place_in = place_in + 1u == p.units ? 0u : place_in + 1u;
    };
    // Waits for the oldest unit: all but the issued - consumed - 1 youngest groups have to be there.
    auto await_unit = [&]() {
        const uint32_t younger = issued - consumed - 1u;
        if (younger == 1u) cp_async_wait<1>();
        else if (younger == 2u) cp_async_wait<2>();
        else if (younger == 0u) cp_async_wait<0>();
        else if (younger == 3u) cp_async_wait<3>();
        else if (younger == 4u) cp_async_wait<4>();
        else cp_async_wait<5>();
        __syncwarp();
    };
    auto release_unit = [&]() {
        __syncwarp();   // every lane is done with this unit before it is refilled
        ++consumed;
        place_out = place_out + 1u == p.units ? 0u : place_out + 1u;
    };
#pragma unroll 1
    for (uint32_t i = 1; i < p.units; ++i) issue();

    // Products run transposed, so that the 16 rows of the A operand are slots (scores) and dims (values) and the heads sit
    // in the eight columns: S^T = K Q^T, O^T += V^T P^T.  A by ldmatrix out of the XOR-swizzled unit, Q and P^T in registers.
    const uint32_t lm_j = lane >> 3, lm_r = lane & 7u;
    const uint32_t k_row = ((lm_j & 1u) * 8u + lm_r) * G::kRow, k_chunk = lm_j >> 1;
    const uint32_t v_row = ((lm_j >> 1) * 8u + lm_r) * G::kRow, v_chunk = lm_j & 1u;

    // Q as the B operand: of up to eight heads in registers, lane (g, t) holding dims 16 ks + 2t, +1 | +8, +9 of head g; of more, out of
    // shared memory step by step (rows swizzled as the units are).
    uint32_t qf[kTiles == 1 ? kSteps : 1][2];
    uint4 qn[kTiles == 2 ? D / 64 : 1];
    const uint32_t q_row = smem_u32(query) + ((lm_j >> 1) * 8u + lm_r) * G::kRow, q_chunk = lm_j & 1u;
    auto load_query = [&](const uint4& it) {
        const uint8_t* base = p.q + ((it.x & 0xFFFFu) * p.query_stride + uint64_t((it.x >> 16) * p.group) * D) * 2u;
        if constexpr (kTiles == 1) {
            const uint32_t* row = reinterpret_cast<const uint32_t*>(base + (g < p.group ? g : 0u) * (D * 2u));
#pragma unroll
            for (uint32_t ks = 0; ks < kSteps; ++ks) {
                qf[ks][0] = g < p.group ? __ldcg(row + ks * 8u + t) : 0u;
                qf[ks][1] = g < p.group ? __ldcg(row + ks * 8u + 4u + t) : 0u;
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < D / 64; ++i) {
                const uint32_t c = threadIdx.x + i * kPdThreads, head = c / G::kChunks;
                const uint32_t* from = reinterpret_cast<const uint32_t*>(base + (head < p.group ? c : 0u) * 16u);
                qn[i] = head < p.group ? make_uint4(__ldcg(from), __ldcg(from + 1), __ldcg(from + 2), __ldcg(from + 3)) : make_uint4(0u, 0u, 0u, 0u);
            }
        }
    };
    auto store_query = [&]() {
        if constexpr (kTiles == 2) {
#pragma unroll
            for (uint32_t i = 0; i < D / 64; ++i) {
                const uint32_t c = threadIdx.x + i * kPdThreads, head = c / G::kChunks;
                *reinterpret_cast<uint4*>(query + head * G::kRow + (((c % G::kChunks) ^ (head & 7u)) << 4)) = qn[i];
            }
        }
    };
    uint4 ci = make_uint4(0u, 0u, 0u, 0u);
    if (count != 0u) {
        ci = items[0];      // (a warp that has no share of the first items reads ahead of them already)
        load_query(ci);
        store_query();
    }
    if constexpr (kTiles == 2) __syncthreads();
    while (done_items < count) {
        float o[kTiles][kSteps][4], m[kTiles][2], l[kTiles][2];
#pragma unroll
        for (uint32_t nt = 0; nt < kTiles; ++nt) {
#pragma unroll
            for (uint32_t ks = 0; ks < kSteps; ++ks) o[nt][ks][0] = o[nt][ks][1] = o[nt][ks][2] = o[nt][ks][3] = 0.0f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.0f;
        }
        const uint32_t slots = ci.w;
        float* score_base = p.scores == nullptr ? nullptr
                            : p.scores + ((uint64_t(ci.x & 0xFFFFu) * p.cache.kv_heads + (ci.x >> 16)) * p.score_slots + ci.z) * (kTiles * 8u);

        for (uint32_t first = warp * kStep; first < slots; first += kPdWarps * kStep) {
            if (issued - consumed < p.units) issue();
            await_unit();
            const uint32_t kst = ring + place_out * G::kUnit + k_row;
            const uint32_t gone = absent >> (place_out * kR);
            float s[kR][kTiles][4], s2[kR][kTiles][4];
#pragma unroll
            for (uint32_t i = 0; i < kR; ++i) {
#pragma unroll
                for (uint32_t nt = 0; nt < kTiles; ++nt)
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) s[i][nt][e] = s2[i][nt][e] = 0.0f;
#pragma unroll
                for (uint32_t ks = 0; ks < kSteps; ++ks) {
                    uint32_t a0, a1, a2, a3;
                    // (the swizzle only touches the low three bits of a chunk: every fourth step shares its offset)
                    ldmatrix_x4(kst + i * kPagedSlice * G::kRow + ks / 4u * 128u + (((ks % 4u * 2u + k_chunk) ^ lm_r) << 4), a0, a1, a2, a3);
                    float (&sum)[kTiles][4] = ks % 2u == 0u ? s[i] : s2[i];   // two chains of additions
                    if constexpr (kTiles == 1) {
                        Half<T>::mma(sum[0], a0, a1, a2, a3, qf[ks][0], qf[ks][1]);
                    } else {
                        uint32_t b0, b1, b2, b3;
                        ldmatrix_x4(q_row + ks / 4u * 128u + (((ks % 4u * 2u + q_chunk) ^ lm_r) << 4), b0, b1, b2, b3);
                        Half<T>::mma(sum[0], a0, a1, a2, a3, b0, b1);
                        Half<T>::mma(sum[kTiles - 1], a0, a1, a2, a3, b2, b3);
                    }
                }
            }
            release_unit();
            issue();
            // lane (g, t): slots g and g + 8 of each slice, heads 2t and 2t + 1 of each tile
            bool higher = false;
#pragma unroll
            for (uint32_t i = 0; i < kR; ++i) {
                const bool exists = ((gone >> i) & 1u) == 0u;
                const uint32_t slot = first + i * kPagedSlice + g;
                const bool live0 = exists && slot < slots, live1 = exists && slot + 8u < slots;
#pragma unroll
                for (uint32_t nt = 0; nt < kTiles; ++nt) {
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        s[i][nt][e] = (e < 2 ? live0 : live1) ? (s[i][nt][e] + s2[i][nt][e]) * p.scale_log2e : -INFINITY;
                        higher = higher || s[i][nt][e] > m[nt][e & 1u];
                    }
                }
                if (score_base != nullptr) {
#pragma unroll
                    for (uint32_t nt = 0; nt < kTiles; ++nt) {
                        float* to = score_base + uint64_t(slot) * (kTiles * 8u) + nt * 8u + 2u * t;
                        if (slot < slots) *reinterpret_cast<float2*>(to) = make_float2(s[i][nt][0], s[i][nt][1]);
                        if (slot + 8u < slots) *reinterpret_cast<float2*>(to + 8u * kTiles * 8u) = make_float2(s[i][nt][2], s[i][nt][3]);
                    }
                }
            }
            // The maximum rises a few times at the start of an item and hardly ever later: only then is it looked for across the step's
            // slots and everything summed so far scaled down.
            if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
                for (uint32_t nt = 0; nt < kTiles; ++nt) {
                    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
                    for (uint32_t i = 0; i < kR; ++i) {
                        mx0 = fmaxf(mx0, fmaxf(s[i][nt][0], s[i][nt][2]));
                        mx1 = fmaxf(mx1, fmaxf(s[i][nt][1], s[i][nt][3]));
                    }
#pragma unroll
                    for (uint32_t off = 4; off < 32; off <<= 1) {
                        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
                        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
                    }
                    mx0 = fmaxf(m[nt][0], mx0);
                    mx1 = fmaxf(m[nt][1], mx1);
                    // (a column still at -inf has no sum yet: its factor 2^(-inf) is 0 against any finite base)
                    const float a0 = exp2_fast(m[nt][0] - (mx0 == -INFINITY ? 0.0f : mx0)), a1 = exp2_fast(m[nt][1] - (mx1 == -INFINITY ? 0.0f : mx1));
                    m[nt][0] = mx0;
                    m[nt][1] = mx1;
                    l[nt][0] *= a0;
                    l[nt][1] *= a1;
#pragma unroll
                    for (uint32_t ks = 0; ks < kSteps; ++ks) {
                        o[nt][ks][0] *= a0;
                        o[nt][ks][1] *= a1;
                        o[nt][ks][2] *= a0;
                        o[nt][ks][3] *= a1;
                    }
                }
            }
            uint32_t pb[kR][kTiles][2], rest[kR][kTiles][2];
#pragma unroll
            for (uint32_t nt = 0; nt < kTiles; ++nt) {
                const float b0 = m[nt][0] == -INFINITY ? 0.0f : m[nt][0], b1 = m[nt][1] == -INFINITY ? 0.0f : m[nt][1];
#pragma unroll
                for (uint32_t i = 0; i < kR; ++i) {
                    const float p0 = weight_of<T>(s[i][nt][0] - b0), p1 = weight_of<T>(s[i][nt][1] - b1);
                    const float p2 = weight_of<T>(s[i][nt][2] - b0), p3 = weight_of<T>(s[i][nt][3] - b1);
                    l[nt][0] += p0 + p2;
                    l[nt][1] += p1 + p3;
                    two_terms<T>(p0, p1, pb[i][nt][0], rest[i][nt][0]);
                    two_terms<T>(p2, p3, pb[i][nt][1], rest[i][nt][1]);
                    pb[i][nt][0] = movmatrix_trans(pb[i][nt][0]);            // slots 2t, 2t+1 of head g
                    pb[i][nt][1] = movmatrix_trans(pb[i][nt][1]);            // slots 2t+8, 2t+9 of head g
                    rest[i][nt][0] = movmatrix_trans(rest[i][nt][0]);
                    rest[i][nt][1] = movmatrix_trans(rest[i][nt][1]);
                }
            }
            await_unit();
            const uint32_t vst = ring + place_out * G::kUnit + v_row;
#pragma unroll
            for (uint32_t i = 0; i < kR; ++i) {
#pragma unroll
                for (uint32_t ks = 0; ks < kSteps; ++ks) {
                    uint32_t a0, a1, a2, a3;
                    ldmatrix_x4_trans(vst + i * kPagedSlice * G::kRow + ks / 4u * 128u + (((ks % 4u * 2u + v_chunk) ^ lm_r) << 4), a0, a1, a2, a3);
#pragma unroll
                    for (uint32_t nt = 0; nt < kTiles; ++nt) {
                        Half<T>::mma(o[nt][ks], a0, a1, a2, a3, rest[i][nt][0], rest[i][nt][1]);
                        Half<T>::mma(o[nt][ks], a0, a1, a2, a3, pb[i][nt][0], pb[i][nt][1]);
                    }
                }
            }
            release_unit();
        }

        // the next item's query is on its way while this item's warps are joined
        const uint4 done = ci;
        ++done_items;
        if (done_items < count) {
            ci = items[done_items % kPdItems];
            load_query(ci);
        }
        // ---- the four warps' parts of the item, joined eight heads at a time.  Each warp lays its rows over the unit of its ring
        // that it read last: the others are in flight or waiting, that one is free until the next issue().  Dims are
        // XORed with a multiple of 8 by head so that the four heads that a warp stores at once fall into different banks.
        const uint32_t free_place = place_out == 0u ? p.units - 1u : place_out - 1u;
        float* merge_mine = reinterpret_cast<float*>(smem + (warp * p.units + free_place) * G::kUnit);
        if (lane == 0) warp_word[warp] = free_place;
#pragma unroll
        for (uint32_t nt = 0; nt < kTiles; ++nt) {
#pragma unroll
            for (uint32_t off = 4; off < 32; off <<= 1) {
                l[nt][0] += __shfl_xor_sync(0xffffffffu, l[nt][0], off);
                l[nt][1] += __shfl_xor_sync(0xffffffffu, l[nt][1], off);
            }
            float* mo = merge_mine + 2u * t * D;
            if (nt * 8u + 2u * t < p.group) {
#pragma unroll
                for (uint32_t ks = 0; ks < kSteps; ++ks) {
                    const uint32_t d0 = (ks * 16u + g) ^ (t << 3), d1 = (ks * 16u + 8u + g) ^ (t << 3);
                    mo[d0] = o[nt][ks][0];
                    mo[D + d0] = o[nt][ks][1];
                    mo[d1] = o[nt][ks][2];
                    mo[D + d1] = o[nt][ks][3];
                }
            }
            if (g == 0) {
                merge_ml[warp * 8u + 2u * t] = make_float2(m[nt][0], l[nt][0]);
                merge_ml[warp * 8u + 2u * t + 1u] = make_float2(m[nt][1], l[nt][1]);
            }
            __syncthreads();
            const uint32_t h = threadIdx.x >> 4, head = nt * 8u + h;
            if (head < p.group) {
                float wt[kPdWarps], top = -INFINITY, sum = 0.0f;
#pragma unroll
                for (uint32_t w = 0; w < kPdWarps; ++w) top = fmaxf(top, merge_ml[w * 8u + h].x);
#pragma unroll
                for (uint32_t w = 0; w < kPdWarps; ++w) {
                    const float2 ml = merge_ml[w * 8u + h];
                    wt[w] = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - top);
                    sum = fmaf(wt[w], ml.y, sum);
                }
                const uint64_t record = (uint64_t(done.x & 0xFFFFu) * p.q_heads + (done.x >> 16) * p.group + head) * p.parts + done.y;
                float4* dst = reinterpret_cast<float4*>(p.sums + record * D);
#pragma unroll
                for (uint32_t d4 = threadIdx.x & 15u; d4 < D / 4; d4 += 16u) {
                    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (uint32_t w = 0; w < kPdWarps; ++w) {
                        const float4 v = *reinterpret_cast<const float4*>(smem + (w * p.units + warp_word[w]) * G::kUnit +
                                                                          (h * D + ((d4 * 4u) ^ ((h >> 1) << 3))) * 4u);
                        acc.x = fmaf(wt[w], v.x, acc.x);
                        acc.y = fmaf(wt[w], v.y, acc.y);
                        acc.z = fmaf(wt[w], v.z, acc.z);
                        acc.w = fmaf(wt[w], v.w, acc.w);
                    }
                    dst[d4] = acc;
                }
                if ((threadIdx.x & 15u) == 0u) p.stats[record] = make_float2(top, sum);
            }
            // every warp has read this item's query: the next one's takes its place
            if (nt == 0u) store_query();
            // half of the descriptors lie behind every warp's arithmetic: the half after the other one takes their place
            if (nt + 1u == kTiles && done_items % (kPdItems / 2u) == 0u) {
                if (threadIdx.x < kPdItems / 2u) describe(done_items + kPdItems / 2u + threadIdx.x);
                // A warp without a share in a run of items has not read ahead past them and may stand among the replaced: it goes on from the
                // item under way (left there, it would take descriptors of 128 items on for those it passes).
                if (at < done_items && done_items < count) {
                    at = done_items;
                    turn = 0;
                    pi = items[at % kPdItems];
                    settle(pi, 0u, fetch_pages(pi, 0u));
                    if (at + 1u < count) next_pages = fetch_pages(items[(at + 1u) % kPdItems], 0u);
                }
            }
            __syncthreads();
        }
    }
    cp_async_wait<0>();
}

// ---- the join -----------------------------------------------------------------------------
// With a mass, the first `walkers` CTAs add the weights to it, kMassSpan slots of a kv head at a time; the others finish 64 dims of a
// head each, or a head.
// Bound by latency for a lane alone (3 us behind the first kernel), by L2 in a batch (records, scores and mass of 32 lanes of 4096 to
// 32768 slots: 10 us).
constexpr uint32_t kMassSpan = 1024;

// How a piece is finished: 64 dims by a CTA (few heads: the shortest way), 64 dims by a warp (no lane has more than 16 partitions), or a whole
// head by a CTA (many heads: a quarter of the CTAs, each weighing its partitions once).  The same additions in the same order, so the
// form is free to follow from the call's bounds.
enum JoinForm { kJoinSlice, kJoinWarp, kJoinHead };
template <typename T, int D, JoinForm kForm>
__global__ void __launch_bounds__(kJoinThreads)
paged_join_kernel(const __grid_constant__ PagedDecodeParams p, const uint32_t walkers) {
    __shared__ uint32_t item_start[TATARA_MAX_LANES + 1], lane_keys[TATARA_MAX_LANES], warp_total[kJoinWarps];
    __shared__ float weight[kSmCount * 2];                 // per_wave at most
    __shared__ float red[kJoinWarps], red_sum[kJoinWarps];
    constexpr uint32_t kWidth = kForm == kJoinHead ? D : kJoinDims;             // dims of a piece
    __shared__ __align__(16) float acc_s[kJoinPhases][kWidth];
    __shared__ float2 final_ml[16];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    constexpr uint32_t kSlices = D / kWidth;
    wait_for_predecessor();
    release_dependents();
    if (blockIdx.x >= walkers) {
        const uint32_t piece = kForm == kJoinWarp ? (blockIdx.x - walkers) * kJoinWarps + warp : blockIdx.x - walkers;
        const uint32_t slice = piece % kSlices, rest = piece / kSlices, head = rest % p.q_heads, row = rest / p.q_heads;
        if (row >= p.n_lanes) return;
        const uint32_t n = __ldcg(&p.lanes[row].keys);
        if (n > p.max_keys) return;                        // refused: its row stays as it is
        const uint32_t parts = n == 0u ? 0u : p.cut.parts(n);
        const uint64_t record = (uint64_t(row) * p.q_heads + head) * p.parts;
        // a thread owns two dims and kOwn of the phases
        constexpr uint32_t kColumns = kWidth / 2u, kOwn = kJoinPhases * kColumns / kJoinThreads;
        const uint32_t pair = threadIdx.x % kColumns, phase = threadIdx.x / kColumns * kOwn;
        const float* base = p.sums + record * D + slice * kWidth + pair * 2u;
        const uint64_t out_row = row * p.query_stride + uint64_t(head) * D + slice * kWidth;
        if constexpr (kForm == kJoinWarp) {
            const uint64_t at = (out_row + pair * 2u) * 2u;
            float gate0 = 0.0f, gate1 = 0.0f;
            if (p.gate != nullptr) {
                gate0 = Half<T>::load(p.gate + at);
                gate1 = Half<T>::load(p.gate + at + 2u);
            }
            const float2 ml = lane < parts ? __ldcg(&p.stats[record + lane]) : make_float2(-INFINITY, 0.0f);
            float a[kJoinPhases][2];
#pragma unroll
            for (uint32_t f = 0; f < kJoinPhases; ++f) a[f][0] = a[f][1] = 0.0f;
            float top = ml.x, mine = 0.0f, sum = 0.0f;
#pragma unroll
            for (uint32_t off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            mine = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - top);
            sum = fmaf(mine, ml.y, 0.0f);
#pragma unroll
            for (uint32_t off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            for (uint32_t part0 = 0; part0 < parts; part0 += kJoinPhases) {
                float2 x[kJoinPhases];
#pragma unroll
                for (uint32_t f = 0; f < kJoinPhases; ++f)
                    if (part0 + f < parts) x[f] = __ldcg(reinterpret_cast<const float2*>(base + uint64_t(part0 + f) * D));
#pragma unroll
                for (uint32_t f = 0; f < kJoinPhases; ++f) {
                    const float w = __shfl_sync(0xffffffffu, mine, (part0 + f) & 31u);
                    if (part0 + f < parts) {
                        a[f][0] = fmaf(w, x[f].x, a[f][0]);
                        a[f][1] = fmaf(w, x[f].y, a[f][1]);
                    }
                }
            }
            float n0 = 0.0f, n1 = 0.0f;
#pragma unroll
            for (uint32_t f = 0; f < kJoinPhases; ++f) {
                n0 += a[f][0];
                n1 += a[f][1];
            }
            float r0 = sum == 0.0f ? 0.0f : n0 / sum, r1 = sum == 0.0f ? 0.0f : n1 / sum;   // no slot at all: zero
            if (p.gate != nullptr) {
                r0 *= 1.0f / (1.0f + expf(-gate0));
                r1 *= 1.0f / (1.0f + expf(-gate1));
            }
            Half<T>::store(p.out + at, r0);
            Half<T>::store(p.out + at + 2u, r1);
            return;
        }
        const uint64_t at = (out_row + threadIdx.x) * 2u;
        float gate = 0.0f;
        if (threadIdx.x < kWidth && p.gate != nullptr) gate = Half<T>::load(p.gate + at);
        // the first partitions' sums are asked for before their weights are known
        constexpr uint32_t kAhead = kOwn == 1u ? 10u : 3u;
        float2 v[kAhead][kOwn];
        auto ask = [&](uint32_t round0) {
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i)
#pragma unroll
                for (uint32_t f = 0; f < kOwn; ++f) {
                    const uint32_t part = (round0 + i) * kJoinPhases + phase + f;
                    if (part < parts) v[i][f] = __ldcg(reinterpret_cast<const float2*>(base + uint64_t(part) * D));
                }
        };
        ask(0u);
        static_assert(kSmCount * 2u <= 2u * kJoinThreads, "two partitions a thread");
        float2 ml[2];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            const uint32_t part = threadIdx.x + i * kJoinThreads;
            ml[i] = part < parts ? __ldcg(&p.stats[record + part]) : make_float2(-INFINITY, 0.0f);
        }
        float top = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
        for (uint32_t off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        if (lane == 0) red[warp] = top;
        __syncthreads();
        top = red[0];
#pragma unroll
        for (uint32_t w = 1; w < kJoinWarps; ++w) top = fmaxf(top, red[w]);
        float sum = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            const uint32_t part = threadIdx.x + i * kJoinThreads;
            const float w = ml[i].x == -INFINITY ? 0.0f : exp2f(ml[i].x - top);
            if (part < parts) weight[part] = w;
            sum = fmaf(w, ml[i].y, sum);
        }
#pragma unroll
        for (uint32_t off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (lane == 0) red_sum[warp] = sum;
        __syncthreads();
        float2 a[kOwn];
#pragma unroll
        for (uint32_t f = 0; f < kOwn; ++f) a[f] = make_float2(0.0f, 0.0f);
        for (uint32_t round0 = 0; round0 * kJoinPhases < parts; round0 += kAhead) {
            if (round0 != 0u) ask(round0);
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i)
#pragma unroll
                for (uint32_t f = 0; f < kOwn; ++f) {
                    const uint32_t part = (round0 + i) * kJoinPhases + phase + f;
                    if (part < parts) {
                        a[f].x = fmaf(weight[part], v[i][f].x, a[f].x);
                        a[f].y = fmaf(weight[part], v[i][f].y, a[f].y);
                    }
                }
        }
#pragma unroll
        for (uint32_t f = 0; f < kOwn; ++f) *reinterpret_cast<float2*>(&acc_s[phase + f][pair * 2u]) = a[f];
        __syncthreads();
        if (threadIdx.x < kWidth) {
            float num = 0.0f, den = 0.0f;
#pragma unroll
            for (uint32_t ph = 0; ph < kJoinPhases; ++ph) num += acc_s[ph][threadIdx.x];
#pragma unroll
            for (uint32_t w = 0; w < kJoinWarps; ++w) den += red_sum[w];
            float r = den == 0.0f ? 0.0f : num / den;      // no slot at all: zero
            if (p.gate != nullptr) r *= 1.0f / (1.0f + expf(-gate));
            Half<T>::store(p.out + at, r);
        }
        return;
    }
    scan_items<kJoinThreads>(p, item_start, lane_keys, warp_total, false, [](uint32_t n) { return (n + kMassSpan - 1u) / kMassSpan; });
    const uint32_t total = item_start[p.n_lanes], row_floats = (p.group + 7u) / 8u * 8u;
    for (uint32_t item = blockIdx.x; item < total; item += walkers) {
        const PagedItem it = item_at(p, item_start, lane_keys, item, [](uint32_t) { return kMassSpan; });
        const uint32_t parts = p.cut.parts(lane_keys[it.lane]);
        const uint64_t head_row = uint64_t(it.lane) * p.cache.kv_heads + it.kv;
        const float* scores = p.scores + (head_row * p.score_slots + it.begin) * row_floats;
        float* mass = p.cache.mass + head_row * p.cache.capacity + it.begin;
        // the heads' maximum and the reciprocal of their sum
        for (uint32_t h = warp; h < p.group; h += kJoinWarps) {
            const float2* st = p.stats + (uint64_t(it.lane) * p.q_heads + it.kv * p.group + h) * p.parts;
            float top = -INFINITY, sum = 0.0f;
            for (uint32_t part0 = 0; part0 < parts; part0 += 160u) {
                float2 ml[5];
                float big = top;
#pragma unroll
                for (uint32_t i = 0; i < 5; ++i) {
                    const uint32_t part = part0 + i * 32u + lane;
                    ml[i] = part < parts ? __ldcg(&st[part]) : make_float2(-INFINITY, 0.0f);
                    big = fmaxf(big, ml[i].x);
                }
#pragma unroll
                for (uint32_t off = 16; off; off >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
                sum *= top == -INFINITY ? 0.0f : exp2f(top - big);
#pragma unroll
                for (uint32_t i = 0; i < 5; ++i) sum = fmaf(ml[i].x == -INFINITY ? 0.0f : exp2f(ml[i].x - big), ml[i].y, sum);
                top = big;
            }
#pragma unroll
            for (uint32_t off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            if (lane == 0) final_ml[h] = make_float2(top == -INFINITY ? 0.0f : top, sum == 0.0f ? 0.0f : exp2f(Half<T>::kTopLog2) / sum);
        }
        __syncthreads();
        constexpr uint32_t kOwn = kMassSpan / kJoinThreads;
        float w[kOwn], before[kOwn];
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) {
            const uint32_t slot = i * kJoinThreads + threadIdx.x;
            before[i] = slot < it.slots ? __ldcg(mass + slot) : 0.0f;
            w[i] = 0.0f;
        }
        for (uint32_t h0 = 0; h0 < p.group; h0 += 4u) {
            float4 v[kOwn];
#pragma unroll
            for (uint32_t i = 0; i < kOwn; ++i) {
                const uint32_t slot = i * kJoinThreads + threadIdx.x;
                v[i] = __ldcg(reinterpret_cast<const float4*>(scores + uint64_t(slot < it.slots ? slot : 0u) * row_floats + h0));
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                if (h0 + j >= p.group) break;
                const float2 ml = final_ml[h0 + j];
#pragma unroll
                for (uint32_t i = 0; i < kOwn; ++i)
                    w[i] = fmaf(exp2f((j == 0 ? v[i].x : j == 1 ? v[i].y : j == 2 ? v[i].z : v[i].w) - ml.x), ml.y, w[i]);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) {
            const uint32_t slot = i * kJoinThreads + threadIdx.x;
            if (slot < it.slots) mass[slot] = before[i] + w[i];
        }
        __syncthreads();
    }
}

// ---- host side -------------------------------------------------------------------------
struct PagedDecodeLayout {
    PagedCut cut;
    uint32_t parts, score_slots, row_floats;
    uint64_t stats_at, scores_at, bytes;
};
static PagedDecodeLayout pd_layout(const tatara_paged_cache& c, uint32_t n_lanes, uint32_t max_keys, uint32_t q_heads) {
    PagedDecodeLayout l{};
    l.cut = PagedCut{pd_per_wave(c.kv_heads, c.head_dim), pd_min_part(q_heads / c.kv_heads)};
    const uint32_t shortest = (max_keys + l.cut.least - 1u) / l.cut.least;   // cut.parts(n) <= both for every n <= max_keys
    l.parts = shortest < l.cut.per_wave ? shortest : l.cut.per_wave;
    l.score_slots = (max_keys + kPagedSlice - 1u) / kPagedSlice * kPagedSlice;
    l.row_floats = (q_heads / c.kv_heads + 7u) / 8u * 8u;
    const uint64_t records = uint64_t(n_lanes) * q_heads * l.parts;
    l.stats_at = records * c.head_dim * 4u;
    l.scores_at = (l.stats_at + records * 8u + 255u) / 256u * 256u;
    l.bytes = l.scores_at + (c.mass == nullptr ? 0u : uint64_t(n_lanes) * c.kv_heads * l.score_slots * l.row_floats * 4u);
    return l;
}

template <typename T, int D, int kTiles>
static tatara_status launch_paged_decode(tatara_ctx* ctx, cudaStream_t stream, PagedDecodeParams p) {
    using G = PdGeometry<D>;
    constexpr uint32_t kCtas = pd_ctas(D);
    static bool configured[64] = {false};
    if (!configured[ctx->device & 63]) {
        if (cudaFuncSetAttribute(paged_decode_kernel<T, D, kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::smem(G::units(1u), kTiles == 2)) != cudaSuccess)
            return check_launch(ctx, "attn_decode_paged: shared memory attribute");
        configured[ctx->device & 63] = true;
    }
    const uint64_t items = uint64_t(p.n_lanes) * p.parts * p.cache.kv_heads, sms = ctx->sm_count;
    const uint32_t ctas = items >= kCtas * sms ? kCtas : uint32_t((items + sms - 1u) / sms);   // on an SM
    p.units = G::units(ctas);
    // Asking ahead pays for long partitions (one lane of 262144 slots 86.7 -> 84.2 us, of 131072 with head_dim 128 48 -> 45), costs 0.2 us
    // where they are the shortest, and slows the arithmetic-bound wide groups (28 -> 32 us).
    p.ahead_slots = items <= kCtas * sms && kTiles == 1 && p.cut.part_slots(p.max_keys) > p.cut.least ? ctx->decode_l2_prefetch_keys : 0u;
    // Shared memory for just the CTAs that are to share an SM, the rest stays L1 -- and one CTA an SM stays one (one lane of 131072 slots 46.8 ->
    // 45.4 us against the driver's choice, of 32768 18.8 -> 18.2).
    constexpr uint32_t kSmMemory = 228u * 1024u, kReserved = 1024u;   // of a CTA
    const uint32_t smem = G::smem(p.units, kTiles == 2), share = (ctas * (smem + kReserved) * 100u + kSmMemory - 1u) / kSmMemory;
    const dim3 grid(uint32_t(items < kCtas * sms ? items : kCtas * sms));
    (void)launch_staged_carved(int(share < 100u ? share : 100u), paged_decode_kernel<T, D, kTiles>, grid, kPdThreads, smem, stream, p);
    const tatara_status st = check_launch(ctx, "attn_decode_paged");
    if (st != TATARA_OK) return st;
    const uint32_t pieces = p.n_lanes * p.q_heads * (D / kJoinDims);
    const uint64_t spans = uint64_t(p.n_lanes) * p.cache.kv_heads * ((p.max_keys + kMassSpan - 1u) / kMassSpan);
    const uint32_t walkers = p.cache.mass == nullptr ? 0u : uint32_t(spans < 4u * ctx->sm_count ? spans : 4u * ctx->sm_count);
    auto join = p.parts <= 16u ? paged_join_kernel<T, D, kJoinWarp> : paged_join_kernel<T, D, kJoinSlice>;
    uint32_t join_ctas = p.parts <= 16u ? (pieces + kJoinWarps - 1u) / kJoinWarps : pieces;
    if constexpr (D != kJoinDims) {   // (a slice is a head there)
        if (p.parts > 16u && pieces > 4u * sms) {
            join = paged_join_kernel<T, D, kJoinHead>;
            join_ctas = p.n_lanes * p.q_heads;
        }
    }
    (void)launch_staged(join, dim3(join_ctas + walkers), kJoinThreads, 0u, stream, p, walkers);
    return check_launch(ctx, "attn_decode_paged: join");
}

template <typename T>
static tatara_status pick_paged_decode(tatara_ctx* ctx, cudaStream_t stream, const PagedDecodeParams& p, uint32_t head_dim) {
    const bool wide = p.group > 8u;
    switch (head_dim) {
    case 64: return wide ? launch_paged_decode<T, 64, 2>(ctx, stream, p) : launch_paged_decode<T, 64, 1>(ctx, stream, p);
    case 128: return wide ? launch_paged_decode<T, 128, 2>(ctx, stream, p) : launch_paged_decode<T, 128, 1>(ctx, stream, p);
    default: return wide ? launch_paged_decode<T, 256, 2>(ctx, stream, p) : launch_paged_decode<T, 256, 1>(ctx, stream, p);
    }
}

} // namespace tb

using namespace tb;

extern "C" uint64_t tatara_attn_decode_paged_scratch_bytes(const tatara_paged_cache* cache, uint32_t n_lanes, uint32_t max_keys,
                                                           uint32_t q_heads) {
    if (cache == nullptr || cache->kv_heads == 0 || cache->head_dim == 0 || cache->head_dim > 256u || max_keys > TATARA_MAX_CONTEXT) return 0;
    return pd_layout(*cache, n_lanes, max_keys, q_heads).bytes;
}

extern "C" tatara_status tatara_attn_decode_paged(tatara_ctx* ctx, void* stream, const tatara_paged_cache* cache,
                                                  const tatara_paged_lane* lanes_device, uint32_t n_lanes, uint32_t max_keys,
                                                  const void* q, const void* gate, uint32_t q_heads, uint64_t query_stride,
                                                  float scale, void* out, void* scratch, uint64_t scratch_bytes) {
    if (ctx == nullptr) return TATARA_INVALID_BUFFER;
    const tatara_status st = check_paged(ctx, cache, lanes_device, n_lanes);
    if (st != TATARA_OK) return st;
    if (!q || !out || !scratch) return fail(ctx, TATARA_INVALID_BUFFER, "attn_decode_paged: null buffer");
    if (!aligned(q, 4) || !aligned(gate, 2) || !aligned(out, 2) || !aligned(scratch, 16))
        return fail(ctx, TATARA_INVALID_BUFFER, "attn_decode_paged: misaligned buffer");
    if (q_heads == 0 || q_heads % cache->kv_heads != 0 || q_heads / cache->kv_heads > TATARA_MAX_GROUP)
        return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "attn_decode_paged: query heads per kv head");
    if (query_stride < uint64_t(q_heads) * cache->head_dim || query_stride % 2u)
        return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "attn_decode_paged: query stride");
    if (!std::isfinite(scale)) return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "attn_decode_paged: scale");
    if (max_keys == 0 || max_keys > cache->table_pages * cache->page_slots || max_keys > TATARA_MAX_CONTEXT)
        return fail(ctx, TATARA_CONTEXT_OUT_OF_RANGE, "attn_decode_paged: max_keys beyond the page table or the longest context");
    const PagedDecodeLayout l = pd_layout(*cache, n_lanes, max_keys, q_heads);
    if (scratch_bytes < l.bytes) return fail(ctx, TATARA_SCRATCH_TOO_SMALL, "attn_decode_paged: scratch");
    PagedDecodeParams p{};
    p.cache = paged_view(ctx, *cache);
    p.lanes = lanes_device;
    p.q = static_cast<const uint8_t*>(q);
    p.gate = static_cast<const uint8_t*>(gate);
    p.out = static_cast<uint8_t*>(out);
    p.sums = static_cast<float*>(scratch);
    p.stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(scratch) + l.stats_at);
    p.scores = cache->mass == nullptr ? nullptr : reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + l.scores_at);
    p.query_stride = query_stride;
    p.n_lanes = n_lanes;
    p.max_keys = max_keys;
    p.q_heads = q_heads;
    p.group = q_heads / cache->kv_heads;
    p.cut = l.cut;
    p.parts = l.parts;
    p.score_slots = l.score_slots;
    p.page_slices = cache->page_slots / kPagedSlice;
    p.page_magic = uint32_t((1ull << 32) / p.page_slices) + 1u;   // (a single slice to a page is taken apart: 2^32 does not fit)
    p.scale_log2e = scale * kPdLog2e;
    const DeviceGuard guard(ctx);
    return cache->dtype == TATARA_BF16 ? pick_paged_decode<__nv_bfloat16>(ctx, static_cast<cudaStream_t>(stream), p, cache->head_dim)
                                       : pick_paged_decode<__half>(ctx, static_cast<cudaStream_t>(stream), p, cache->head_dim);
}
