// Rows into a paged KV cache: the append of K and V rows, the model's q/k norm + rope + append, and the lane table's step.
// All three move bytes: each row is read once and written once.
#include "paged.cuh"

#include <cmath>

namespace tb {

// ---- append ------------------------------------------------------------------------------
// A thread copies 16-byte chunks; a tile of rows, all their heads, makes a CTA's work, so the search for a row's lane and the
// page-table entry are shared by the tile's heads.
constexpr uint32_t kAppendThreads = 256;

struct PagedAppendParams {
    PagedView cache;
    const tatara_paged_lane* lanes;
    const uint8_t* keys;
    const uint8_t* values;
    uint64_t row_bytes, source_head_bytes;
    const uint32_t* row_starts;
    uint32_t n_lanes, n_rows, tile_rows;
};

// Where row `row` goes: its lane and slot; false for padding rows and rows without a slot.
__device__ __forceinline__ bool append_target(const PagedAppendParams& p, uint32_t row, uint32_t& lane, uint32_t& slot, uint32_t& position) {
    uint32_t back = 1u;   // 1 for a lane's newest row
    if (p.row_starts == nullptr) {
        lane = row;
    } else {
        if (row < __ldcg(p.row_starts) || row >= __ldcg(p.row_starts + p.n_lanes)) return false;
        uint32_t lo = 0, hi = p.n_lanes;   // last lane with row_starts <= row
        while (hi - lo > 1u) {
            const uint32_t mid = (lo + hi) >> 1;
            if (__ldcg(p.row_starts + mid) <= row) lo = mid; else hi = mid;
        }
        lane = lo;
        back = __ldcg(p.row_starts + lo + 1u) - row;
    }
    const uint2 l = __ldcg(reinterpret_cast<const uint2*>(p.lanes + lane));   // keys, position
    if (l.x == 0u) return false;                                              // idle
    if (l.x > p.cache.capacity || back == 0u || back > l.x) {
        latch_out_of_range(p.cache, lane);
        return false;
    }
    slot = l.x - back;
    position = l.y + 1u - back;
    return true;
}

template <uint32_t kChunks>   // 16-byte chunks of a row
__global__ void __launch_bounds__(kAppendThreads)
paged_append_kernel(const __grid_constant__ PagedAppendParams p) {
    extern __shared__ __align__(16) uint8_t append_smem[];
    uint64_t* dst = reinterpret_cast<uint64_t*>(append_smem);   // [tile_rows]: byte offset of head 0's row, ~0 = none
    wait_for_predecessor();
    if (blockIdx.x == 0u && threadIdx.x == 0u && p.row_starts != nullptr && __ldcg(p.row_starts + p.n_lanes) > p.n_rows)
        latch_out_of_range(p.cache, p.n_lanes);   // rows that were promised and are not there
    const uint32_t first = blockIdx.x * p.tile_rows, rows = min(p.tile_rows, p.n_rows - first), heads = p.cache.kv_heads;
    for (uint32_t r = threadIdx.x; r < rows; r += kAppendThreads) {
        uint32_t lane, slot, position;
        uint64_t offset = 0;
        const bool ok = append_target(p, first + r, lane, slot, position) && slot_offset(p.cache, lane, 0u, slot, offset);
        dst[r] = ok ? offset : ~0ull;
        if (ok) {
            for (uint32_t h = 0; h < heads; ++h) {
                const uint64_t at = plane_row(p.cache, lane, h) + slot;
                if (p.cache.mass != nullptr) p.cache.mass[at] = 0.0f;
                if (p.cache.positions != nullptr) p.cache.positions[at] = position;
            }
        }
    }
    __syncthreads();
    // Four loads of K and of V are on their way before the first store; stores that stream past L2's working set: 74k rows of 2 kv
    // heads of 256 take 51 us (6.0 TB/s read and written) against 57 one after another, 52 with plain stores.
    const uint32_t chunk = threadIdx.x % kChunks;
    constexpr uint32_t kStep = kAppendThreads / kChunks, kBatch = 4;
    for (uint32_t i0 = threadIdx.x / kChunks; i0 < rows * heads; i0 += kStep * kBatch) {
        uint4 k[kBatch], v[kBatch];
        uint64_t to[kBatch];
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) {
            const uint32_t i = i0 + j * kStep, h = i / rows, r = i - h * rows;   // rows of one head run together in a contiguous cache
            to[j] = i < rows * heads ? dst[r] : ~0ull;
            if (to[j] == ~0ull) continue;
            const uint64_t src = (first + r) * p.row_bytes + h * p.source_head_bytes + chunk * 16u;
            to[j] += h * p.cache.head_bytes + chunk * 16u;
            k[j] = __ldcs(reinterpret_cast<const uint4*>(p.keys + src));
            v[j] = __ldcs(reinterpret_cast<const uint4*>(p.values + src));
        }
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) {
            if (to[j] == ~0ull) continue;
            __stcs(reinterpret_cast<uint4*>(p.cache.keys + to[j]), k[j]);
            __stcs(reinterpret_cast<uint4*>(p.cache.values + to[j]), v[j]);
        }
    }
}

// ---- q/k norm + rope + append --------------------------------------------------------------
// A warp owns one (head, row): lane l holds dims 8l .. 8l+7 (16-byte accesses), dims d and d + 32 of a rotated pair are
// four lanes apart.  Lane l evaluates the angle of pair l, in turns: the product and the fraction in double, since a far position
// loses its angle in f32 (2^18 / 1.6 has a last place of 1/64), then one sincospif; lanes 0 .. 7 take theirs by shuffles.  Latency
// bound: 2.4 us for 8 lanes, 4.4 for 256 (9.4 MB).
constexpr uint32_t kRopeWarps = 4;

// Turns of each pair from one position to the next; the model's divisors are base^(pair / 32) rounded to f32.
struct RopeTurns {
    double of[kRopePairs];
    RopeTurns() {
        for (uint32_t i = 0; i < kRopePairs; ++i)
            of[i] = 1.0 / (6.283185307179586476925286766559 * double(static_cast<float>(std::pow(1.0e7, double(i) / 32.0))));
    }
};

struct PagedRopeParams {
    PagedView cache;
    const tatara_paged_lane* lanes;
    const __nv_bfloat16* projection;
    const __nv_bfloat16* q_weight;
    const __nv_bfloat16* k_weight;
    __nv_bfloat16* q_out;
    __nv_bfloat16* gate_out;
    uint64_t projection_stride, query_stride;
    uint32_t n_lanes;
    RopeTurns turns;
};

__device__ __forceinline__ void unpack8(const uint4 raw, float (&out)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        out[2 * i] = __uint_as_float(w[i] << 16);
        out[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}

__global__ void __launch_bounds__(kRopeWarps * 32)
paged_rope_kernel(const __grid_constant__ PagedRopeParams p) {
    const uint32_t lane = threadIdx.x & 31u, unit = blockIdx.x * kRopeWarps + (threadIdx.x >> 5);
    const uint32_t row = unit / (kQHeads + kKvHeads), head = unit - row * (kQHeads + kKvHeads);
    if (row >= p.n_lanes) return;
    wait_for_predecessor();
    release_dependents();   // (a decode kernel that follows asks rows into L2 and then waits)
    const bool is_q = head < kQHeads;
    const uint32_t local = is_q ? head : head - kQHeads;
    const __nv_bfloat16* proj = p.projection + row * p.projection_stride;
    // (every load is on its way before the lane's state decides; an idle lane has a projection row too)
    const uint2 l = __ldcg(reinterpret_cast<const uint2*>(p.lanes + row));   // keys, position
    const uint4 raw = __ldcg(reinterpret_cast<const uint4*>(proj + (is_q ? head * 2u * kHeadDim : kAttnKOff + local * kHeadDim) + lane * 8u));
    // what is copied through: the gate of a query head, the values of a key head
    const uint4 through = __ldcg(reinterpret_cast<const uint4*>(proj + (is_q ? head * 2u * kHeadDim + kHeadDim : kAttnVOff + local * kHeadDim) + lane * 8u));
    const uint4 wraw = __ldcg(reinterpret_cast<const uint4*>((is_q ? p.q_weight : p.k_weight) + lane * 8u));
    if (l.x == 0u) return;                                                   // idle
    if (l.x > p.cache.capacity) {
        if (lane == 0) latch_out_of_range(p.cache, row);
        return;
    }
    float x[8], w[8];
    unpack8(raw, x);
    unpack8(wraw, w);
    float acc = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) acc = fmaf(x[i], x[i], acc);
    acc = warp_sum(acc);
    const float inverse = 1.0f / sqrtf(acc / float(kHeadDim) + kRmsEps);
    const double turns = double(l.y) * p.turns.of[lane];
    float sine, cosine;
    sincospif(2.0f * float(turns - rint(turns)), &sine, &cosine);
    __nv_bfloat16 res[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        x[i] = w[i] * (x[i] * inverse);
        const uint32_t pair = (lane & 3u) * 8u + i;
        const float partner = __shfl_xor_sync(0xffffffffu, x[i], 4);   // dim +- 32 (used by lanes 0..7)
        const float s = __shfl_sync(0xffffffffu, sine, pair), c = __shfl_sync(0xffffffffu, cosine, pair);
        if (lane < 8u) x[i] = lane < 4u ? fmaf(-partner, s, x[i] * c) : fmaf(partner, s, x[i] * c);
        res[i] = f2bf(x[i]);
    }
    if (is_q) {
        const uint64_t at = row * p.query_stride + head * kHeadDim + lane * 8u;
        *reinterpret_cast<uint4*>(p.q_out + at) = *reinterpret_cast<const uint4*>(res);
        *reinterpret_cast<uint4*>(p.gate_out + at) = through;
        return;
    }
    uint64_t offset;
    if (!slot_offset(p.cache, row, local, l.x - 1u, offset)) return;
    *reinterpret_cast<uint4*>(p.cache.keys + offset + lane * 16u) = *reinterpret_cast<const uint4*>(res);
    *reinterpret_cast<uint4*>(p.cache.values + offset + lane * 16u) = through;
    if (lane == 0) {
        const uint64_t at = plane_row(p.cache, row, local) + l.x - 1u;
        if (p.cache.mass != nullptr) p.cache.mass[at] = 0.0f;
        if (p.cache.positions != nullptr) p.cache.positions[at] = l.y;
    }
}

// ---- the lane table between tokens ---------------------------------------------------------
__global__ void paged_lanes_step_kernel(tatara_paged_lane* lanes, uint32_t n_lanes, uint32_t keep, uint32_t advance) {
    const uint32_t i = threadIdx.x;
    wait_for_predecessor();
    if (i >= n_lanes) return;
    const uint2 l = __ldcg(reinterpret_cast<const uint2*>(lanes + i));   // keys, position
    if (l.x != 0u) lanes[i] = tatara_paged_lane{min(l.x, keep) + advance, l.y + advance};
}

} // namespace tb

using namespace tb;

extern "C" tatara_status tatara_paged_append(tatara_ctx* ctx, void* stream, const tatara_paged_cache* cache,
                                             const tatara_paged_lane* lanes_device, uint32_t n_lanes, const void* keys,
                                             const void* values, uint64_t row_stride, uint64_t source_head_stride,
                                             const uint32_t* row_starts, uint32_t n_rows) {
    if (ctx == nullptr) return TATARA_INVALID_BUFFER;
    const tatara_status st = check_paged(ctx, cache, lanes_device, n_lanes);
    if (st != TATARA_OK) return st;
    if (!keys || !values) return fail(ctx, TATARA_INVALID_BUFFER, "paged_append: null buffer");
    if (!aligned(keys, 16) || !aligned(values, 16) || !aligned(row_starts, 4))
        return fail(ctx, TATARA_INVALID_BUFFER, "paged_append: misaligned buffer");
    if (row_stride % 8u || source_head_stride % 8u || row_stride < cache->head_dim || source_head_stride < cache->head_dim)
        return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged_append: strides are multiples of 8 elements, at least head_dim");
    if (n_rows == 0 || n_rows > (1u << 28) || (row_starts == nullptr && n_rows != n_lanes))
        return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged_append: rows");
    PagedAppendParams p{};
    p.cache = paged_view(ctx, *cache);
    p.lanes = lanes_device;
    p.keys = static_cast<const uint8_t*>(keys);
    p.values = static_cast<const uint8_t*>(values);
    p.row_bytes = row_stride * 2u;
    p.source_head_bytes = source_head_stride * 2u;
    p.row_starts = row_starts;
    p.n_lanes = n_lanes;
    p.n_rows = n_rows;
    // rows of a CTA: one while there are SMs to spare, up to 16 to share the look-ups
    const uint32_t spread = n_rows / (2u * uint32_t(ctx->sm_count));
    p.tile_rows = spread < 1u ? 1u : spread > 16u ? 16u : spread;
    const uint32_t tiles = (n_rows + p.tile_rows - 1u) / p.tile_rows;
    const DeviceGuard guard(ctx);
    auto kernel = cache->head_dim == 64u ? paged_append_kernel<8> : cache->head_dim == 128u ? paged_append_kernel<16> : paged_append_kernel<32>;
    (void)launch_staged(kernel, dim3(tiles), kAppendThreads, p.tile_rows * 8u, static_cast<cudaStream_t>(stream), p);
    return check_launch(ctx, "paged_append");
}

extern "C" tatara_status tatara_attn_qk_rope_paged(tatara_ctx* ctx, void* stream, const tatara_paged_cache* cache,
                                                   const tatara_paged_lane* lanes_device, uint32_t n_lanes,
                                                   const void* projection, const void* q_weight, const void* k_weight,
                                                   void* q_out, void* gate_out, uint64_t projection_stride,
                                                   uint64_t query_stride) {
    if (ctx == nullptr) return TATARA_INVALID_BUFFER;
    const tatara_status st = check_paged(ctx, cache, lanes_device, n_lanes);
    if (st != TATARA_OK) return st;
    if (!projection || !q_weight || !k_weight || !q_out || !gate_out)
        return fail(ctx, TATARA_INVALID_BUFFER, "attn_qk_rope_paged: null buffer");
    if (!aligned(projection, 16) || !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(q_out, 16) || !aligned(gate_out, 16))
        return fail(ctx, TATARA_INVALID_BUFFER, "attn_qk_rope_paged: misaligned buffer");
    if (cache->dtype != TATARA_BF16 || cache->kv_heads != kKvHeads || cache->head_dim != kHeadDim)
        return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "attn_qk_rope_paged: the model's cache is bf16, 2 kv heads of 256");
    if (projection_stride < kAttnProj || query_stride < kQHeads * kHeadDim || projection_stride % 8u || query_stride % 8u)
        return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "attn_qk_rope_paged: stride");
    PagedRopeParams p{};
    p.cache = paged_view(ctx, *cache);
    p.lanes = lanes_device;
    p.projection = static_cast<const __nv_bfloat16*>(projection);
    p.q_weight = static_cast<const __nv_bfloat16*>(q_weight);
    p.k_weight = static_cast<const __nv_bfloat16*>(k_weight);
    p.q_out = static_cast<__nv_bfloat16*>(q_out);
    p.gate_out = static_cast<__nv_bfloat16*>(gate_out);
    p.projection_stride = projection_stride;
    p.query_stride = query_stride;
    p.n_lanes = n_lanes;
    static const RopeTurns turns;
    p.turns = turns;
    const DeviceGuard guard(ctx);
    const uint32_t units = n_lanes * (kQHeads + kKvHeads);
    (void)launch_staged(paged_rope_kernel, dim3((units + kRopeWarps - 1u) / kRopeWarps), kRopeWarps * 32u, 0u,
                        static_cast<cudaStream_t>(stream), p);
    return check_launch(ctx, "attn_qk_rope_paged");
}

extern "C" tatara_status tatara_paged_lanes_step(tatara_ctx* ctx, void* stream, tatara_paged_lane* lanes_device,
                                                 uint32_t n_lanes, uint32_t keep, uint32_t advance) {
    if (ctx == nullptr) return TATARA_INVALID_BUFFER;
    if (lanes_device == nullptr || !aligned(lanes_device, 8)) return fail(ctx, TATARA_INVALID_BUFFER, "paged_lanes_step: lane table");
    if (n_lanes == 0 || n_lanes > TATARA_MAX_LANES) return fail(ctx, TATARA_INVALID_STREAM_GROUP, "paged_lanes_step: lane count");
    if (keep == 0 || advance > TATARA_MAX_CONTEXT) return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged_lanes_step: keep, advance");
    const DeviceGuard guard(ctx);
    (void)launch_staged(paged_lanes_step_kernel, dim3(1), TATARA_MAX_LANES, 0u, static_cast<cudaStream_t>(stream), lanes_device, n_lanes, keep, advance);
    return check_launch(ctx, "paged_lanes_step");
}
