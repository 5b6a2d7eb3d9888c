// Shared pieces of the paged KV cache operators: the device view of a cache, the checks that stand
// before every access, the host-side validation of a cache description, the current-device guard.
#pragma once

#include "warp_tiles.cuh"

#include <cuda_fp16.h>

namespace tb {

constexpr uint32_t kPagedSlice = 16;        // slots of one slice: a page holds a whole number of them
constexpr uint32_t kPagedMaxPageSlots = 1024;

// What the kernels need of a tatara_paged_cache, by value.
struct PagedView {
    uint8_t* keys;
    uint8_t* values;
    uint64_t page_bytes, head_bytes, slot_bytes;
    const uint32_t* page_table;
    float* mass;
    uint32_t* positions;
    uint32_t table_pages, n_pages, page_slots, kv_heads;
    uint32_t capacity;      // slots a lane's row of the page table can address
    uint32_t* status;       // the context's device status words
};

__device__ __forceinline__ void latch_out_of_range(const PagedView& c, uint32_t detail) {
    if (atomicCAS(c.status + kStatusCode, 0u, uint32_t(TATARA_CONTEXT_OUT_OF_RANGE)) == 0u) c.status[kStatusDetail] = detail;
}
__device__ __forceinline__ uint64_t plane_row(const PagedView& c, uint32_t lane, uint32_t head) {
    return (uint64_t(lane) * c.kv_heads + head) * c.capacity;
}
// Byte offset of a slot's row in either pool; false (and the status latched) where the page does not exist.
// The caller has checked slot < capacity.
__device__ __forceinline__ bool slot_offset(const PagedView& c, uint32_t lane, uint32_t head, uint32_t slot, uint64_t& offset) {
    const uint32_t column = slot / c.page_slots;
    const uint32_t page = __ldcg(c.page_table + uint64_t(lane) * c.table_pages + column);
    if (page >= c.n_pages) {
        latch_out_of_range(c, lane);
        return false;
    }
    offset = page * c.page_bytes + head * c.head_bytes + (slot - column * c.page_slots) * c.slot_bytes;
    return true;
}

inline PagedView paged_view(const tatara_ctx* ctx, const tatara_paged_cache& c) {
    PagedView v{};
    v.keys = static_cast<uint8_t*>(c.keys);
    v.values = static_cast<uint8_t*>(c.values);
    v.page_bytes = c.page_stride * 2u;
    v.head_bytes = c.head_stride * 2u;
    v.slot_bytes = c.slot_stride * 2u;
    v.page_table = c.page_table;
    v.mass = c.mass;
    v.positions = c.positions;
    v.table_pages = c.table_pages;
    v.n_pages = c.n_pages;
    v.page_slots = c.page_slots;
    v.kv_heads = c.kv_heads;
    v.capacity = c.table_pages * c.page_slots;
    v.status = ctx->device_status;
    return v;
}

// The checks every paged call makes of its cache and lane table before anything is enqueued.
inline tatara_status check_paged(tatara_ctx* ctx, const tatara_paged_cache* c, const void* lanes, uint32_t n_lanes) {
    if (c == nullptr || lanes == nullptr || !c->keys || !c->values || !c->page_table)
        return fail(ctx, TATARA_INVALID_BUFFER, "paged cache: null buffer");
    if (!aligned(c->keys, 16) || !aligned(c->values, 16) || !aligned(c->page_table, 4) || !aligned(c->mass, 4) ||
        !aligned(c->positions, 4) || !aligned(lanes, 8))
        return fail(ctx, TATARA_INVALID_BUFFER, "paged cache: misaligned buffer");
    if (c->dtype != TATARA_BF16 && c->dtype != TATARA_F16)
        return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged cache: dtype");
    if (c->head_dim != 64u && c->head_dim != 128u && c->head_dim != 256u)
        return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged cache: head_dim is 64, 128 or 256");
    if (c->kv_heads == 0 || c->kv_heads > 1024u) return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged cache: kv heads");
    if (c->page_slots == 0 || c->page_slots % kPagedSlice != 0 || c->page_slots > kPagedMaxPageSlots)
        return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged cache: page_slots is a multiple of 16, at most 1024");
    if (c->table_pages == 0 || c->n_pages == 0 || c->table_lanes == 0 ||
        uint64_t(c->table_pages) * c->page_slots > (1ull << 30))
        return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged cache: page table");
    if (c->page_stride % 8u || c->head_stride % 8u || c->slot_stride % 8u || c->slot_stride < c->head_dim ||
        c->head_stride < c->head_dim || c->page_stride < c->head_dim)
        return fail(ctx, TATARA_INVALID_DISPATCH_EXTENT, "paged cache: strides are multiples of 8 elements, at least head_dim");
    if (n_lanes == 0 || n_lanes > TATARA_MAX_LANES || n_lanes > c->table_lanes)
        return fail(ctx, TATARA_INVALID_STREAM_GROUP, "paged cache: lane count");
    return TATARA_OK;
}

// Makes the context's device current for the length of a call.
struct DeviceGuard {
    int before = -1;
    bool switched = false;
    explicit DeviceGuard(const tatara_ctx* ctx) {
        if (cudaGetDevice(&before) == cudaSuccess && before != ctx->device) switched = cudaSetDevice(ctx->device) == cudaSuccess;
    }
    ~DeviceGuard() {
        if (switched) cudaSetDevice(before);
    }
};

// A launch that may be staged while its predecessor in the stream finishes (the kernel waits for it itself).  carveout: the share
// of an SM's memory, in percent, that is to be shared memory; -1: the driver's choice.
template <typename... Params, typename... Args>
inline cudaError_t launch_staged_carved(int carveout, void (*kernel)(Params...), dim3 grid, uint32_t threads, uint32_t smem, cudaStream_t stream,
                                        Args&&... args) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributePreferredSharedMemoryCarveout;
    attr[1].val.sharedMemCarveout = uint32_t(carveout);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = carveout < 0 ? 1 : 2;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}
template <typename... Params, typename... Args>
inline cudaError_t launch_staged(void (*kernel)(Params...), dim3 grid, uint32_t threads, uint32_t smem, cudaStream_t stream, Args&&... args) {
    return launch_staged_carved(-1, kernel, grid, threads, smem, stream, static_cast<Args&&>(args)...);
}
__device__ __forceinline__ void wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void release_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

} // namespace tb
