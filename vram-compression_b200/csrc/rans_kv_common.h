// What the kernels of the paged key-value cache share: the cache as a kernel
// argument, page lookups with their bounds check, and the host's checks.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

#include "../../include/rans_kv.h"

namespace rb200kv {

constexpr int kSms = 148;                // B200; grids are sized by it, no kernel depends on it
constexpr int kMaxSubgroups = 16;        // head groups of one kv head (see rans_kv_attend.cu)

__device__ __forceinline__ void raise(const RansKvCache& c, int bit) { atomicOr(c.status, bit); }

// Division of 0 <= n < 2^31 by a fixed number: (umulhi(n, mul) + n) >> shift, with mul = floor(2^32 (2^shift - d) / d) + 1
// and shift = ceil(log2 d).  The compiler's division is some thirty instructions, more than the rest of a page lookup.
struct Divider {
    uint32_t mul;
    int shift;
    __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
    static Divider of(uint32_t d) {
        int shift = 0;
        while (((uint64_t)1 << shift) < d) ++shift;
        return {(uint32_t)(((((uint64_t)1 << shift) - d) << 32) / d + 1), shift};
    }
};

// length[b] within what the table can hold; never follows a bad one.
__device__ __forceinline__ int checked_length(const RansKvCache& c, int b) {
    const int n = c.length[b];
    const int64_t room = (int64_t)c.table_cols * c.page;
    if (n < 0 || n > room) {
        raise(c, RANS_KV_BAD_LENGTH);
        return n < 0 ? 0 : (int)room;
    }
    return n;
}

// The page that holds place t of sequence b, or -1.
__device__ __forceinline__ int checked_page(const RansKvCache& c, int b, int page_of_t) {
    const int p = c.table[(int64_t)b * c.table_cols + page_of_t];
    if (p < 0 || p >= c.pages) {
        raise(c, RANS_KV_BAD_PAGE);
        return -1;
    }
    return p;
}

// The kernels of a step follow one another: each may start while the one before it ends, waits for it (its writes are
// then visible) before it reads anything that changes, and lets its own follower start.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class Args>
inline int launch_after(void (*kernel)(Args), dim3 grid, int threads, size_t shared, int cluster, cudaStream_t stream, const Args& args) {
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, args);
    return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

inline int64_t counter_bytes(const RansKvCache& c) {
    return 256 + (((int64_t)c.batch * c.kv_heads * kMaxSubgroups * 4 + 255) & ~(int64_t)255);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// 0, -1 or -2 (rans_kv.h).
inline int check_cache(const RansKvCache* c) {
    if (c == nullptr) return -2;
    if (c->kind != RANS_KV_BF16 && c->kind != RANS_KV_FP16 && c->kind != RANS_KV_MXFP4) return -1;
    if (c->dim != 64 && c->dim != 128 && c->dim != 256) return -1;
    if (c->pages < 1 || c->page < 16 || c->page % 16 != 0 || c->page > (1 << 20) || c->kv_heads < 1 || c->kv_heads > 1024 || c->batch < 1 ||
        c->batch > RANS_KV_MAX_BATCH || (int64_t)c->batch * c->kv_heads > 65535 || c->table_cols < 1 || c->reserved != 0)
        return -2;
    if ((int64_t)c->table_cols * c->page > (int64_t)1 << 30) return -2;
    if ((int64_t)c->pages * c->kv_heads * c->page > (int64_t)1 << 40) return -2;
    if (c->k == nullptr || c->v == nullptr || c->table == nullptr || c->length == nullptr || c->seen == nullptr ||
        c->status == nullptr || c->workspace == nullptr || !aligned16(c->k) || !aligned16(c->v) ||
        !aligned16(c->workspace))
        return -2;
    if (c->kind == RANS_KV_MXFP4) {
        if (c->k_scale == nullptr || c->v_scale == nullptr || !aligned16(c->k_scale) || !aligned16(c->v_scale)) return -2;
    } else if ((c->k_page | c->k_head | c->k_slot | c->v_page | c->v_head | c->v_slot) & 15) {
        return -2;
    }
    if (c->workspace_bytes < counter_bytes(*c)) return -3;
    return 0;
}

// Row addresses.  4-bit pages are contiguous, so their strides follow from the shape.
inline void fill_strides(RansKvCache& c) {
    if (c.kind != RANS_KV_MXFP4) return;
    c.k_slot = c.v_slot = c.dim / 2;
    c.k_head = c.v_head = (int64_t)c.page * (c.dim / 2);
    c.k_page = c.v_page = c.k_head * c.kv_heads;
}

}  // namespace rb200kv
