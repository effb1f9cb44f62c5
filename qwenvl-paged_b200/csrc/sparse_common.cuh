// Shared by the sparse-attention kernels (rotary append, block summaries,
// block selection, decode over selected blocks): 16-byte vectors of either
// element type, minimum and maximum that keep NaN, launch with programmatic
// stream serialization, and the argument checks the four calls have in common.
#pragma once

#include "qvp_device.cuh"
#include "qvp_internal.h"

namespace qvp {

// VEC elements of T, loaded and stored as one 16-byte word (VEC = 1: one by one).
template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Vec {
    T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Vec<T, VEC> load_vec(const T* p) {
    static_assert(VEC == 1 || VEC * sizeof(T) == 16, "16-byte vectors");
    Vec<T, VEC> r;
    if constexpr (VEC == 1)
        r.v[0] = *p;
    else
        *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
    return r;
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, VEC>& r) {
    if constexpr (VEC == 1)
        *p = r.v[0];
    else
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
}

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ __nv_bfloat16 min_nan(__nv_bfloat16 a, __nv_bfloat16 b) { return __hmin_nan(a, b); }
__device__ __forceinline__ __nv_bfloat16 max_nan(__nv_bfloat16 a, __nv_bfloat16 b) { return __hmax_nan(a, b); }

// lo = min(lo, x), hi = max(hi, x) element by element; a NaN stays (a summary
// that hid one would hide it from the score).
template <typename T, int VEC>
__device__ __forceinline__ void widen(Vec<T, VEC>& lo, Vec<T, VEC>& hi, const Vec<T, VEC>& xlo, const Vec<T, VEC>& xhi) {
    if constexpr (sizeof(T) == 2 && VEC > 1) {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            auto& l = *reinterpret_cast<__nv_bfloat162*>(&lo.v[i]);
            auto& h = *reinterpret_cast<__nv_bfloat162*>(&hi.v[i]);
            l = __hmin2_nan(l, *reinterpret_cast<const __nv_bfloat162*>(&xlo.v[i]));
            h = __hmax2_nan(h, *reinterpret_cast<const __nv_bfloat162*>(&xhi.v[i]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            lo.v[i] = min_nan(lo.v[i], xlo.v[i]);
            hi.v[i] = max_nan(hi.v[i], xhi.v[i]);
        }
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void start_range(Vec<T, VEC>& lo, Vec<T, VEC>& hi) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        lo.v[i] = from_float<T>(INFINITY);
        hi.v[i] = from_float<T>(-INFINITY);
    }
}

// The kernels are launched as programmatic dependents: their CTAs may be
// placed while the kernel before them drains. They touch no memory before
// this wait, which ends when that kernel is complete and its writes visible.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the next programmatic dependent be placed (it waits as above).
__device__ __forceinline__ void allow_next_kernel() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launches `kern` on `st` as a programmatic dependent of what precedes it,
// in clusters of `cluster` CTAs along x (1 = none).
template <typename... Params, typename... Args>
int launch_dependent(const char* what, void (*kern)(Params...), dim3 grid, uint32_t threads, size_t smem,
                     uint32_t cluster, cudaStream_t st, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cluster > 1) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster;
        attr[1].val.clusterDim.y = 1;
        attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    return check_cuda(cudaLaunchKernelEx(&cfg, kern, args...), what);
}

inline bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Shape, dtype and layer of a call of the sparse-attention group.
inline int check_shape(const qvp_block_shape& sh, int32_t dtype, uint32_t layer) {
    if (sh.tokens_per_block == 0 || sh.num_layers == 0 || sh.num_kv_heads == 0 || sh.head_dim == 0)
        return fail(QVP_ERR_INVALID, "block shape has a zero field");
    const uint32_t elem = dtype == QVP_DTYPE_F32 ? 4u : dtype == QVP_DTYPE_BF16 ? 2u : 0u;
    if (elem == 0) return fail(QVP_ERR_INVALID, "unknown dtype %d", dtype);
    if (sh.bytes_per_element != elem)
        return fail(QVP_ERR_INVALID, "bytes_per_element %u does not match the dtype", sh.bytes_per_element);
    if (layer >= sh.num_layers) return fail(QVP_ERR_INVALID, "layer %u >= num_layers %u", layer, sh.num_layers);
    if (sh.head_dim > 256) return fail(QVP_ERR_UNSUPPORTED, "head_dim %u above 256", sh.head_dim);
    // table capacities are compared as 32-bit token counts on the device
    if (sh.tokens_per_block > 65536u || sh.num_kv_heads > 65535u)
        return fail(QVP_ERR_UNSUPPORTED, "blocks of more than 65536 tokens or 65535 heads");
    // elements within a block's K are counted in 32 bits
    if (static_cast<uint64_t>(sh.tokens_per_block) * sh.num_kv_heads * sh.head_dim > 0x7fffffffu)
        return fail(QVP_ERR_UNSUPPORTED, "blocks of more than 2^31 - 1 elements of K in a layer");
    // the rows of a summary pool are counted in 32 bits; a block then has below
    // 2^59 bytes (2^16 tokens, 2^32 rows, 2^8 elements), so its size does not wrap
    if (static_cast<uint64_t>(sh.num_layers) * sh.num_kv_heads > 0xffffffffu)
        return fail(QVP_ERR_UNSUPPORTED, "more than 2^32 - 1 (layer, kv head) pairs");
    return QVP_OK;
}

// A pool of blocks of `bytes` bytes each and its tables.
inline int check_pool(const char* name, const void* base, size_t stride, size_t bytes, uint32_t elem,
                      uint32_t num_blocks) {
    if (base == nullptr) return fail(QVP_ERR_INVALID, "null %s", name);
    if (stride < bytes) return fail(QVP_ERR_INVALID, "%s stride below the block size", name);
    if (!aligned_to(base, elem) || stride % elem != 0) return fail(QVP_ERR_INVALID, "%s is not element-aligned", name);
    if (num_blocks == 0) return fail(QVP_ERR_INVALID, "empty %s", name);
    if (num_blocks > 0x7fffffffu) return fail(QVP_ERR_UNSUPPORTED, "%s of more than 2^31 blocks", name);
    if (stride > SIZE_MAX / num_blocks) return fail(QVP_ERR_UNSUPPORTED, "%s of more than 2^64 bytes", name);
    return QVP_OK;
}

// Arrays of 32-bit values that a kernel reads or writes one by one; null ones
// are fine here.
template <typename... P>
int check_words(const P*... arrays) {
    if ((... && aligned_to(arrays, 4))) return QVP_OK;
    return fail(QVP_ERR_INVALID, "an int32 or float array is not 4-byte aligned");
}

inline int check_tables(const int32_t* tables, const int32_t* lens, uint32_t pitch, uint32_t batch) {
    if (tables == nullptr || lens == nullptr) return fail(QVP_ERR_INVALID, "null table or length pointer");
    if (pitch == 0) return fail(QVP_ERR_INVALID, "empty block table");
    if (batch > 65535u) return fail(QVP_ERR_UNSUPPORTED, "batch above 65535");
    return QVP_OK;
}

// Tokens the table rows can name, as the device compares lengths with it.
inline uint32_t token_capacity(uint32_t pitch, uint32_t tokens_per_block) {
    const uint64_t n = static_cast<uint64_t>(pitch) * tokens_per_block;
    return n < 0x7fffffffu ? static_cast<uint32_t>(n) : 0x7fffffffu;
}

}  // namespace qvp
