// What the quantised-pool operators share: the geometry of a pool of codes with its scales, checked once
// when a descriptor is created (include/infiniop/ops/quant_paged_caching.h says what is accepted).
#ifndef INFINIOP_B200_QUANT_POOL_H
#define INFINIOP_B200_QUANT_POOL_H

#include "../common.h"

#include <cstdlib>
#include <new>

namespace b200::quant_paged_cache {

constexpr int kGroup4 = 32; // elements that share a scale in the 4-bit form

// One of the two pools; strides of the codes in bytes, of the scales in elements.
struct Pool {
    size_t head = 0;
    size_t groups = 0;
    ptrdiff_t block = 0, kv_head = 0, slot = 0;
    ptrdiff_t s_block = 0, s_head = 0, s_slot = 0;
};

struct Pools {
    int bits = 0;
    size_t num_blocks = 0, num_kv_heads = 0, block_size = 0;
    Pool k, v;
};

inline infiniStatus_t describePool(Pool &p, int bits, infiniopTensorDescriptor_t codes, infiniopTensorDescriptor_t scales) {
    p.head = codes->dim(3) * (bits == 4 ? 2 : 1);
    p.groups = scales->dim(3);
    B200_RETURN_IF(p.head == 0 || p.head % 32 != 0 || p.head > 1024, INFINI_STATUS_BAD_TENSOR_SHAPE);
    B200_RETURN_IF(p.groups != (bits == 4 ? p.head / kGroup4 : 1), INFINI_STATUS_BAD_TENSOR_SHAPE);
    for (size_t i = 0; i < 3; ++i) {
        B200_RETURN_IF(codes->dim(i) != scales->dim(i), INFINI_STATUS_BAD_TENSOR_SHAPE);
    }
    B200_RETURN_IF(codes->stride(3) != 1 || (p.groups > 1 && scales->stride(3) != 1), INFINI_STATUS_BAD_TENSOR_STRIDES);
    p.block = codes->stride(0);
    p.kv_head = codes->stride(1);
    p.slot = codes->stride(2);
    p.s_block = scales->stride(0);
    p.s_head = scales->stride(1);
    p.s_slot = scales->stride(2);
    return INFINI_STATUS_SUCCESS;
}

inline infiniStatus_t describePools(Pools &out, infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache,
                                    infiniopTensorDescriptor_t k_scales, infiniopTensorDescriptor_t v_scales) {
    B200_RETURN_IF(k_cache->dtype != INFINI_DTYPE_I8 && k_cache->dtype != INFINI_DTYPE_U8, INFINI_STATUS_BAD_TENSOR_DTYPE);
    B200_RETURN_IF(v_cache->dtype != k_cache->dtype, INFINI_STATUS_BAD_TENSOR_DTYPE);
    B200_RETURN_IF(k_scales->dtype != INFINI_DTYPE_BF16 || v_scales->dtype != INFINI_DTYPE_BF16, INFINI_STATUS_BAD_TENSOR_DTYPE);
    B200_RETURN_IF(k_cache->ndim() != 4 || v_cache->ndim() != 4 || k_scales->ndim() != 4 || v_scales->ndim() != 4,
                   INFINI_STATUS_BAD_TENSOR_SHAPE);
    out.bits = k_cache->dtype == INFINI_DTYPE_U8 ? 4 : 8;
    out.num_blocks = k_cache->dim(0);
    out.num_kv_heads = k_cache->dim(1);
    out.block_size = k_cache->dim(2);
    for (size_t i = 0; i < 3; ++i) {
        B200_RETURN_IF(v_cache->dim(i) != k_cache->dim(i), INFINI_STATUS_BAD_TENSOR_SHAPE);
    }
    B200_RETURN_IF(out.block_size == 0 || out.block_size > 65536u || out.num_blocks > 0x7fffffffu || out.num_kv_heads > 65535u,
                   INFINI_STATUS_BAD_TENSOR_SHAPE); // kernels count these in 32 bits
    const infiniStatus_t st = describePool(out.k, out.bits, k_cache, k_scales);
    B200_RETURN_IF(st != INFINI_STATUS_SUCCESS, st);
    return describePool(out.v, out.bits, v_cache, v_scales);
}

inline bool envIs(const char *name, char value) {
    const char *v = std::getenv(name);
    return v != nullptr && v[0] == value;
}

inline bool alignedTo(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

} // namespace b200::quant_paged_cache

#endif
