/*
 * Paged caching into pools held in 8 or 4 bits: new K/V rows are quantised as they are written to
 * their slots, and rows are turned back into values as they are gathered by slot.  No counterpart in
 * the reference, whose pools keep the dtype of the rows (include/infiniop/ops/paged_caching.h:24-75).
 *
 * Storage (the same for the three quantised operators):
 *   k_cache   [num_blocks, num_kv_heads, block_size, head_size]       I8: 8-bit codes, or
 *             [num_blocks, num_kv_heads, block_size, head_size / 2]   U8: two 4-bit codes a byte, the even
 *                                                                     element in bits 0-3, two's complement
 *   v_cache   the same with v_head_size, the same dtype
 *   k_scales  [num_blocks, num_kv_heads, block_size, groups]          BF16; groups = 1 (I8: one scale for a
 *   v_scales  the same                                                 row) or head size / 32 (U8: one scale
 *                                                                     for each 32 elements)
 * Any block, head and slot strides; the last stride is 1.  Head sizes are multiples of 32 up to 1024.
 *
 * Scales are never negative.  Quantising a group of values x with A = max |x| and Q = 127 (I8) or 7 (U8):
 *   scale = A / Q rounded to fp32, then to bf16 (both to nearest even), or 0 where that is below 2^-126;
 *   code  = x / scale to the nearest integer, halves away from zero, so |code| <= Q;
 *   a group that holds an infinity or a NaN gets the scale NaN and codes 0: it reads back as NaN.
 * A code stands for the value code * scale.  A pool of zero bytes stands for zeros.
 *
 * Pools may have no blocks, and null addresses then: no sequence has a token there, every slot is outside and
 * treated as padding, reported as in checked mode (include/infiniop/ops/kernel_status.h) where it is not negative.
 */
#ifndef __INFINIOP_QUANT_PAGED_CACHING_API_H__
#define __INFINIOP_QUANT_PAGED_CACHING_API_H__

#include "../operator_descriptor.h"

typedef struct InfiniopDescriptor *infiniopQuantPagedCachingDescriptor_t;
typedef struct InfiniopDescriptor *infiniopQuantPagedCacheReadDescriptor_t;

/*
 * Write: row i of k [num_tokens, num_kv_heads, head_size] and v [.., v_head_size] (F16 | BF16, last
 * stride 1) goes to slot slot_mapping[i] (I64, dense): block slot / block_size, offset slot %
 * block_size.  A negative slot marks padding and is skipped.  The non-negative slots of one call must
 * differ: of two rows for the same slot, parts of both may remain.  Workspace size is 0.
 */
__INFINI_C __export infiniStatus_t infiniopCreateQuantPagedCachingDescriptor(
    infiniopHandle_t handle,
    infiniopQuantPagedCachingDescriptor_t *desc_ptr,
    infiniopTensorDescriptor_t k_cache_desc,
    infiniopTensorDescriptor_t v_cache_desc,
    infiniopTensorDescriptor_t k_scales_desc,
    infiniopTensorDescriptor_t v_scales_desc,
    infiniopTensorDescriptor_t k_desc,
    infiniopTensorDescriptor_t v_desc,
    infiniopTensorDescriptor_t slot_mapping_desc);

__INFINI_C __export infiniStatus_t infiniopGetQuantPagedCachingWorkspaceSize(
    infiniopQuantPagedCachingDescriptor_t desc, size_t *size);

__INFINI_C __export infiniStatus_t infiniopQuantPagedCaching(
    infiniopQuantPagedCachingDescriptor_t desc,
    void *workspace,
    size_t workspace_size,
    void *k_cache,
    void *v_cache,
    void *k_scales,
    void *v_scales,
    const void *k,
    const void *v,
    const void *slot_mapping,
    void *stream);

__INFINI_C __export infiniStatus_t infiniopDestroyQuantPagedCachingDescriptor(
    infiniopQuantPagedCachingDescriptor_t desc);

/*
 * Read: row i of k [num_tokens, num_kv_heads, head_size] and v [.., v_head_size] (F16 | BF16 | F32, last
 * stride 1) becomes the values of slot slot_mapping[i], each product code * scale rounded once to the
 * rows' type; zeros where the slot is negative.  Slots may repeat and come in any order: with the slots
 * of a sequence's tokens in order this is its history as dense rows.  Workspace size is 0.
 */
__INFINI_C __export infiniStatus_t infiniopCreateQuantPagedCacheReadDescriptor(
    infiniopHandle_t handle,
    infiniopQuantPagedCacheReadDescriptor_t *desc_ptr,
    infiniopTensorDescriptor_t k_desc,
    infiniopTensorDescriptor_t v_desc,
    infiniopTensorDescriptor_t k_cache_desc,
    infiniopTensorDescriptor_t v_cache_desc,
    infiniopTensorDescriptor_t k_scales_desc,
    infiniopTensorDescriptor_t v_scales_desc,
    infiniopTensorDescriptor_t slot_mapping_desc);

__INFINI_C __export infiniStatus_t infiniopGetQuantPagedCacheReadWorkspaceSize(
    infiniopQuantPagedCacheReadDescriptor_t desc, size_t *size);

__INFINI_C __export infiniStatus_t infiniopQuantPagedCacheRead(
    infiniopQuantPagedCacheReadDescriptor_t desc,
    void *workspace,
    size_t workspace_size,
    void *k,
    void *v,
    const void *k_cache,
    const void *v_cache,
    const void *k_scales,
    const void *v_scales,
    const void *slot_mapping,
    void *stream);

__INFINI_C __export infiniStatus_t infiniopDestroyQuantPagedCacheReadDescriptor(
    infiniopQuantPagedCacheReadDescriptor_t desc);

#endif
