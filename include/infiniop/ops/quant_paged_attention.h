/*
 * Paged-attention decode over pools held in 8 or 4 bits: infiniopPagedAttention
 * (include/infiniop/ops/paged_attention.h) with K and V given as codes and scales.  No counterpart in
 * the reference.
 *
 * Tensors:
 *   out           [num_seqs, num_heads, head_size]     F16 | BF16, last stride 1
 *   q             [num_seqs, num_heads, head_size]     same dtype, last stride 1
 *   k_cache, v_cache, k_scales, v_scales               as in quant_paged_caching.h, equal K and V head sizes:
 *                                                      64, 128, 192 or 256
 *   block_tables  [num_seqs, max_num_blocks_per_seq]   I64 | I32 | U32
 *   seq_lens      [num_seqs]                           same index dtype
 *   alibi_slopes  [num_heads] F32, optional (descriptor and pointer may be NULL)
 *
 * With k and v the values that the codes stand for and n = seq_lens[i] (at most block_size times the
 * table's width, also where a U32 length is 2^31 or more):
 *   out[i, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[i, h] . k_j + slope_h (j - (n - 1))),  0 <= j < n,
 * where token j of sequence i is at cache[block_tables[i][j / block_size], h / (num_heads /
 * num_kv_heads), j % block_size].  A sequence with n <= 0 leaves its output rows untouched; what the
 * pools hold behind a sequence's last token does not matter, NaN scales included.  With pools of no blocks no
 * sequence has a token, and their addresses may be NULL.
 *
 * Scores, sums and outputs are held in 32 bits.  The weights p_j times the V scale of a group (of 32 elements, or of the
 * row) are rounded to fp16 relative to the largest of their head and group, once for BF16 outputs, in two halves
 * (2^-13) for F16 ones, so that groups of any size keep their precision; those with scales below 2^-100 keep less, and F16
 * outputs of more than 4 q heads a kv head whose groups differ in size by more than 2^6 have the one rounding.
 *
 * The workspace is caller-owned scratch of at least GetWorkspaceSize bytes, 256-byte aligned, contents
 * undefined on entry; calls that may overlap on the GPU need one each.  Execute is asynchronous on
 * `stream` (NULL = the default stream), performs no allocation and no host<->device synchronisation.
 */
#ifndef __INFINIOP_QUANT_PAGED_ATTENTION_API_H__
#define __INFINIOP_QUANT_PAGED_ATTENTION_API_H__

#include "../operator_descriptor.h"

typedef struct InfiniopDescriptor *infiniopQuantPagedAttentionDescriptor_t;

__INFINI_C __export infiniStatus_t infiniopCreateQuantPagedAttentionDescriptor(
    infiniopHandle_t handle,
    infiniopQuantPagedAttentionDescriptor_t *desc_ptr,
    infiniopTensorDescriptor_t out_desc,
    infiniopTensorDescriptor_t q_desc,
    infiniopTensorDescriptor_t k_cache_desc,
    infiniopTensorDescriptor_t v_cache_desc,
    infiniopTensorDescriptor_t k_scales_desc,
    infiniopTensorDescriptor_t v_scales_desc,
    infiniopTensorDescriptor_t block_tables_desc,
    infiniopTensorDescriptor_t seq_lens_desc,
    infiniopTensorDescriptor_t alibi_slopes_desc,
    float scale);

__INFINI_C __export infiniStatus_t infiniopGetQuantPagedAttentionWorkspaceSize(
    infiniopQuantPagedAttentionDescriptor_t desc, size_t *size);

__INFINI_C __export infiniStatus_t infiniopQuantPagedAttention(
    infiniopQuantPagedAttentionDescriptor_t desc,
    void *workspace,
    size_t workspace_size,
    void *out,
    const void *q,
    const void *k_cache,
    const void *v_cache,
    const void *k_scales,
    const void *v_scales,
    const void *block_tables,
    const void *seq_lens,
    const void *alibi_slopes,
    void *stream);

__INFINI_C __export infiniStatus_t infiniopDestroyQuantPagedAttentionDescriptor(
    infiniopQuantPagedAttentionDescriptor_t desc);

#endif
