// infiniopQuantPagedAttention: the descriptor, and the kernel for layouts that the tiles kernel (attention_tiles.cu)
// does not take: blocks that are no multiple of 8 tokens, strides or addresses that are no multiple of 16 bytes, K and V
// pools laid out differently.
//
// quantAttentionRowsKernel: one CTA of four warps per (sequence, q head).  Warp w walks tokens w, w + 4, ...;
// its lanes split the head in pairs, a shuffle reduction makes the score, and each warp keeps a running
// maximum and sum of the softmax (one pass over the codes), merged through shared memory at the end.  It reads
// single bytes, so pools of any stride and alignment go through it; every q head of a group reads the codes
// again.
#include "attention.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>

namespace b200::quant_paged_cache {

struct AttentionDescriptor {
    OpDescriptorBase base;
    AttentionInfo info;
    TilesPlan tiles;
};

constexpr int kRowWarps = 4;
constexpr int kMaxPairs = 4; // 256 elements: four pairs a lane

__device__ __forceinline__ float loadValue(const void *p, long long i, int is_bf16) {
    return is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]) : __half2float(static_cast<const __half *>(p)[i]);
}

__device__ __forceinline__ void storeValue(void *p, long long i, float v, int is_bf16) {
    if (is_bf16) {
        static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    } else {
        static_cast<__half *>(p)[i] = __float2half_rn(v);
    }
}

template <int BITS>
__device__ __forceinline__ float2 valuePair(const unsigned char *row, const unsigned short *scales, int d) {
    if constexpr (BITS == 8) {
        const float s = __uint_as_float(static_cast<unsigned>(scales[0]) << 16);
        return make_float2(static_cast<float>(static_cast<signed char>(row[d])) * s, static_cast<float>(static_cast<signed char>(row[d + 1])) * s);
    } else {
        const float s = __uint_as_float(static_cast<unsigned>(scales[d / kGroup4]) << 16);
        const int b = row[d >> 1];
        return make_float2(static_cast<float>((b << 28) >> 28) * s, static_cast<float>((b << 24) >> 28) * s);
    }
}

template <int BITS>
__global__ void __launch_bounds__(kRowWarps * 32) quantAttentionRowsKernel(const AttentionArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ float smem[]; // q[head] | per warp: m, l, acc[head]
    const int head = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.num_heads));
    const int seq = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.num_heads));
    const long long len = tokensOf(a, seq);
    if (len == 0) {
        return;
    }
    const int kv_head = head / a.group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float *q_s = smem;
    float *merge = smem + a.head_size;
    const int merge_stride = a.head_size + 2;
    for (int i = threadIdx.x; i < a.head_size; i += blockDim.x) {
        q_s[i] = loadValue(a.q, seq * a.q_seq + head * a.q_head + i, a.is_bf16);
    }
    __syncthreads();
    const float slope = a.alibi != nullptr ? a.alibi[head] * 1.4426950408889634f : 0.f;

    float m = kLowest, l = 0.f;
    float2 acc[kMaxPairs];
#pragma unroll
    for (int i = 0; i < kMaxPairs; ++i) {
        acc[i] = make_float2(0.f, 0.f);
    }
    // a table may name more than 2^31 tokens: they are counted in 64 bits, and pages without a division
    long long page = warp / a.block_size;
    int off = warp % a.block_size;
    for (long long t = warp; t < len; t += kRowWarps) {
        const long long block = blockAt(a, seq * a.table_seq, page);
        const unsigned char *k = a.k_codes + block * a.k_block + kv_head * a.k_head + off * a.k_slot;
        const unsigned char *v = a.v_codes + block * a.v_block + kv_head * a.v_head + off * a.v_slot;
        const unsigned short *ks = a.k_scales + block * a.ks_block + kv_head * a.ks_head + off * a.ks_slot;
        const unsigned short *vs = a.v_scales + block * a.vs_block + kv_head * a.vs_head + off * a.vs_slot;
        float dot = 0.f;
        for (int d = 2 * lane; d < a.head_size; d += 64) {
            const float2 x = valuePair<BITS>(k, ks, d);
            dot = fmaf(q_s[d], x.x, dot);
            dot = fmaf(q_s[d + 1], x.y, dot);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            dot += __shfl_xor_sync(0xffffffffu, dot, o);
        }
        float s = dot * a.scale_log2e;
        if (slope != 0.f) {
            s += slope * static_cast<float>(t - (len - 1));
        }
        const float m_new = maxNan(m, s);
        const float alpha = exp2f(m - m_new); // the first token: 0
        const float p = exp2f(s - m_new);
        l = l * alpha + p;
        m = m_new;
#pragma unroll
        for (int i = 0; i < kMaxPairs; ++i) {
            const int d = 2 * lane + 64 * i;
            if (d < a.head_size) {
                const float2 x = valuePair<BITS>(v, vs, d);
                acc[i].x = fmaf(p, x.x, acc[i].x * alpha);
                acc[i].y = fmaf(p, x.y, acc[i].y * alpha);
            }
        }
        for (off += kRowWarps; off >= a.block_size; off -= a.block_size) {
            ++page;
        }
    }
    float *mine = merge + warp * merge_stride;
    if (lane == 0) {
        mine[0] = m;
        mine[1] = l;
    }
#pragma unroll
    for (int i = 0; i < kMaxPairs; ++i) {
        const int d = 2 * lane + 64 * i;
        if (d < a.head_size) {
            mine[2 + d] = acc[i].x;
            mine[2 + d + 1] = acc[i].y;
        }
    }
    __syncthreads();
    float m_all = kLowest;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
        m_all = maxNan(m_all, merge[w * merge_stride]);
    }
    float weight[kRowWarps], l_all = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
        weight[w] = exp2f(merge[w * merge_stride] - m_all); // a warp without a token has kLowest and 0
        l_all += weight[w] * merge[w * merge_stride + 1];
    }
    const float inv = 1.f / l_all;
    for (int d = threadIdx.x; d < a.head_size; d += blockDim.x) {
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) {
            o = fmaf(weight[w], merge[w * merge_stride + 2 + d], o);
        }
        storeValue(a.out, seq * a.o_seq + head * a.o_head + d, o * inv, a.is_bf16);
    }
}

infiniStatus_t launchRows(const AttentionInfo &info, const AttentionArgs &a, cudaStream_t stream) {
    const unsigned long long ctas = static_cast<unsigned long long>(a.num_seqs) * static_cast<unsigned long long>(a.num_heads);
    B200_RETURN_IF(ctas > 0x7fffffffull, INFINI_STATUS_BAD_TENSOR_SHAPE);
    const size_t smem = sizeof(float) * (a.head_size + kRowWarps * (a.head_size + 2));
    cudaLaunchAttribute pdl;
    pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl.val.programmaticStreamSerializationAllowed = info.use_pdl ? 1 : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(kRowWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &pdl;
    cfg.numAttrs = 1;
    (void)cudaLaunchKernelEx(&cfg, info.pools.bits == 4 ? quantAttentionRowsKernel<4> : quantAttentionRowsKernel<8>, a);
    return checkLaunch("quantAttentionRowsKernel");
}

static infiniStatus_t makeInfo(AttentionInfo &I, infiniopTensorDescriptor_t out, infiniopTensorDescriptor_t q,
                               infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache, infiniopTensorDescriptor_t k_scales,
                               infiniopTensorDescriptor_t v_scales, infiniopTensorDescriptor_t tables, infiniopTensorDescriptor_t lens,
                               infiniopTensorDescriptor_t alibi, float scale) {
    B200_RETURN_IF(q->dtype != INFINI_DTYPE_F16 && q->dtype != INFINI_DTYPE_BF16, INFINI_STATUS_BAD_TENSOR_DTYPE);
    B200_RETURN_IF(out->dtype != q->dtype, INFINI_STATUS_BAD_TENSOR_DTYPE);
    const infiniDtype_t ix = tables->dtype;
    B200_RETURN_IF((ix != INFINI_DTYPE_I64 && ix != INFINI_DTYPE_I32 && ix != INFINI_DTYPE_U32) || lens->dtype != ix,
                   INFINI_STATUS_BAD_TENSOR_DTYPE);
    B200_RETURN_IF(q->ndim() != 3 || out->ndim() != 3 || tables->ndim() != 2 || lens->ndim() != 1, INFINI_STATUS_BAD_TENSOR_SHAPE);
    infiniStatus_t st = describePools(I.pools, k_cache, v_cache, k_scales, v_scales);
    B200_RETURN_IF(st != INFINI_STATUS_SUCCESS, st);
    I.num_seqs = q->dim(0);
    I.num_heads = q->dim(1);
    I.head_size = q->dim(2);
    I.max_blocks = tables->dim(1);
    const size_t hd = I.head_size, kvh = I.pools.num_kv_heads;
    B200_RETURN_IF(hd != 64 && hd != 128 && hd != 192 && hd != 256, INFINI_STATUS_BAD_TENSOR_SHAPE);
    B200_RETURN_IF(I.pools.k.head != hd || I.pools.v.head != hd, INFINI_STATUS_BAD_TENSOR_SHAPE);
    B200_RETURN_IF(kvh == 0 || I.num_heads % kvh != 0, INFINI_STATUS_BAD_TENSOR_SHAPE);
    B200_RETURN_IF(out->dim(0) != I.num_seqs || out->dim(1) != I.num_heads || out->dim(2) != hd, INFINI_STATUS_BAD_TENSOR_SHAPE);
    B200_RETURN_IF(tables->dim(0) != I.num_seqs || lens->dim(0) != I.num_seqs, INFINI_STATUS_BAD_TENSOR_SHAPE);
    B200_RETURN_IF(I.num_seqs > 0x7fffffffu || I.num_heads > 65535u || I.max_blocks > 0x7fffffffu, INFINI_STATUS_BAD_TENSOR_SHAPE);
    B200_RETURN_IF(q->stride(2) != 1 || out->stride(2) != 1, INFINI_STATUS_BAD_TENSOR_STRIDES);
    B200_RETURN_IF((I.max_blocks > 1 && tables->stride(1) != 1) || (I.num_seqs > 1 && lens->stride(0) != 1), INFINI_STATUS_BAD_TENSOR_STRIDES);
    I.has_alibi = alibi != nullptr;
    if (I.has_alibi) {
        B200_RETURN_IF(alibi->dtype != INFINI_DTYPE_F32, INFINI_STATUS_BAD_TENSOR_DTYPE);
        B200_RETURN_IF(alibi->ndim() != 1 || alibi->dim(0) != I.num_heads, INFINI_STATUS_BAD_TENSOR_SHAPE);
        B200_RETURN_IF(I.num_heads > 1 && alibi->stride(0) != 1, INFINI_STATUS_BAD_TENSOR_STRIDES);
    }
    I.dtype = q->dtype;
    I.index_dtype = ix;
    I.q_seq = q->stride(0);
    I.q_head = q->stride(1);
    I.o_seq = out->stride(0);
    I.o_head = out->stride(1);
    I.table_seq = tables->stride(0);
    I.scale = scale;
    return INFINI_STATUS_SUCCESS;
}

static AttentionArgs makeArgs(const AttentionInfo &I) {
    AttentionArgs a = {};
    a.num_seqs = static_cast<int>(I.num_seqs);
    a.num_heads = static_cast<int>(I.num_heads);
    a.num_kv_heads = static_cast<int>(I.pools.num_kv_heads);
    a.group = a.num_heads / a.num_kv_heads;
    a.head_size = static_cast<int>(I.head_size);
    a.block_size = static_cast<int>(I.pools.block_size);
    a.max_blocks = static_cast<int>(I.max_blocks);
    a.index_is_64 = I.index_dtype == INFINI_DTYPE_I64 ? 1 : 0;
    a.length_kind = a.index_is_64 ? kLength64 : I.index_dtype == INFINI_DTYPE_U32 ? kLengthU32 : kLength32;
    a.is_bf16 = I.dtype == INFINI_DTYPE_BF16 ? 1 : 0;
    a.q_seq = I.q_seq;
    a.q_head = I.q_head;
    a.o_seq = I.o_seq;
    a.o_head = I.o_head;
    a.table_seq = I.table_seq;
    const Pool &k = I.pools.k, &v = I.pools.v;
    a.k_block = k.block, a.k_head = k.kv_head, a.k_slot = k.slot;
    a.v_block = v.block, a.v_head = v.kv_head, a.v_slot = v.slot;
    a.ks_block = k.s_block, a.ks_head = k.s_head, a.ks_slot = k.s_slot;
    a.vs_block = v.s_block, a.vs_head = v.s_head, a.vs_slot = v.s_slot;
    a.scale_log2e = I.scale * 1.4426950408889634f;
    a.kernel_flags = I.kernel_flags;
    a.check_indices = (I.check_indices && I.kernel_flags != nullptr) ? 1 : 0;
    a.num_blocks = static_cast<long long>(I.pools.num_blocks);
    return a;
}

} // namespace b200::quant_paged_cache

using b200::OpKind;
using b200::quant_paged_cache::AttentionDescriptor;
namespace qc = b200::quant_paged_cache;

__INFINI_C infiniStatus_t infiniopCreateQuantPagedAttentionDescriptor(
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
    float scale) {
    B200_RETURN_IF(handle == nullptr || desc_ptr == nullptr, INFINI_STATUS_NULL_POINTER);
    B200_RETURN_IF(out_desc == nullptr || q_desc == nullptr || k_cache_desc == nullptr || v_cache_desc == nullptr || k_scales_desc == nullptr
                       || v_scales_desc == nullptr || block_tables_desc == nullptr || seq_lens_desc == nullptr,
                   INFINI_STATUS_NULL_POINTER);
    B200_RETURN_IF(handle->device != INFINI_DEVICE_NVIDIA, INFINI_STATUS_DEVICE_TYPE_NOT_SUPPORTED);
    qc::AttentionInfo info = {};
    const infiniStatus_t st = qc::makeInfo(info, out_desc, q_desc, k_cache_desc, v_cache_desc, k_scales_desc, v_scales_desc,
                                           block_tables_desc, seq_lens_desc, alibi_slopes_desc, scale);
    B200_RETURN_IF(st != INFINI_STATUS_SUCCESS, st);
    auto *h = reinterpret_cast<b200::Handle *>(handle);
    info.kernel_flags = h->props->kernel_flags;
    info.check_indices = qc::envIs("INFINIOP_PAGED_CHECK_INDICES", '1');
    info.use_pdl = !qc::envIs("INFINIOP_PAGED_DECODE_PDL", '0');
    auto *d = new (std::nothrow) AttentionDescriptor{{handle->device, handle->device_id, OpKind::QuantPagedAttention, h->props}, info, {}};
    B200_RETURN_IF(d == nullptr, INFINI_STATUS_INTERNAL_ERROR);
    // INFINIOP_QUANT_ATTENTION_PATH = auto (default) | rows
    if (!qc::envIs("INFINIOP_QUANT_ATTENTION_PATH", 'r')) {
        d->tiles = qc::planTiles(info, *h->props);
    }
    *desc_ptr = reinterpret_cast<infiniopQuantPagedAttentionDescriptor_t>(d);
    return INFINI_STATUS_SUCCESS;
}

__INFINI_C infiniStatus_t infiniopGetQuantPagedAttentionWorkspaceSize(
    infiniopQuantPagedAttentionDescriptor_t desc, size_t *size) {
    B200_RETURN_IF(desc == nullptr || size == nullptr, INFINI_STATUS_NULL_POINTER);
    auto *d = reinterpret_cast<AttentionDescriptor *>(desc);
    B200_RETURN_IF(d->base.kind != OpKind::QuantPagedAttention, INFINI_STATUS_BAD_PARAM);
    *size = d->tiles.workspace_bytes;
    return INFINI_STATUS_SUCCESS;
}

__INFINI_C infiniStatus_t infiniopQuantPagedAttention(
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
    void *stream) {
    B200_RETURN_IF(desc == nullptr, INFINI_STATUS_NULL_POINTER);
    auto *d = reinterpret_cast<AttentionDescriptor *>(desc);
    B200_RETURN_IF(d->base.kind != OpKind::QuantPagedAttention, INFINI_STATUS_BAD_PARAM);
    const qc::AttentionInfo &I = d->info;
    if (I.num_seqs == 0 || I.num_heads == 0 || I.max_blocks == 0) {
        return INFINI_STATUS_SUCCESS; // no row, or no row with a token
    }
    B200_RETURN_IF(out == nullptr || q == nullptr || block_tables == nullptr || seq_lens == nullptr, INFINI_STATUS_NULL_POINTER);
    B200_RETURN_IF(I.has_alibi && alibi_slopes == nullptr, INFINI_STATUS_NULL_POINTER);
    if (I.pools.num_blocks == 0) {
        return INFINI_STATUS_SUCCESS; // no sequence has a token, and there is no block that a bad table entry could stand for
    }
    B200_RETURN_IF(k_cache == nullptr || v_cache == nullptr || k_scales == nullptr || v_scales == nullptr, INFINI_STATUS_NULL_POINTER);
    B200_RETURN_IF(workspace_size < d->tiles.workspace_bytes, INFINI_STATUS_INSUFFICIENT_WORKSPACE);
    B200_RETURN_IF(d->tiles.workspace_bytes > 0 && workspace == nullptr, INFINI_STATUS_NULL_POINTER);
    qc::AttentionArgs a = qc::makeArgs(I);
    a.out = out;
    a.q = q;
    a.k_codes = static_cast<const unsigned char *>(k_cache);
    a.v_codes = static_cast<const unsigned char *>(v_cache);
    a.k_scales = static_cast<const unsigned short *>(k_scales);
    a.v_scales = static_cast<const unsigned short *>(v_scales);
    a.block_tables = block_tables;
    a.seq_lens = seq_lens;
    a.alibi = I.has_alibi ? static_cast<const float *>(alibi_slopes) : nullptr;
    auto s = static_cast<cudaStream_t>(stream);
    return qc::tilesTakePointers(d->tiles, a, workspace) ? qc::launchTiles(I, d->tiles, a, workspace, s) : qc::launchRows(I, a, s);
}

__INFINI_C infiniStatus_t infiniopDestroyQuantPagedAttentionDescriptor(
    infiniopQuantPagedAttentionDescriptor_t desc) {
    B200_RETURN_IF(desc == nullptr, INFINI_STATUS_NULL_POINTER);
    auto *d = reinterpret_cast<AttentionDescriptor *>(desc);
    B200_RETURN_IF(d->base.kind != OpKind::QuantPagedAttention, INFINI_STATUS_BAD_PARAM);
    delete d;
    return INFINI_STATUS_SUCCESS;
}
