// Launch interface between the descriptor of the quantised paged attention and its kernels.
#ifndef INFINIOP_B200_QUANT_ATTENTION_H
#define INFINIOP_B200_QUANT_ATTENTION_H

#include "lengths.h"
#include "quant_pool.h"

namespace b200::quant_paged_cache {

struct AttentionInfo {
    Pools pools;
    infiniDtype_t dtype; // of q and out
    infiniDtype_t index_dtype;
    size_t num_seqs, num_heads, head_size, max_blocks;
    ptrdiff_t q_seq, q_head, o_seq, o_head, table_seq; // element strides
    bool has_alibi;
    float scale;
    unsigned int *kernel_flags;
    bool check_indices;
    bool use_pdl;
};

struct AttentionArgs {
    void *out;
    const void *q;
    const unsigned char *k_codes, *v_codes;
    const unsigned short *k_scales, *v_scales;
    const void *block_tables, *seq_lens;
    const float *alibi;

    int num_seqs, num_heads, num_kv_heads, group; // group: q heads of a kv head
    int head_size, block_size, max_blocks;
    int index_is_64, is_bf16;
    int length_kind; // LengthKind
    long long q_seq, q_head, o_seq, o_head, table_seq;
    long long k_block, k_head, k_slot, v_block, v_head, v_slot;             // bytes
    long long ks_block, ks_head, ks_slot, vs_block, vs_head, vs_slot;       // elements
    float scale_log2e; // scores are kept in the log2 domain

    unsigned int *kernel_flags;
    int check_indices;
    long long num_blocks;
};

__device__ __forceinline__ long long indexAt(const AttentionArgs &a, const void *base, long long i) {
    return a.index_is_64 ? static_cast<const long long *>(base)[i] : static_cast<long long>(static_cast<const int *>(base)[i]);
}

// Length of a sequence, never beyond what its row of the table can name.
__device__ __forceinline__ long long tokensOf(const AttentionArgs &a, int seq) {
    return liveTokens(storedLength(a.seq_lens, seq, a.length_kind), static_cast<long long>(a.max_blocks) * a.block_size);
}

// A block-table entry; in checked mode one outside the pool raises a flag and becomes block 0.
__device__ __forceinline__ long long blockAt(const AttentionArgs &a, long long row, long long i) {
    const long long b = indexAt(a, a.block_tables, row + i);
    if (a.check_indices && static_cast<unsigned long long>(b) >= static_cast<unsigned long long>(a.num_blocks)) {
        atomicOr(a.kernel_flags, INFINIOP_KERNEL_FLAG_BLOCK_OUT_OF_RANGE);
        return 0;
    }
    return b;
}

// Where a running maximum starts: finite, so that scores of -inf (an overflow) weigh 0 and not NaN.
constexpr float kLowest = -3.402823466e38f;

// The larger of two, NaN if one is: a NaN score has to reach the result.
__device__ __forceinline__ float maxNan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The tiles kernel (attention_tiles.cu): whether a layout suits it, and what a launch needs.
struct TilesPlan {
    bool eligible = false;
    bool dense = false; // 16 tokens of a head are one run of memory
    int grid = 0;
    int subs = 0;       // kv heads * head tiles of a group
    int head_tiles = 0;
    unsigned half_magic = 0, half_self = 0; // division by block_size / 8
    int half_shift = 0;
    bool out_words = false;
    bool unit_of_cta = false;  // no unit is cut between CTAs
    bool task_of_unit = false; // how the combine kernel's tasks are numbered
    int tasks = 0, combine_heads = 0, combine_parts = 0;
    size_t tasks_bytes = 0;
    size_t workspace_bytes = 0;
    mutable int ready = 0; // the kernel may use its shared memory
};
TilesPlan planTiles(const AttentionInfo &info, const DeviceProps &props);
bool tilesTakePointers(const TilesPlan &plan, const AttentionArgs &a, const void *workspace);
infiniStatus_t launchTiles(const AttentionInfo &info, const TilesPlan &plan, const AttentionArgs &a, void *workspace, cudaStream_t stream);

// One CTA for each (sequence, q head), any layout (attention.cu).
infiniStatus_t launchRows(const AttentionInfo &info, const AttentionArgs &a, cudaStream_t stream);

} // namespace b200::quant_paged_cache

#endif
