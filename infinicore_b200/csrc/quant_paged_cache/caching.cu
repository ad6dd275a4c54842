// infiniopQuantPagedCaching and infiniopQuantPagedCacheRead: rows of K and V into pools of 8- or 4-bit codes
// and back.
//
// Both kernels give a lane eight neighbouring elements of a row (16 bytes of a 16-bit row; 8 or 4 bytes of
// codes), a row a power of two of lanes, and let one lane move its eight elements of the K row and of the V
// row of one (token, kv head), so that both loads are in flight before the first is used.  Consecutive lanes
// take consecutive words, so every access of a warp covers whole rows.  A step's rows are a launch's latency;
// a prefill's are bound by HBM.
//
// Quantising without a division per element: with s the group's scale, code = x / s to the nearest, halves
// away from zero, is the nearest integer to x * r for r = (1 + 2^-21) / s rounded to fp32.  x has at most 11
// significant bits and s 8, so x / s is either exactly k + 1/2 or at least 2^-16 (relative) away from it: with
// 2x = X 2^a and (2k + 1) s = Y 2^b, X < 2^12, Y < 2^16, the difference is a multiple of the smaller power.
// x * r is above x / s in magnitude by a relative 2^-21 +- 2^-22, which moves an exact half up and carries
// nothing else across a half.  The sum fma(x, r, 1.5 * 2^23) then rounds once, to the nearest integer, and
// leaves it in the low bits of the float.
#include "quant_pool.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>
#include <type_traits>

namespace b200::quant_paged_cache {

struct CachingDescriptor {
    OpDescriptorBase base;
    Pools pools;
    infiniDtype_t dtype;
    size_t num_tokens;
    ptrdiff_t k_token, k_head, v_token, v_head; // of the dense rows, in elements
    bool use_pdl;
    bool check_indices;
};

struct Side { // K or V; strides of codes in bytes, of scales and rows in elements
    void *codes;
    void *scales;
    void *rows;
    long long block, head, slot;
    long long s_block, s_head, s_slot;
    long long r_token, r_head;
    int width;  // elements of a row
    int groups; // scales of a row
};

struct CachingArgs {
    Side k, v;
    const int64_t *slot_mapping;
    long long num_pairs; // tokens * kv heads
    int num_kv_heads;
    int block_size;
    int lanes_log2; // lanes of a row
    unsigned int *kernel_flags;
    long long num_slots;
    int check_indices;
};

constexpr int kThreads = 128;

__device__ __forceinline__ void gridDependency() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// The (token, kv head) of this thread's lanes, and the slot; false for nothing to do.
__device__ __forceinline__ bool locate(const CachingArgs &a, long long &token, int &head, int &lane, long long &slot) {
    const long long thread = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
    const long long pair = thread >> a.lanes_log2;
    lane = static_cast<int>(thread) & ((1 << a.lanes_log2) - 1);
    if (pair >= a.num_pairs) {
        return false;
    }
    if (pair <= 0xffffffffLL) {
        const unsigned p = static_cast<unsigned>(pair);
        const unsigned t = p / static_cast<unsigned>(a.num_kv_heads);
        token = t;
        head = static_cast<int>(p - t * a.num_kv_heads);
    } else {
        token = pair / a.num_kv_heads;
        head = static_cast<int>(pair - token * a.num_kv_heads);
    }
    slot = a.slot_mapping[token];
    if (a.check_indices && slot >= a.num_slots) {
        if (lane == 0 && head == 0) {
            atomicOr(a.kernel_flags, INFINIOP_KERNEL_FLAG_SLOT_OUT_OF_RANGE);
        }
        slot = -1;
    }
    return true;
}

__device__ __forceinline__ void splitSlot(const CachingArgs &a, long long slot, long long &block, long long &off) {
    if (slot <= 0x7fffffffLL) {
        const unsigned s = static_cast<unsigned>(slot), b = s / static_cast<unsigned>(a.block_size);
        block = b;
        off = s - b * static_cast<unsigned>(a.block_size);
    } else {
        block = slot / a.block_size;
        off = slot - block * a.block_size;
    }
}

template <typename T>
__device__ __forceinline__ float bitsToFloat(unsigned half);
template <>
__device__ __forceinline__ float bitsToFloat<__half>(unsigned h) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
}
template <>
__device__ __forceinline__ float bitsToFloat<__nv_bfloat16>(unsigned h) {
    return __uint_as_float(h << 16);
}

template <bool VEC>
__device__ __forceinline__ uint4 loadEight(const unsigned short *p) {
    if constexpr (VEC) {
        return *reinterpret_cast<const uint4 *>(p);
    } else {
        uint4 w;
        w.x = p[0] | (static_cast<unsigned>(p[1]) << 16);
        w.y = p[2] | (static_cast<unsigned>(p[3]) << 16);
        w.z = p[4] | (static_cast<unsigned>(p[5]) << 16);
        w.w = p[6] | (static_cast<unsigned>(p[7]) << 16);
        return w;
    }
}

// Largest magnitude among the 16-bit values of the lanes that share a scale, as the bits of a magnitude
// (which order like the values, infinities and NaN last).
__device__ __forceinline__ unsigned largestOf(const uint4 &w) {
    const unsigned m = 0x7fff7fffu;
    const unsigned a = __vmaxu2(__vmaxu2(w.x & m, w.y & m), __vmaxu2(w.z & m, w.w & m));
    return max(a & 0xffffu, a >> 16);
}

template <int BITS, typename T, bool VEC>
__device__ __forceinline__ void storeCodes(unsigned char *dst, const uint4 &w, float r, bool zero) {
    const unsigned in[4] = {w.x, w.y, w.z, w.w};
    unsigned c[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[2 * i] = __float_as_uint(fmaf(bitsToFloat<T>(in[i] & 0xffffu), r, 12582912.f));
        c[2 * i + 1] = __float_as_uint(fmaf(bitsToFloat<T>(in[i] >> 16), r, 12582912.f));
    }
    if constexpr (BITS == 8) {
        unsigned lo = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
        unsigned hi = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
        lo = zero ? 0u : lo;
        hi = zero ? 0u : hi;
        if constexpr (VEC) {
            *reinterpret_cast<uint2 *>(dst) = make_uint2(lo, hi);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                dst[i] = static_cast<unsigned char>(lo >> (8 * i));
                dst[4 + i] = static_cast<unsigned char>(hi >> (8 * i));
            }
        }
    } else {
        unsigned word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            word |= (c[i] & 15u) << (4 * i);
        }
        word = zero ? 0u : word;
        if constexpr (VEC) {
            *reinterpret_cast<unsigned *>(dst) = word;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                dst[i] = static_cast<unsigned char>(word >> (8 * i));
            }
        }
    }
}

// The scale of a group, and r.
template <int BITS, typename T>
__device__ __forceinline__ unsigned short scaleOf(unsigned largest, float &r, bool &zero) {
    constexpr unsigned kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    const float s = __fdiv_rn(bitsToFloat<T>(largest), BITS == 8 ? 127.f : 7.f);
    unsigned short bits = __bfloat16_as_ushort(__float2bfloat16_rn(s));
    if (largest >= kInf) {
        bits = 0x7fffu; // NaN
    } else if (bits < 0x0080u) {
        bits = 0; // below 2^-126
    }
    zero = bits == 0 || largest >= kInf;
    r = zero ? 0.f : __frcp_rn(__uint_as_float(static_cast<unsigned>(bits) << 16)) * (1.f + 4.76837158203125e-7f);
    return bits;
}

// NV: vectors of eight elements a lane has of a row (1 up to 256 elements, 4 up to 1024).
template <int BITS, typename T, int NV, bool VEC>
__device__ __forceinline__ void writeRow(const Side &s, const uint4 (&w)[NV], long long block, int head, long long off, int lane, int lanes,
                                         unsigned mask) {
    unsigned char *codes = static_cast<unsigned char *>(s.codes) + block * s.block + head * s.head + off * s.slot;
    unsigned short *scales = static_cast<unsigned short *>(s.scales) + block * s.s_block + head * s.s_head + off * s.s_slot;
    constexpr int kBytes = BITS; // codes of eight elements
    if constexpr (BITS == 8) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            m = max(m, largestOf(w[i])); // vectors beyond the row hold zeros
        }
        for (int o = 1; o < lanes; o <<= 1) {
            m = max(m, __shfl_xor_sync(mask, m, o));
        }
        float r;
        bool zero;
        const unsigned short bits = scaleOf<BITS, T>(m, r, zero);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = 8 * (lane + i * lanes);
            if (e < s.width) {
                storeCodes<BITS, T, VEC>(codes + (lane + i * lanes) * kBytes, w[i], r, zero);
            }
        }
        if (lane == 0) {
            scales[0] = bits;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            unsigned m = largestOf(w[i]);
            m = max(m, __shfl_xor_sync(mask, m, 1));
            m = max(m, __shfl_xor_sync(mask, m, 2));
            float r;
            bool zero;
            const unsigned short bits = scaleOf<BITS, T>(m, r, zero);
            const int vec = lane + i * lanes;
            if (8 * vec < s.width) {
                storeCodes<BITS, T, VEC>(codes + vec * kBytes, w[i], r, zero);
                if ((vec & 3) == 0) {
                    scales[vec >> 2] = bits;
                }
            }
        }
    }
}

template <int BITS, typename T, int NV, bool VEC>
__global__ void __launch_bounds__(kThreads) quantPagedCachingKernel(const CachingArgs a) {
    gridDependency();
    long long token, slot;
    int head, lane;
    const bool mine = locate(a, token, head, lane, slot) && slot >= 0;
    // whole rows leave together: the lanes of a row are neighbours in one warp and agree on `mine`
    const unsigned mask = __ballot_sync(0xffffffffu, mine);
    if (!mine) {
        return;
    }
    const int lanes = 1 << a.lanes_log2;
    const unsigned short *k = static_cast<const unsigned short *>(a.k.rows) + token * a.k.r_token + head * a.k.r_head;
    const unsigned short *v = static_cast<const unsigned short *>(a.v.rows) + token * a.v.r_token + head * a.v.r_head;
    uint4 kw[NV], vw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = 8 * (lane + i * lanes);
        kw[i] = e < a.k.width ? loadEight<VEC>(k + e) : make_uint4(0, 0, 0, 0);
        vw[i] = e < a.v.width ? loadEight<VEC>(v + e) : make_uint4(0, 0, 0, 0);
    }
    long long block, off;
    splitSlot(a, slot, block, off);
    writeRow<BITS, T, NV, VEC>(a.k, kw, block, head, off, lane, lanes, mask);
    writeRow<BITS, T, NV, VEC>(a.v, vw, block, head, off, lane, lanes, mask);
}

// ---- reading back ------------------------------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ T roundTo(float v);
template <>
__device__ __forceinline__ float roundTo<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half roundTo<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 roundTo<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight codes: one or two words.
template <int BITS, bool VEC>
__device__ __forceinline__ uint2 loadCodes(const unsigned char *p) {
    uint2 w = make_uint2(0, 0);
    if constexpr (BITS == 8) {
        if constexpr (VEC) {
            w = *reinterpret_cast<const uint2 *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w.x |= static_cast<unsigned>(p[i]) << (8 * i);
                w.y |= static_cast<unsigned>(p[4 + i]) << (8 * i);
            }
        }
    } else {
        if constexpr (VEC) {
            w.x = *reinterpret_cast<const unsigned *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w.x |= static_cast<unsigned>(p[i]) << (8 * i);
            }
        }
    }
    return w;
}

template <int BITS, typename T, bool VEC>
__device__ __forceinline__ void storeValues(T *dst, uint2 codes, float s) {
    T out[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        int c;
        if constexpr (BITS == 8) {
            c = static_cast<int>((i < 4 ? codes.x : codes.y) << (24 - 8 * (i & 3))) >> 24;
        } else {
            c = static_cast<int>(codes.x << (28 - 4 * i)) >> 28;
        }
        out[i] = roundTo<T>(static_cast<float>(c) * s); // the product has at most 15 bits: one rounding
    }
    if constexpr (VEC) {
        constexpr int kWords = 8 * sizeof(T) / 16;
        uint4 w[kWords];
        memcpy(w, out, sizeof(out));
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            reinterpret_cast<uint4 *>(dst)[i] = w[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            dst[i] = out[i];
        }
    }
}

template <int BITS, typename T, int NV, bool VEC>
__global__ void __launch_bounds__(kThreads) quantPagedCacheReadKernel(const CachingArgs a) {
    gridDependency();
    long long token, slot;
    int head, lane;
    if (!locate(a, token, head, lane, slot)) {
        return;
    }
    const int lanes = 1 << a.lanes_log2;
    long long block = 0, off = 0;
    if (slot >= 0) {
        splitSlot(a, slot, block, off);
    }
    const Side *const sides[2] = {&a.k, &a.v};
    uint2 codes[2][NV];
    float scale[2][NV];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const Side &s = *sides[x];
        const unsigned char *c = static_cast<const unsigned char *>(s.codes) + block * s.block + head * s.head + off * s.slot;
        const unsigned short *f = static_cast<const unsigned short *>(s.scales) + block * s.s_block + head * s.s_head + off * s.s_slot;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int vec = lane + i * lanes;
            codes[x][i] = make_uint2(0, 0);
            scale[x][i] = 0.f;
            if (slot >= 0 && 8 * vec < s.width) {
                codes[x][i] = loadCodes<BITS, VEC>(c + vec * BITS);
                scale[x][i] = bitsToFloat<__nv_bfloat16>(f[BITS == 8 ? 0 : vec >> 2]);
            }
        }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const Side &s = *sides[x];
        T *rows = static_cast<T *>(s.rows) + token * s.r_token + head * s.r_head;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int vec = lane + i * lanes;
            if (8 * vec < s.width) {
                storeValues<BITS, T, VEC>(rows + 8 * vec, codes[x][i], scale[x][i]);
            }
        }
    }
}

// ---- host --------------------------------------------------------------------------------------------------

static infiniStatus_t create(CachingDescriptor **out, b200::Handle *h, OpKind kind,
                             infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache,
                             infiniopTensorDescriptor_t k_scales, infiniopTensorDescriptor_t v_scales,
                             infiniopTensorDescriptor_t k, infiniopTensorDescriptor_t v, infiniopTensorDescriptor_t slots) {
    const bool read = kind == OpKind::QuantPagedCacheRead;
    B200_RETURN_IF(k->dtype != INFINI_DTYPE_F16 && k->dtype != INFINI_DTYPE_BF16 && !(read && k->dtype == INFINI_DTYPE_F32),
                   INFINI_STATUS_BAD_TENSOR_DTYPE);
    B200_RETURN_IF(v->dtype != k->dtype || slots->dtype != INFINI_DTYPE_I64, INFINI_STATUS_BAD_TENSOR_DTYPE);
    B200_RETURN_IF(k->ndim() != 3 || v->ndim() != 3 || slots->ndim() != 1, INFINI_STATUS_BAD_TENSOR_SHAPE);
    Pools pools;
    const infiniStatus_t st = describePools(pools, k_cache, v_cache, k_scales, v_scales);
    B200_RETURN_IF(st != INFINI_STATUS_SUCCESS, st);
    const size_t tokens = slots->dim(0);
    B200_RETURN_IF(tokens > 0x7fffffffu, INFINI_STATUS_BAD_TENSOR_SHAPE);
    B200_RETURN_IF(k->dim(0) != tokens || v->dim(0) != tokens || k->dim(1) != pools.num_kv_heads || v->dim(1) != pools.num_kv_heads
                       || k->dim(2) != pools.k.head || v->dim(2) != pools.v.head,
                   INFINI_STATUS_BAD_TENSOR_SHAPE);
    B200_RETURN_IF(k->stride(2) != 1 || v->stride(2) != 1 || (tokens > 1 && slots->stride(0) != 1), INFINI_STATUS_BAD_TENSOR_STRIDES);

    auto *d = new (std::nothrow) CachingDescriptor{
        {h->base.device, h->base.device_id, kind, h->props}, pools, k->dtype, tokens, k->stride(0), k->stride(1), v->stride(0), v->stride(1),
        !envIs("INFINIOP_PAGED_DECODE_PDL", '0'), envIs("INFINIOP_PAGED_CHECK_INDICES", '1')};
    B200_RETURN_IF(d == nullptr, INFINI_STATUS_INTERNAL_ERROR);
    *out = d;
    return INFINI_STATUS_SUCCESS;
}

// Whether codes, scales and rows of one side can be moved in whole vectors of eight elements.
static bool vectors(const Side &s, int bits, size_t row_elem) {
    auto ok = [](long long stride, long long bytes, long long unit) { return (stride * bytes) % unit == 0; };
    const long long e = static_cast<long long>(row_elem);
    return alignedTo(s.codes, bits) && ok(s.block, 1, bits) && ok(s.head, 1, bits) && ok(s.slot, 1, bits)
        && alignedTo(s.rows, 16) && ok(s.r_token, e, 16) && ok(s.r_head, e, 16);
}

using Kernel = void (*)(CachingArgs);

template <int BITS, typename T>
static Kernel pick(bool read, int nv, bool vec) {
    if (read) {
        return nv == 1 ? (vec ? quantPagedCacheReadKernel<BITS, T, 1, true> : quantPagedCacheReadKernel<BITS, T, 1, false>)
                       : (vec ? quantPagedCacheReadKernel<BITS, T, 4, true> : quantPagedCacheReadKernel<BITS, T, 4, false>);
    }
    if constexpr (!std::is_same<T, float>::value) {
        return nv == 1 ? (vec ? quantPagedCachingKernel<BITS, T, 1, true> : quantPagedCachingKernel<BITS, T, 1, false>)
                       : (vec ? quantPagedCachingKernel<BITS, T, 4, true> : quantPagedCachingKernel<BITS, T, 4, false>);
    } else {
        return nullptr;
    }
}

template <typename T>
static Kernel pick(bool read, int bits, int nv, bool vec) {
    return bits == 4 ? pick<4, T>(read, nv, vec) : pick<8, T>(read, nv, vec);
}

static Side side(const Pool &p, void *codes, void *scales, void *rows, ptrdiff_t token, ptrdiff_t head) {
    return {codes,  scales, rows, p.block, p.kv_head, p.slot, p.s_block, p.s_head, p.s_slot, token, head, static_cast<int>(p.head),
            static_cast<int>(p.groups)};
}

static infiniStatus_t launch(const CachingDescriptor &d, void *k_cache, void *v_cache, void *k_scales, void *v_scales, void *k, void *v,
                             const void *slots, cudaStream_t stream) {
    const Pools &P = d.pools;
    const bool read = d.base.kind == OpKind::QuantPagedCacheRead;
    CachingArgs a;
    a.k = side(P.k, k_cache, k_scales, k, d.k_token, d.k_head);
    a.v = side(P.v, v_cache, v_scales, v, d.v_token, d.v_head);
    a.slot_mapping = static_cast<const int64_t *>(slots);
    a.num_pairs = static_cast<long long>(d.num_tokens) * static_cast<long long>(P.num_kv_heads);
    a.num_kv_heads = static_cast<int>(P.num_kv_heads);
    a.block_size = static_cast<int>(P.block_size);
    a.kernel_flags = d.base.props->kernel_flags;
    a.num_slots = static_cast<long long>(P.num_blocks) * static_cast<long long>(P.block_size);
    a.check_indices = (d.check_indices && a.kernel_flags != nullptr) ? 1 : 0;

    const int widest = a.k.width > a.v.width ? a.k.width : a.v.width;
    a.lanes_log2 = 2; // a group of 32 elements is four lanes
    while (a.lanes_log2 < 5 && (8 << a.lanes_log2) < widest) {
        ++a.lanes_log2;
    }
    const int nv = widest <= 256 ? 1 : 4;
    const size_t elem = dtypeSize(d.dtype);
    const bool vec = vectors(a.k, P.bits, elem) && vectors(a.v, P.bits, elem);
    const long long blocks = ((a.num_pairs << a.lanes_log2) + kThreads - 1) / kThreads;
    B200_RETURN_IF(blocks > 0x7fffffffLL, INFINI_STATUS_BAD_TENSOR_SHAPE);

    const Kernel kernel = d.dtype == INFINI_DTYPE_F16    ? pick<__half>(read, P.bits, nv, vec)
                        : d.dtype == INFINI_DTYPE_BF16 ? pick<__nv_bfloat16>(read, P.bits, nv, vec)
                                                       : pick<float>(read, P.bits, nv, vec);
    cudaLaunchAttribute pdl;
    pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl.val.programmaticStreamSerializationAllowed = d.use_pdl ? 1 : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cfg.attrs = &pdl;
    cfg.numAttrs = 1;
    (void)cudaLaunchKernelEx(&cfg, kernel, a);
    return checkLaunch(read ? "quantPagedCacheReadKernel" : "quantPagedCachingKernel");
}

static infiniStatus_t execute(InfiniopDescriptor *desc, OpKind kind, void *k_cache, void *v_cache, void *k_scales, void *v_scales, void *k,
                              void *v, const void *slots, void *stream) {
    B200_RETURN_IF(desc == nullptr, INFINI_STATUS_NULL_POINTER);
    auto *d = reinterpret_cast<CachingDescriptor *>(desc);
    B200_RETURN_IF(d->base.kind != kind, INFINI_STATUS_BAD_PARAM);
    if (d->num_tokens == 0 || d->pools.num_kv_heads == 0) {
        return INFINI_STATUS_SUCCESS;
    }
    B200_RETURN_IF(k_cache == nullptr || v_cache == nullptr || k_scales == nullptr || v_scales == nullptr || k == nullptr || v == nullptr
                       || slots == nullptr,
                   INFINI_STATUS_NULL_POINTER);
    return launch(*d, k_cache, v_cache, k_scales, v_scales, k, v, slots, static_cast<cudaStream_t>(stream));
}

static infiniStatus_t createChecked(InfiniopDescriptor **desc_ptr, infiniopHandle_t handle, OpKind kind,
                                    infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache,
                                    infiniopTensorDescriptor_t k_scales, infiniopTensorDescriptor_t v_scales,
                                    infiniopTensorDescriptor_t k, infiniopTensorDescriptor_t v, infiniopTensorDescriptor_t slots) {
    B200_RETURN_IF(handle == nullptr || desc_ptr == nullptr, INFINI_STATUS_NULL_POINTER);
    B200_RETURN_IF(k_cache == nullptr || v_cache == nullptr || k_scales == nullptr || v_scales == nullptr || k == nullptr || v == nullptr
                       || slots == nullptr,
                   INFINI_STATUS_NULL_POINTER);
    B200_RETURN_IF(handle->device != INFINI_DEVICE_NVIDIA, INFINI_STATUS_DEVICE_TYPE_NOT_SUPPORTED);
    CachingDescriptor *d = nullptr;
    const infiniStatus_t st = create(&d, reinterpret_cast<b200::Handle *>(handle), kind, k_cache, v_cache, k_scales, v_scales, k, v, slots);
    B200_RETURN_IF(st != INFINI_STATUS_SUCCESS, st);
    *desc_ptr = reinterpret_cast<InfiniopDescriptor *>(d);
    return INFINI_STATUS_SUCCESS;
}

static infiniStatus_t destroy(InfiniopDescriptor *desc, OpKind kind) {
    B200_RETURN_IF(desc == nullptr, INFINI_STATUS_NULL_POINTER);
    auto *d = reinterpret_cast<CachingDescriptor *>(desc);
    B200_RETURN_IF(d->base.kind != kind, INFINI_STATUS_BAD_PARAM);
    delete d;
    return INFINI_STATUS_SUCCESS;
}

static infiniStatus_t noWorkspace(InfiniopDescriptor *desc, size_t *size) {
    B200_RETURN_IF(desc == nullptr || size == nullptr, INFINI_STATUS_NULL_POINTER);
    *size = 0;
    return INFINI_STATUS_SUCCESS;
}

} // namespace b200::quant_paged_cache

using b200::OpKind;
namespace qc = b200::quant_paged_cache;

__INFINI_C infiniStatus_t infiniopCreateQuantPagedCachingDescriptor(
    infiniopHandle_t handle,
    infiniopQuantPagedCachingDescriptor_t *desc_ptr,
    infiniopTensorDescriptor_t k_cache_desc,
    infiniopTensorDescriptor_t v_cache_desc,
    infiniopTensorDescriptor_t k_scales_desc,
    infiniopTensorDescriptor_t v_scales_desc,
    infiniopTensorDescriptor_t k_desc,
    infiniopTensorDescriptor_t v_desc,
    infiniopTensorDescriptor_t slot_mapping_desc) {
    return qc::createChecked(desc_ptr, handle, OpKind::QuantPagedCaching, k_cache_desc, v_cache_desc, k_scales_desc, v_scales_desc, k_desc,
                             v_desc, slot_mapping_desc);
}

__INFINI_C infiniStatus_t infiniopGetQuantPagedCachingWorkspaceSize(
    infiniopQuantPagedCachingDescriptor_t desc, size_t *size) {
    return qc::noWorkspace(desc, size);
}

__INFINI_C infiniStatus_t infiniopQuantPagedCaching(
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
    void *stream) {
    (void)workspace;
    (void)workspace_size;
    return qc::execute(desc, OpKind::QuantPagedCaching, k_cache, v_cache, k_scales, v_scales, const_cast<void *>(k), const_cast<void *>(v),
                       slot_mapping, stream);
}

__INFINI_C infiniStatus_t infiniopDestroyQuantPagedCachingDescriptor(
    infiniopQuantPagedCachingDescriptor_t desc) {
    return qc::destroy(desc, OpKind::QuantPagedCaching);
}

__INFINI_C infiniStatus_t infiniopCreateQuantPagedCacheReadDescriptor(
    infiniopHandle_t handle,
    infiniopQuantPagedCacheReadDescriptor_t *desc_ptr,
    infiniopTensorDescriptor_t k_desc,
    infiniopTensorDescriptor_t v_desc,
    infiniopTensorDescriptor_t k_cache_desc,
    infiniopTensorDescriptor_t v_cache_desc,
    infiniopTensorDescriptor_t k_scales_desc,
    infiniopTensorDescriptor_t v_scales_desc,
    infiniopTensorDescriptor_t slot_mapping_desc) {
    return qc::createChecked(desc_ptr, handle, OpKind::QuantPagedCacheRead, k_cache_desc, v_cache_desc, k_scales_desc, v_scales_desc, k_desc,
                             v_desc, slot_mapping_desc);
}

__INFINI_C infiniStatus_t infiniopGetQuantPagedCacheReadWorkspaceSize(
    infiniopQuantPagedCacheReadDescriptor_t desc, size_t *size) {
    return qc::noWorkspace(desc, size);
}

__INFINI_C infiniStatus_t infiniopQuantPagedCacheRead(
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
    void *stream) {
    (void)workspace;
    (void)workspace_size;
    return qc::execute(desc, OpKind::QuantPagedCacheRead, const_cast<void *>(k_cache), const_cast<void *>(v_cache),
                       const_cast<void *>(k_scales), const_cast<void *>(v_scales), k, v, slot_mapping, stream);
}

__INFINI_C infiniStatus_t infiniopDestroyQuantPagedCacheReadDescriptor(
    infiniopQuantPagedCacheReadDescriptor_t desc) {
    return qc::destroy(desc, OpKind::QuantPagedCacheRead);
}
