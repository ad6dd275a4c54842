// infiniopQuantPagedCaching and infiniopQuantPagedCacheRead: rows of K and V into pools of 8- or 4-bit codes
// and back.
//
// Both kernels give a lane 16 neighbouring elements of a row (32 bytes of a 16-bit row in one access; 16 or 8 bytes of
// codes), a row a power of two of lanes, and let one lane move its elements of the K row and of the V row of kTokens
// tokens, so that all loads are in flight before the first is used.  Consecutive lanes take consecutive words, so every
// access of a warp covers whole rows.  A step's rows are a launch's latency; a prefill's are bound by HBM.
// Measured with 8 heads of 128, bf16: 64 rows at 8 bits 2.2 us to write and 2.2 to read; 16384 rows at 4 bits 17.7 us
// (4.9 TB/s) and 16.7 (5.1); 65536 rows at 4 bits read in 60.6 (5.7).
//
// Quantising without a division per element: with s the group's scale, code = x / s to the nearest, halves away from
// zero, is the nearest integer to x * r for r = (1 + 2^-21) / s to 1.5 ulp.  x has at most 11 significant bits and s 8, so
// x / s is either exactly k + 1/2 or at least 2^-16 (relative) away from it: with 2x = X 2^a and (2k + 1) s = Y 2^b,
// X < 2^11, Y < 2^16, the difference is a multiple of the smaller power.  x * r is above x / s in magnitude by a relative
// 2^-21 +- 2^-22, which moves an exact half up and carries nothing else across a half.  The sum fma(x, r, 1.5 * 2^23) then
// rounds once, to the nearest integer, and leaves it in the low bits of the float.
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

};

struct CachingArgs {
    Side k, v;
    const int64_t *slot_mapping;
    long long num_tokens;
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

constexpr int kElems = 16; // of a lane

// The first token, the kv head and the lane's place in a row; false behind the last pair.
template <int TOKENS>
__device__ __forceinline__ bool locate(const CachingArgs &a, long long &token, int &head, int &lane) {
    const long long thread = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
    const long long pair = thread >> a.lanes_log2; // (TOKENS tokens, kv head)
    lane = static_cast<int>(thread) & ((1 << a.lanes_log2) - 1);
    if (pair <= 0xffffffffLL) {
        const unsigned p = static_cast<unsigned>(pair);
        const unsigned t = p / static_cast<unsigned>(a.num_kv_heads);
        token = t;
        head = static_cast<int>(p - t * a.num_kv_heads);
    } else {
        token = pair / a.num_kv_heads;
        head = static_cast<int>(pair - token * a.num_kv_heads);
    }
    token *= TOKENS;
    return token < a.num_tokens;
}

// A token's slot, negative for padding; in checked mode one outside the pool raises a flag and counts as padding.
__device__ __forceinline__ long long slotOf(const CachingArgs &a, long long token, bool report) {
    long long slot = a.slot_mapping[token];
    if (a.check_indices && slot >= a.num_slots) {
        if (report) {
            atomicOr(a.kernel_flags, INFINIOP_KERNEL_FLAG_SLOT_OUT_OF_RANGE);
        }
        slot = -1;
    }
    return slot;
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

struct Words { // 32 bytes
    unsigned w[8];
};

__device__ __forceinline__ Words load32(const void *p) {
    Words x;
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(x.w[0]), "=r"(x.w[1]), "=r"(x.w[2]), "=r"(x.w[3]), "=r"(x.w[4]), "=r"(x.w[5]), "=r"(x.w[6]), "=r"(x.w[7])
                 : "l"(p));
    return x;
}

__device__ __forceinline__ void store32(void *p, const Words &x) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(x.w[0]), "r"(x.w[1]), "r"(x.w[2]), "r"(x.w[3]), "r"(x.w[4]),
                 "r"(x.w[5]), "r"(x.w[6]), "r"(x.w[7])
                 : "memory");
}

// 16 elements of 16 bits
template <bool VEC>
__device__ __forceinline__ Words loadRow(const unsigned short *p) {
    if constexpr (VEC) {
        return load32(p);
    } else {
        Words x;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x.w[i] = p[2 * i] | (static_cast<unsigned>(p[2 * i + 1]) << 16);
        }
        return x;
    }
}

// Largest magnitude among 16-bit values, as the bits of a magnitude (which order like the values, infinities and NaN last).
__device__ __forceinline__ unsigned largestOf(const Words &x) {
    const unsigned m = 0x7fff7fffu;
    unsigned a = x.w[0] & m;
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        a = __vmaxu2(a, x.w[i] & m);
    }
    return max(a & 0xffffu, a >> 16);
}

template <int BITS, typename T, bool VEC>
__device__ __forceinline__ void storeCodes(unsigned char *dst, const Words &x, float r, bool zero) {
    constexpr int kWords = BITS / 2, kPer = 32 / BITS; // 16 codes
    constexpr unsigned kOne = 1u << BITS;
    // a word is sum_i (code_i + half a field) * field^i, which has no borrows, and every field's top bit flipped; the codes come as
    // the bits of 1.5 * 2^23 + code
    constexpr unsigned kOnes = 0xffffffffu / (kOne - 1), kTops = kOnes << (BITS - 1);
    constexpr unsigned kAdd = kTops - 0x4b400000u * kOnes;
    unsigned out[kWords];
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
        unsigned word = 0;
#pragma unroll
        for (int i = kPer - 1; i >= 0; --i) {
            const int e = k * kPer + i;
            const unsigned half = e & 1 ? x.w[e / 2] >> 16 : x.w[e / 2] & 0xffffu;
            word = word * kOne + __float_as_uint(fmaf(bitsToFloat<T>(half), r, 12582912.f));
        }
        out[k] = zero ? 0u : (word + kAdd) ^ kTops;
    }
    if constexpr (VEC && BITS == 8) {
        *reinterpret_cast<uint4 *>(dst) = make_uint4(out[0], out[1], out[2], out[3]);
    } else if constexpr (VEC) {
        *reinterpret_cast<uint2 *>(dst) = make_uint2(out[0], out[1]);
    } else {
#pragma unroll
        for (int i = 0; i < 4 * kWords; ++i) {
            dst[i] = static_cast<unsigned char>(out[i / 4] >> (8 * (i % 4)));
        }
    }
}

// The scale of a group, and r.
template <int BITS, typename T>
__device__ __forceinline__ unsigned short scaleOf(unsigned largest, float &r, bool &zero) {
    constexpr unsigned kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    // A / Q to bf16.  A has at most 11 bits, so A / Q is a relative 2^-12 or more away from the middle of two neighbouring bf16, or on
    // it (Q = 7 and fp16 only); the residual makes a quotient that fits fp32 exact.
    constexpr float kQ = BITS == 8 ? 127.f : 7.f, kInverse = 1.f / kQ;
    const float largest_f = bitsToFloat<T>(largest), about = largest_f * kInverse;
    const float s = fmaf(fmaf(-about, kQ, largest_f), kInverse, about);
    unsigned short bits = __bfloat16_as_ushort(__float2bfloat16_rn(s));
    if (largest >= kInf) {
        bits = 0x7fffu; // NaN
    } else if (bits < 0x0080u) {
        bits = 0; // below 2^-126
    }
    zero = bits == 0 || largest >= kInf;
    float inverse; // to 1 ulp
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(__uint_as_float(static_cast<unsigned>(bits) << 16)));
    r = inverse * (1.f + 4.76837158203125e-7f); // not used where the codes are 0
    return bits;
}

// NV: vectors of 16 elements a lane has of a row (1 up to 512 elements, 2 up to 1024).  All lanes of a warp come here;
// `live`: whether this row is written.
template <int BITS, typename T, int NV, bool VEC>
__device__ __forceinline__ void writeRow(const Side &s, const Words (&x)[NV], bool live, long long block, int head, long long off, int lane, int lanes) {
    unsigned char *codes = static_cast<unsigned char *>(s.codes) + block * s.block + head * s.head + off * s.slot;
    unsigned short *scales = static_cast<unsigned short *>(s.scales) + block * s.s_block + head * s.s_head + off * s.s_slot;
    unsigned whole = 0;
    if constexpr (BITS == 8) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            whole = max(whole, largestOf(x[i])); // vectors beyond the row hold zeros
        }
        for (int o = 1; o < lanes; o <<= 1) {
            whole = max(whole, __shfl_xor_sync(0xffffffffu, whole, o));
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        unsigned m = whole;
        if constexpr (BITS == 4) {
            m = largestOf(x[i]);
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1)); // a group is two lanes
        }
        float r;
        bool zero;
        const unsigned short bits = scaleOf<BITS, T>(m, r, zero);
        const int vec = lane + i * lanes;
        if (live && kElems * vec < s.width) {
            storeCodes<BITS, T, VEC>(codes + vec * (2 * BITS), x[i], r, zero);
            if (BITS == 8 ? vec == 0 : (vec & 1) == 0) {
                scales[BITS == 8 ? 0 : vec >> 1] = bits;
            }
        }
    }
}

template <int BITS, typename T, int NV, bool VEC, int TOKENS>
__global__ void __launch_bounds__(kThreads) quantPagedCachingKernel(const CachingArgs a) {
    gridDependency();
    long long token0;
    int head, lane;
    const bool any = locate<TOKENS>(a, token0, head, lane);
    const int lanes = 1 << a.lanes_log2;
    long long slot[TOKENS];
    Words k[TOKENS][NV], v[TOKENS][NV];
#pragma unroll
    for (int u = 0; u < TOKENS; ++u) {
        const long long token = token0 + u;
        const bool here = any && token < a.num_tokens;
        slot[u] = here ? slotOf(a, token, lane == 0 && head == 0) : -1;
        const unsigned short *kr = static_cast<const unsigned short *>(a.k.rows) + token * a.k.r_token + head * a.k.r_head;
        const unsigned short *vr = static_cast<const unsigned short *>(a.v.rows) + token * a.v.r_token + head * a.v.r_head;
#pragma unroll
        for (int i = 0; i < NV; ++i) { // rows of padding too: the slot need not have come
            const int e = kElems * (lane + i * lanes);
            k[u][i] = v[u][i] = Words{};
            if (here && e < a.k.width) {
                k[u][i] = loadRow<VEC>(kr + e);
            }
            if (here && e < a.v.width) {
                v[u][i] = loadRow<VEC>(vr + e);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < TOKENS; ++u) {
        long long block = 0, off = 0;
        if (slot[u] >= 0) {
            splitSlot(a, slot[u], block, off);
        }
        writeRow<BITS, T, NV, VEC>(a.k, k[u], slot[u] >= 0, block, head, off, lane, lanes);
        writeRow<BITS, T, NV, VEC>(a.v, v[u], slot[u] >= 0, block, head, off, lane, lanes);
    }
}

// ---- reading back ------------------------------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ unsigned roundPair(float lo, float hi);
template <>
__device__ __forceinline__ unsigned roundPair<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned *>(&h);
}
template <>
__device__ __forceinline__ unsigned roundPair<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned *>(&h);
}

// 16 codes: two or four words.
template <int BITS, bool VEC>
__device__ __forceinline__ void loadCodes(unsigned (&w)[BITS / 2], const unsigned char *p) {
    if constexpr (VEC && BITS == 8) {
        const uint4 x = *reinterpret_cast<const uint4 *>(p);
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else if constexpr (VEC) {
        const uint2 x = *reinterpret_cast<const uint2 *>(p);
        w[0] = x.x, w[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < BITS / 2; ++i) {
            w[i] = p[4 * i] | (static_cast<unsigned>(p[4 * i + 1]) << 8) | (static_cast<unsigned>(p[4 * i + 2]) << 16)
                 | (static_cast<unsigned>(p[4 * i + 3]) << 24);
        }
    }
}

template <int BITS, typename T, bool VEC>
__device__ __forceinline__ void storeValues(T *dst, const unsigned (&codes)[BITS / 2], float s) {
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        constexpr int kPer = 32 / BITS;
        const int c = static_cast<int>(codes[e / kPer] << (32 - BITS - BITS * (e % kPer))) >> (32 - BITS);
        v[e] = static_cast<float>(c) * s; // at most 15 bits: rounded once, below
    }
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            Words x;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x.w[i] = __float_as_uint(v[8 * h + i]);
            }
            if constexpr (VEC) {
                store32(dst + 8 * h, x);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    dst[8 * h + i] = v[8 * h + i];
                }
            }
        }
    } else {
        Words x;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x.w[i] = roundPair<T>(v[2 * i], v[2 * i + 1]);
        }
        if constexpr (VEC) {
            store32(dst, x);
        } else {
            unsigned short *p = reinterpret_cast<unsigned short *>(dst);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                p[i] = static_cast<unsigned short>(x.w[i / 2] >> (16 * (i & 1)));
            }
        }
    }
}

template <int BITS, typename T, int NV, bool VEC, int TOKENS>
__global__ void __launch_bounds__(kThreads) quantPagedCacheReadKernel(const CachingArgs a) {
    gridDependency();
    long long token0;
    int head, lane;
    if (!locate<TOKENS>(a, token0, head, lane)) {
        return;
    }
    const int lanes = 1 << a.lanes_log2;
    long long slot[TOKENS];
#pragma unroll
    for (int u = 0; u < TOKENS; ++u) {
        slot[u] = token0 + u < a.num_tokens ? slotOf(a, token0 + u, lane == 0 && head == 0) : -1;
    }
    const Side *const sides[2] = {&a.k, &a.v};
    unsigned codes[TOKENS][2][NV][BITS / 2];
    unsigned scale[TOKENS][2][NV];
#pragma unroll
    for (int u = 0; u < TOKENS; ++u) {
        long long block = 0, off = 0;
        if (slot[u] >= 0) {
            splitSlot(a, slot[u], block, off);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const Side &s = *sides[x];
            const unsigned char *c = static_cast<const unsigned char *>(s.codes) + block * s.block + head * s.head + off * s.slot;
            const unsigned short *f = static_cast<const unsigned short *>(s.scales) + block * s.s_block + head * s.s_head + off * s.s_slot;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int vec = lane + i * lanes;
#pragma unroll
                for (int k = 0; k < BITS / 2; ++k) {
                    codes[u][x][i][k] = 0;
                }
                scale[u][x][i] = 0;
                if (slot[u] >= 0 && kElems * vec < s.width) {
                    loadCodes<BITS, VEC>(codes[u][x][i], c + vec * (2 * BITS));
                    scale[u][x][i] = f[BITS == 8 ? 0 : vec >> 1];
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < TOKENS; ++u) {
        if (token0 + u >= a.num_tokens) {
            break;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const Side &s = *sides[x];
            T *rows = static_cast<T *>(s.rows) + (token0 + u) * s.r_token + head * s.r_head;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int vec = lane + i * lanes;
                if (kElems * vec < s.width) {
                    storeValues<BITS, T, VEC>(rows + kElems * vec, codes[u][x][i], bitsToFloat<__nv_bfloat16>(scale[u][x][i]));
                }
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

// Whether codes and rows of one side can be moved in whole vectors of 16 elements.
static bool vectors(const Side &s, int bits, size_t row_elem) {
    auto ok = [](long long stride, long long bytes, long long unit) { return (stride * bytes) % unit == 0; };
    const long long e = static_cast<long long>(row_elem);
    const int codes = 2 * bits;
    return alignedTo(s.codes, codes) && ok(s.block, 1, codes) && ok(s.head, 1, codes) && ok(s.slot, 1, codes)
        && alignedTo(s.rows, 32) && ok(s.r_token, e, 32) && ok(s.r_head, e, 32);
}

using Kernel = void (*)(CachingArgs);

// Several tokens a lane where there are enough to fill the machine and rows are one vector a lane.
constexpr int kTokens = 2;

template <int BITS, typename T, bool READ>
static Kernel pick(int nv, bool vec, bool many) {
    if constexpr (READ) {
        return nv > 1 ? (vec ? quantPagedCacheReadKernel<BITS, T, 2, true, 1> : quantPagedCacheReadKernel<BITS, T, 2, false, 1>)
             : !vec   ? quantPagedCacheReadKernel<BITS, T, 1, false, 1>
                      : (many ? quantPagedCacheReadKernel<BITS, T, 1, true, kTokens> : quantPagedCacheReadKernel<BITS, T, 1, true, 1>);
    } else {
        return nv > 1 ? (vec ? quantPagedCachingKernel<BITS, T, 2, true, 1> : quantPagedCachingKernel<BITS, T, 2, false, 1>)
             : !vec   ? quantPagedCachingKernel<BITS, T, 1, false, 1>
                      : (many ? quantPagedCachingKernel<BITS, T, 1, true, kTokens> : quantPagedCachingKernel<BITS, T, 1, true, 1>);
    }
}

template <int BITS>
static Kernel pick(infiniDtype_t dtype, bool read, int nv, bool vec, bool many) {
    if (dtype == INFINI_DTYPE_F32) { // reading only
        return pick<BITS, float, true>(nv, vec, many);
    }
    if (dtype == INFINI_DTYPE_F16) {
        return read ? pick<BITS, __half, true>(nv, vec, many) : pick<BITS, __half, false>(nv, vec, many);
    }
    return read ? pick<BITS, __nv_bfloat16, true>(nv, vec, many) : pick<BITS, __nv_bfloat16, false>(nv, vec, many);
}

static Side side(const Pool &p, void *codes, void *scales, void *rows, ptrdiff_t token, ptrdiff_t head) {
    return {codes,  scales, rows, p.block, p.kv_head, p.slot, p.s_block, p.s_head, p.s_slot, token, head, static_cast<int>(p.head)};
}

static infiniStatus_t launch(const CachingDescriptor &d, void *k_cache, void *v_cache, void *k_scales, void *v_scales, void *k, void *v,
                             const void *slots, cudaStream_t stream) {
    const Pools &P = d.pools;
    const bool read = d.base.kind == OpKind::QuantPagedCacheRead;
    CachingArgs a;
    a.k = side(P.k, k_cache, k_scales, k, d.k_token, d.k_head);
    a.v = side(P.v, v_cache, v_scales, v, d.v_token, d.v_head);
    a.slot_mapping = static_cast<const int64_t *>(slots);
    a.num_tokens = static_cast<long long>(d.num_tokens);
    a.num_kv_heads = static_cast<int>(P.num_kv_heads);
    a.block_size = static_cast<int>(P.block_size);
    a.kernel_flags = d.base.props->kernel_flags;
    a.num_slots = static_cast<long long>(P.num_blocks) * static_cast<long long>(P.block_size);
    // a pool without blocks, which may have no address, is checked always
    a.check_indices = ((d.check_indices || P.num_blocks == 0) && a.kernel_flags != nullptr) ? 1 : 0;

    const int widest = a.k.width > a.v.width ? a.k.width : a.v.width;
    a.lanes_log2 = 1; // a group of 32 elements is two lanes
    while (a.lanes_log2 < 5 && (kElems << a.lanes_log2) < widest) {
        ++a.lanes_log2;
    }
    const int nv = widest <= 32 * kElems ? 1 : 2;
    const size_t elem = dtypeSize(d.dtype);
    const bool vec = vectors(a.k, P.bits, elem) && vectors(a.v, P.bits, elem);
    const long long pairs = a.num_tokens * static_cast<long long>(P.num_kv_heads);
    const bool many = nv == 1 && vec && (pairs << a.lanes_log2) >= 2048ll * d.base.props->sm_count;
    const int tokens = many ? kTokens : 1;
    const long long threads = ((a.num_tokens + tokens - 1) / tokens * static_cast<long long>(P.num_kv_heads)) << a.lanes_log2;
    const long long blocks = (threads + kThreads - 1) / kThreads;
    B200_RETURN_IF(blocks > 0x7fffffffLL, INFINI_STATUS_BAD_TENSOR_SHAPE);

    const Kernel kernel = P.bits == 4 ? pick<4>(d.dtype, read, nv, vec, many) : pick<8>(d.dtype, read, nv, vec, many);
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
    B200_RETURN_IF(k == nullptr || v == nullptr || slots == nullptr, INFINI_STATUS_NULL_POINTER);
    B200_RETURN_IF(d->pools.num_blocks > 0 && (k_cache == nullptr || v_cache == nullptr || k_scales == nullptr || v_scales == nullptr),
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
