// The fast kernel of infiniopQuantPagedAttention: tiles of 16 to 64 tokens, matrix instructions on the codes.
//
// Work.  A unit is (sequence, kv head, tile of 8 or 16 q heads of its group), as many token tiles long as cover the sequence.
// All units lie end to end in one line, each with unitCost() tiles in front for what a unit costs by itself (q, results),
// and the line is cut into equal ranges, one for each warp of a persistent grid, so that ragged batches, many short and
// few long sequences load the machine alike.  A warp that has a unit to itself stores its rows; pieces of a unit in one
// CTA meet in shared memory at the CTA's end; a unit that is cut between CTAs leaves partial results (maximum, sum,
// unnormalised output) in the workspace, and the combine kernel adds those in the order of the line.  Every sum has
// one order, so the same call gives the same bits.
//
// Loads.  Every warp has a ring of tiles of its own in shared memory, filled by 16-byte asynchronous copies several
// tiles ahead and across the ends of units.  Rows are swizzled in 16-byte chunks so that the matrix loads
// (ldmatrix) touch every bank once.
//
// Arithmetic.  Codes become fp16 exactly by bit operations (1024 + u has u in its low mantissa bits) and one
// addition; the scales never touch them:
//   S[token, head] = sum_g k_scale[token, g] * (codes . Q)_g    a 32-element group is two matrix instructions
//   w[token, g]    = p[token] * v_scale[token, g]               the weights carry the V scales
//   O[dim, head]   = sum_token codes[token, dim] * w[token, g]
// The codes are the first operand both times (all 16 of its rows are used whatever the number of heads): K by rows, V
// through a transposing load.  The weights are transposed in registers, 8 tokens by 8 heads at a time.  In the 4-bit form
// every second element of V keeps a factor of 16 that its output is rid of at the end.
//   q is held in fp16 times a power of two that makes its largest element 1/2..1: exact for every element above
// 2^-13 of that (fp16 and bf16 both have at most 11 bits).
//   w is rounded to fp16 (once, or as two halves: see Split), as w = p * v_scale * 2^k with an exponent k of its own for each head and group of V, so that every group of
// an output has weights of full precision, whatever the sizes of the others.  k is settled at a unit's first tile: it makes the group's
// largest weight 2^7..2^8.  It is settled again, from the same tile's scores once more, when a weight passes what fp16 holds; earlier
// outputs are scaled then, by powers of two.  Where the k of a head's groups are within 2^6 of each other, as they are unless V's channels differ
// in size by far more than that, the smallest serves them all, inside the maximum: w = p * v_scale ("even").
//   Sums, maxima and outputs are fp32.
//
// Measured at 32/8 heads of 128, 64 x 4096 tokens, bf16, the combine kernel's share of 3.5 to 4.6 us included: 8 bits 98 us in a graph of
// ten calls (5.6 TB/s of codes and scales), 100 to 112 over thousands in a row; 4 bits 78 us (3.9 TB/s).  At 4 bits nothing is full (issue slots 63 %,
// ALU 49 %, HBM 46 %): warps wait for their own last instruction, 2.8 to a scheduler.  About 15 us are there at any length: 64 sequences
// of 256, 1024, 4096 tokens on the line take 18.7, 31.1, 78.0 us at 4 bits, 21.3, 36.6, 97.6 at 8.
#include "attention.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b200::quant_paged_cache {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
// What a unit costs beside its tiles, in tiles: the time of 64 tokens.  Measured at 40 ragged sequences (64/8 heads of 128, 4 bits): 0
// tokens 67.5 us, 32 44.5, 64 40.7, 128 40.4; at 62 sequences of 200 to 2000 with their append 31.9, 31.4, 29.5, 30.5.
constexpr int unitCost(int tile) { return 64 / tile; }
// Of a warp: at least two tiles of a unit's first range.  More leaves fewer pieces to combine but warps idle: 6, 12, 24 instead of 2 take
// 13 sequences of 1 to 30001 (16/1 heads of 256, 8 bits) from 26.3 us to 28.8, 31.0, 40.7, the 62 sequences from 29.5 to 29.5, 38.6, 46.4.
constexpr int minRange(int tile) { return unitCost(tile) + 2; }
// What the weights are relative to is settled at a unit's first tile and again when a weight does not fit fp16 (or p comes to kMostP).
// p = exp2(score - top), in the log2 domain: top is then kBelow above the largest score so far.
constexpr float kBelow = 16.f;
constexpr float kMostP = 1.2379400392853803e27f; // 2^90
constexpr float kMostFactor = 126.f; // exponent of a group's factor at most (its reciprocal is a normal number), and at first
constexpr float kLargest = 7.f;      // exponent of a group's largest weight when its factor is set: 2^8 below what fp16 holds
constexpr float kEven = 6.f;         // factors of a head's groups whose exponents are this near count as one: the largest weight of each group
                                     // is 2 or more then, and what is subnormal in fp16 is off by 2^-26 of it at most
constexpr float kLeastCommon = -20.f, kMostCommon = 80.f; // exponents that such a one may have: p times it stays far inside fp32

// One rounding of the weights to fp16 is not seen in bf16 outputs, which are rounded to 8 bits (error against 64 bits 1.66e-3 instead of
// 1.65e-3), but is in fp16 ones (2.9e-4 instead of 2.1e-4, and its whole 2^-11 where a sequence has one token).  There weights are split
// in two: p' * v_scale with the three leading bits of p, which is exact, and the rest.  kColumns: with groups of up to 4 q heads the rests
// take the other half of an instruction's 8 columns, whose q are the same heads again.  kTwice: a second product.  Measured at 64 x 4096
// tokens, 32/8 heads of 128 (us, whole | columns | twice): 4 bits 77.9 | 79.5 | 93.4, 8 bits 97.8 | 98.6 | 106.7; 64/4 heads of 128 (whole | twice):
// 69.7 | 84.7, 72.0 | 82.0.
enum Split : int { kWhole = 0, kColumns = 1, kTwice = 2 };

// What the combine kernel has to do for a unit: nothing, or to add this many pieces from this CTA's on.
struct Task {
    int seq, sub, pieces, cta;
};

// A part of a unit that one warp has done: first tile's position on the line, tiles of the whole unit.
struct Piece {
    long long first;
    int seq, sub, tiles, used;
};

constexpr int kWalkBytes = 20;

template <int BITS, int HD, int HT>
struct Cfg {
    static constexpr int kRowBytes = HD * BITS / 8;
    static constexpr int kChunks = kRowBytes / 16;            // 16-byte chunks of a row
    static constexpr int kGroups = BITS == 4 ? HD / 32 : 1;   // scales of a row
    // A tile is one, two or four times 16 tokens, about 4 KB of codes: what surrounds the matrix instructions costs as many issue slots
    // as 8 tokens' arithmetic.  Measured at 64 x 4096 tokens, 32/8 heads (us): 4 bits, heads of 128, 16 tokens 88.5, 32 77.8; heads of 64,
    // 32 tokens 54.2, 64 50.4; 8 bits, heads of 64, 16 tokens 66.0, 32 57.3.  With 16 heads the weights of 64 tokens do not fit the registers
    // (64/4 heads of 64 at 4 bits: 32 tokens 44.8, 64 50.1).
    static constexpr int kSubs = HD * BITS <= 256 && HT == 8 ? 4 : HD * BITS <= 512 ? 2 : 1;
    static constexpr int kTile = 16 * kSubs;
    static constexpr int kStage = 2 * kTile * kRowBytes + 2 * kTile * kGroups * 2;
    static constexpr int kHeadTiles = HT / 8;
    static constexpr int kStride = HD + 4;                    // floats: rows of two heads apart hit other banks
    static constexpr int kResult = HT * kStride * 4;
    static constexpr int kFactors = HT * (kGroups + 1) * 4; // bytes of a warp
    static constexpr int kFixed = kWarps * (kResult + 2 * HT * 8 + kFactors + 2 * static_cast<int>(sizeof(Piece)) + 2 * kWalkBytes);
    // resident CTAs: what the registers of q, outputs and scales leave room for; 8 bits at heads of 128, heads of 192, 16 q heads and two products
    // spill 4 to 170 bytes
    static constexpr int kCtas = HD * HT <= 1024 ? (BITS == 4 || HT == 16 ? 3 : 4) : HD * HT <= 1536 ? 3 : 2;
    static constexpr int kFit = (227 * 1024 / kCtas - 1024 - kFixed) / (kWarps * kStage);
    static constexpr int kStages = kFit > 4 ? 4 : kFit;
    static_assert(kStages >= 2, "a ring of two tiles at least");
    static constexpr int kRing = kStages * kStage;
    static_assert(kRing >= kResult, "a finished ring holds a result");
    static constexpr int kSmem = kWarps * kRing + kFixed;
    static constexpr int kRecord = HT * HD + 2 * HT; // floats of a partial result: outputs, maxima, sums
};

// ---- instructions ------------------------------------------------------------------------------------------

__device__ __forceinline__ unsigned smemAddr(const void *p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void copy16(unsigned dst, const void *src, unsigned long long policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
// Codes and scales are read once: they leave the L2 first, tables, q and partial results stay.  Measured with | without (us): 64 x 4096
// tokens at 8 bits 97.7 | 100.5, 62 sequences of 200 to 2000 at 4 bits with their append 29.5 | 31.0.
__device__ __forceinline__ unsigned long long readOnce() {
    unsigned long long p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void commitCopies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void waitCopies() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void loadMatrices(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void loadMatricesTransposed(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same onto zeros
__device__ __forceinline__ void mmaFirst(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ unsigned transposed(unsigned x) {
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ float exp2Fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ unsigned packHalves(float lo, float hi) {
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// (x & mask) ^ magic
template <unsigned MASK>
__device__ __forceinline__ unsigned pick(unsigned x, unsigned magic) {
    unsigned r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(x), "n"(MASK), "r"(magic));
    return r;
}
// A constant that stays in a register: an instruction takes one immediate, and a second one costs a move each time.
__device__ __forceinline__ unsigned pinned(unsigned c) {
    unsigned r;
    asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(c));
    return r;
}
__device__ __forceinline__ unsigned addHalves(unsigned x, unsigned y) {
    unsigned r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    return r;
}
__device__ __forceinline__ unsigned fmaHalves(unsigned x, unsigned y, unsigned z) {
    unsigned r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(y), "r"(z));
    return r;
}

constexpr unsigned kMinus1032 = 0xe408e408u; // fp16 pairs
constexpr unsigned kMinus1152 = 0xe480e480u;
constexpr unsigned kMinus72 = 0xd480d480u;

struct Magic { // fp16 pairs and bytes
    unsigned low = pinned(0x64086408u);       // 1024 + 8
    unsigned high = pinned(0x64806480u);      // 1024 + 128
    unsigned sixteenth = pinned(0x2c002c00u);
    unsigned byte = pinned(0x64646464u);
};

// 4-bit: a word of eight codes -> pairs (0,4), (1,5), (2,6), (3,7)
__device__ __forceinline__ void codes4(const Magic &m, unsigned w, unsigned (&b)[4]) {
    const unsigned h = w >> 8;
    b[0] = addHalves(pick<0x000f000fu>(w, m.low), kMinus1032);                 // 1024 + (c + 8) - 1032
    b[1] = fmaHalves(pick<0x00f000f0u>(w, m.high), m.sixteenth, kMinus72);     // (1024 + 16 (c + 8)) / 16 - 72
    b[2] = addHalves(pick<0x000f000fu>(h, m.low), kMinus1032);
    b[3] = fmaHalves(pick<0x00f000f0u>(h, m.high), m.sixteenth, kMinus72);
}
// The same with the odd ones 16 times too large
__device__ __forceinline__ void codes4Odd16(const Magic &m, unsigned w, unsigned (&b)[4]) {
    const unsigned h = w >> 8;
    b[0] = addHalves(pick<0x000f000fu>(w, m.low), kMinus1032);
    b[1] = addHalves(pick<0x00f000f0u>(w, m.high), kMinus1152);
    b[2] = addHalves(pick<0x000f000fu>(h, m.low), kMinus1032);
    b[3] = addHalves(pick<0x00f000f0u>(h, m.high), kMinus1152);
}
// 8-bit: two of a word's codes, by byte selector
template <unsigned SEL>
__device__ __forceinline__ unsigned codes8(const Magic &m, unsigned flipped) {
    return addHalves(__byte_perm(flipped, m.byte, SEL), kMinus1152);
}

// 2^e for a whole number e, -126 to 127
__device__ __forceinline__ float powerOfTwo(float e) { return __uint_as_float(static_cast<unsigned>(static_cast<int>(e) + 127) << 23); }
// x * 2^e for a whole number e up to 126, however low
__device__ __forceinline__ float shifted(float x, float e) {
    const float a = fmaxf(e, -126.f), b = fmaxf(e - a, -126.f);
    return x * powerOfTwo(a) * powerOfTwo(b);
}
// The three leading bits of p
__device__ __forceinline__ float leading(float p) { return __uint_as_float(__float_as_uint(p) & 0xffe00000u); }
// The exponent of x >= 0; -127 of 0 and of subnormal numbers
__device__ __forceinline__ float exponentOf(float x) { return static_cast<float>(static_cast<int>(__float_as_uint(x) >> 23) - 127); }
// The largest among the eight lanes of a head
__device__ __forceinline__ float largestOf(float m) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
    return fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
}

// Columns x of a lane's outputs, those of a group's elements, times 2^e
template <int BITS, int HD>
__device__ __forceinline__ void scaleGroup(float (&o)[HD / 16][4], int group, int x, float e) {
    const float by = e >= -126.f ? powerOfTwo(e) : 0.f;
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) {
        if (BITS == 8 || j / 2 == group) {
            o[j][x] *= by;
            o[j][2 + x] *= by;
        }
    }
}

// ---- the line of tiles -------------------------------------------------------------------------------------

struct TilesArgs {
    unsigned char *workspace; // Task[] | records
    long long tasks_bytes;
    int unit_of_cta;          // every CTA has one unit to itself: nothing to combine
    int task_of_unit;         // tasks are numbered by unit, where there are no more units than CTAs; otherwise by CTA
    int combine_heads;        // of a CTA of the combine kernel
    int subs;                 // kv heads * head tiles of a group
    int head_tiles;
    unsigned halves;          // block_size / 8
    unsigned half_magic;      // division by that
    unsigned half_self;       // all ones where that is a division by 1
    int half_shift;
    int index_shift;          // log2 of the bytes of a table entry
    int out_words;            // rows of out can be stored 8 bytes at a time
};

// planTiles takes no table that names more than kMostTokensInt
__device__ __forceinline__ int lengthOf(const AttentionArgs &a, int seq) { return static_cast<int>(tokensOf(a, seq)); }

template <int TILE>
__device__ __forceinline__ int tilesOf(int len) {
    return len > 0 ? (len + TILE - 1) / TILE : 0;
}
template <int TILE>
__device__ __forceinline__ long long costOf(int len) {
    return len > 0 ? tilesOf<TILE>(len) + unitCost(TILE) : 0;
}

// Where a walk over a warp's range is: the unit, how much of the range lies behind what it takes of that unit.  Kept in
// shared memory, read and written by all lanes alike: the loop over a unit's tiles has no use for it.
struct Walk {
    int seq, sub, tiles, len, budget;

    // To the next unit: how many of its tiles are in the range (0: the range has ended).
    template <int TILE>
    __device__ __forceinline__ int step(const AttentionArgs &a, int subs) {
        budget -= unitCost(TILE); // at or below 0: the range ends in front of the unit's first tile
        if (budget <= 0) {
            return 0;
        }
        if (++sub == subs) {
            sub = 0;
            do {
                len = lengthOf(a, ++seq);
            } while (len <= 0);
            tiles = tilesOf<TILE>(len);
        }
        const int n = min(tiles, budget);
        budget -= n;
        return n;
    }
};

static_assert(sizeof(Walk) == kWalkBytes);

// ---- kernel ------------------------------------------------------------------------------------------------

__device__ __forceinline__ unsigned short roundOut(float v, int is_bf16) {
    return is_bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// N neighbouring elements of a row of out.
template <int N>
__device__ __forceinline__ void storeOut(const AttentionArgs &a, const TilesArgs &p, long long at, const float (&v)[N]) {
    unsigned short *dst = static_cast<unsigned short *>(a.out) + at;
    unsigned short r[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        r[i] = roundOut(v[i], a.is_bf16);
    }
    if (p.out_words) {
        if constexpr (N == 4) {
            *reinterpret_cast<uint2 *>(dst) = make_uint2(r[0] | (static_cast<unsigned>(r[1]) << 16), r[2] | (static_cast<unsigned>(r[3]) << 16));
        } else {
            *reinterpret_cast<unsigned *>(dst) = r[0] | (static_cast<unsigned>(r[1]) << 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            dst[i] = r[i];
        }
    }
}

// DENSE: blocks are multiples of 16 tokens and the rows of a head follow one another in a block, so 16 tokens are one run of
// memory; otherwise blocks are multiples of 8 tokens, rows lie anywhere, and 8 tokens' scales are one run.
// SPLIT: of the weights.
template <int BITS, int HD, int HT, bool DENSE, Split SPLIT>
__global__ void __launch_bounds__(kThreads, (Cfg<BITS, HD, HT>::kCtas)) quantAttentionTilesKernel(const AttentionArgs a, const TilesArgs p) {
    using C = Cfg<BITS, HD, HT>;
    constexpr int NG = C::kGroups, NH = C::kHeadTiles, CPR = C::kChunks, S = C::kStages, TILE = C::kTile, SUBS = C::kSubs;
    extern __shared__ __align__(128) unsigned char smem[];
    float *results = reinterpret_cast<float *>(smem + kWarps * C::kRing);                                     // [warp][head][kStride]
    float2 *sums = reinterpret_cast<float2 *>(reinterpret_cast<unsigned char *>(results) + kWarps * C::kResult); // [warp][2][head]
    float *all_factors = reinterpret_cast<float *>(sums + kWarps * 2 * HT);                                   // [warp][group | least][head]
    Piece *pieces = reinterpret_cast<Piece *>(all_factors + kWarps * (C::kFactors / 4));                                // [warp][2]
    Walk *walks = reinterpret_cast<Walk *>(pieces + kWarps * 2);                                              // [warp][copies | arithmetic]
    const int tid = static_cast<int>(pinned(threadIdx.x)), warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t = lane & 3;

    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (lane < 2) {
        pieces[2 * warp + lane].used = 0;
    }
    // this warp's range
    Task *tasks = reinterpret_cast<Task *>(p.workspace);
    long long total, range; // of the line; of a warp
    long long cta_start;
    Walk first_walk = {};   // unit of the range's start; its position there in `budget`
    if (p.unit_of_cta) {
        // the line is one unit, and a warp's range a fourth of its tiles
        first_walk.seq = static_cast<int>(blockIdx.x) / p.subs;
        first_walk.sub = static_cast<int>(blockIdx.x) - first_walk.seq * p.subs;
        first_walk.len = lengthOf(a, first_walk.seq);
        total = costOf<TILE>(first_walk.len);
        if (total == 0) {
            return;
        }
        range = (tilesOf<TILE>(first_walk.len) + kWarps - 1) / kWarps;
        cta_start = unitCost(TILE);
        first_walk.budget = static_cast<int>(cta_start + range * warp);
    } else {
        // every warp adds up the batch for itself: lane i has sequences i * per to (i + 1) * per - 1
        const int per = (a.num_seqs + 31) / 32;
        long long mine = 0;
#pragma unroll 4
        for (int i = 0; i < per; ++i) {
            const int s = lane * per + i;
            mine += s < a.num_seqs ? costOf<TILE>(lengthOf(a, s)) : 0;
        }
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, upto, o);
            upto += lane >= o ? x : 0;
        }
        total = __shfl_sync(0xffffffffu, upto, 31) * p.subs;
        const int workers = static_cast<int>(gridDim.x) * kWarps;
        range = (total + workers - 1) / workers;
        range = range > minRange(TILE) ? range : minRange(TILE);
        cta_start = range * kWarps * blockIdx.x;
        if (cta_start >= total) {
            if (tid == 0 && !p.task_of_unit) {
                tasks[blockIdx.x].pieces = 0;
            }
            return;
        }
        long long pos = cta_start + range * warp - (upto - mine) * p.subs; // within this lane's sequences, if not negative and before
        const bool here = pos >= 0 && pos < mine * p.subs;                 // their end, which is so for one lane at most
        int s = lane * per;
        if (here) {
            long long cost = costOf<TILE>(lengthOf(a, s)) * p.subs;
            while (pos >= cost) {
                pos -= cost;
                cost = costOf<TILE>(lengthOf(a, ++s)) * p.subs;
            }
        }
        const unsigned who = __ballot_sync(0xffffffffu, here);
        if (who != 0) {
            const int from = __ffs(who) - 1;
            first_walk.seq = __shfl_sync(0xffffffffu, s, from);
            pos = __shfl_sync(0xffffffffu, pos, from);
            first_walk.len = lengthOf(a, first_walk.seq);
            const long long cost = costOf<TILE>(first_walk.len);
            first_walk.sub = static_cast<int>(pos / cost);
            first_walk.budget = static_cast<int>(pos - first_walk.sub * cost);
        }
    }
    const long long cta_range = range * kWarps;
    const long long start = cta_start + warp * range, end = start + range < total ? start + range : total;

    unsigned char *ring = smem + warp * C::kRing;
    if (start < total) {
        const Magic magic;
        const unsigned long long policy = readOnce();
        Walk &copies = walks[2 * warp], &work = walks[2 * warp + 1];
        int tile, left;  // of the unit in work: present tile, tiles from there on in the range
        long long place; // of the present tile on the line
        {
            Walk w = first_walk;
            w.tiles = tilesOf<TILE>(w.len);
            const int in = w.budget - unitCost(TILE); // below 0: in front of the unit's first tile
            tile = in > 0 ? in : 0;
            place = start + (tile - in);
            const int budget = static_cast<int>(end - place);
            left = min(w.tiles - tile, budget);
            w.budget = budget - left;
            copies = work = w;
            __syncwarp();
        }

        // ---- copies: the next tile's block is already looked up
        unsigned f_half = TILE / 8 * static_cast<unsigned>(tile); // first half (8 tokens) of the next tile, within its unit
        int f_left = left;
        const unsigned char *table_row = nullptr;
        // this lane's first 16 bytes of codes (where runs are dense; otherwise the kv head's first) and of scales in block 0
        const unsigned char *k_lane = nullptr, *v_lane = nullptr, *s_lane = nullptr;
        constexpr int kRuns = DENSE ? SUBS : 2 * SUBS; // runs of 16 or 8 tokens, each in one block
        unsigned block[kRuns] = {}, first_slot[kRuns] = {}; // of the next tile's runs: the block, the first slot there
        const unsigned code_block = static_cast<unsigned>(a.k_block), code_slot = static_cast<unsigned>(a.k_slot);
        const unsigned scale_block = 2u * static_cast<unsigned>(a.ks_block);
        auto unit = [&]() {
            const int kv = copies.sub / p.head_tiles;
            table_row = static_cast<const unsigned char *>(a.block_tables) + ((copies.seq * a.table_seq) << p.index_shift);
            const long long codes = kv * a.k_head + (DENSE ? lane * 16 : 0);
            k_lane = a.k_codes + codes;
            v_lane = a.v_codes + codes;
            const bool v = lane >= TILE / 8 * NG;
            const int chunk = lane % NG + (DENSE ? (lane / NG & 1) * NG : 0);
            s_lane = reinterpret_cast<const unsigned char *>((v ? a.v_scales : a.k_scales) + kv * a.ks_head) + chunk * 16;
        };
        auto entry = [&](unsigned page) { // the low word of a 64-bit entry says all that a block in the pool can be
            const unsigned char *at = table_row + (static_cast<unsigned long long>(page) << p.index_shift);
            unsigned b = *reinterpret_cast<const unsigned *>(at);
            if (a.check_indices) {
                const long long whole = p.index_shift == 3 ? *reinterpret_cast<const long long *>(at) : static_cast<long long>(static_cast<int>(b));
                if (static_cast<unsigned long long>(whole) >= static_cast<unsigned long long>(a.num_blocks)) {
                    atomicOr(a.kernel_flags, INFINIOP_KERNEL_FLAG_BLOCK_OUT_OF_RANGE);
                    b = 0;
                }
            }
            return b;
        };
        auto look = [&]() {
            const unsigned page = (__umulhi(f_half, p.half_magic) + (f_half & p.half_self)) >> p.half_shift;
            first_slot[0] = 8u * (f_half - page * p.halves);
            unsigned at = page;
            block[0] = entry(at);
#pragma unroll
            for (int r = 1; r < kRuns; ++r) {
                // a run behind the sequence's end, whose table entry may say anything, is read where the one before is; entries are
                // only loaded here (the same one twice, if it must be): the next fetch is the first to wait for them
                constexpr unsigned kTokens = DENSE ? 16u : 8u;
                const unsigned slot = first_slot[r - 1] + kTokens;
                const bool live = 8 * static_cast<int>(f_half) + r * static_cast<int>(kTokens) < copies.len;
                const bool turn = slot >= static_cast<unsigned>(a.block_size);
                at += live && turn ? 1u : 0u;
                first_slot[r] = !live ? first_slot[r - 1] : turn ? 0u : slot;
                block[r] = entry(at);
            }
        };
        auto fetch = [&](unsigned dst) { // the next tile into a slot of the ring
            if (f_left > 0) {
                constexpr int kCopies = CPR * TILE / 32; // of a lane, for K as for V
                const unsigned char *k_run[kRuns], *v_run[kRuns];
#pragma unroll
                for (int r = 0; r < kRuns; ++r) {
                    const unsigned row = DENSE ? C::kRowBytes : code_slot;
                    k_run[r] = k_lane + static_cast<unsigned long long>(block[r]) * code_block + static_cast<unsigned long long>(first_slot[r]) * row;
                    v_run[r] = v_lane + static_cast<unsigned long long>(block[r]) * code_block + static_cast<unsigned long long>(first_slot[r]) * row;
                }
#pragma unroll
                for (int j = 0; j < kCopies; ++j) {
                    const int i = lane + 32 * j, r = i / CPR, c = i % CPR;
                    const int swz = CPR % 8 == 0 ? (r & 7) : CPR % 4 == 0 ? ((r >> 1) & 3) : ((r >> 2) & 1);
                    const unsigned to = dst + r * C::kRowBytes + ((c ^ swz) << 4);
                    if constexpr (DENSE) {
                        constexpr int kOfRun = kCopies / kRuns; // copies of a run are 512 bytes apart
                        copy16(to, k_run[j / kOfRun] + j % kOfRun * 512, policy);
                        copy16(to + TILE * C::kRowBytes, v_run[j / kOfRun] + j % kOfRun * 512, policy);
                    } else {
                        const int sub = SUBS == 1 ? 0 : 32 * j / CPR / 16; // where there are two, 16 rows are whole rounds of the warp
                        const unsigned in = static_cast<unsigned>(r & 7) * code_slot + c * 16;
                        copy16(to, ((r & 8) ? k_run[kRuns == 1 ? 0 : 2 * sub + 1] : k_run[kRuns == 1 ? 0 : 2 * sub]) + in, policy);
                        copy16(to + TILE * C::kRowBytes, ((r & 8) ? v_run[kRuns == 1 ? 0 : 2 * sub + 1] : v_run[kRuns == 1 ? 0 : 2 * sub]) + in, policy);
                    }
                }
                // scales: 8 rows are one run of NG chunks
                if (lane < TILE / 4 * NG) {
                    const int h = (lane / NG) & (TILE / 8 - 1), r = DENSE ? h >> 1 : h;
                    unsigned b = block[0], at = first_slot[0];
#pragma unroll
                    for (int k = 1; k < kRuns; ++k) {
                        b = r == k ? block[k] : b;
                        at = r == k ? first_slot[k] : at;
                    }
                    copy16(dst + 2 * TILE * C::kRowBytes + lane * 16, s_lane + static_cast<unsigned long long>(b) * scale_block + at * (2u * NG), policy);
                }
                f_half += TILE / 8;
                if (--f_left == 0) {
                    Walk w = copies;
                    f_left = w.step<TILE>(a, p.subs);
                    __syncwarp();
                    copies = w;
                    __syncwarp();
                    f_half = 0;
                    unit();
                }
                if (f_left > 0) {
                    look();
                }
            }
            commitCopies();
        };
        // q of a unit as it lies in memory: heads g and g + 8, at 4 bits 8 elements from 32 j + 8 t, at 8 bits 4 from 32 j + 4 t and 4 from
        // 16 behind; loaded a unit ahead
        uint4 q_raw[NH][HD / 32];
        auto loadQ = [&]() {
            const int kv = work.sub / p.head_tiles, head0 = (work.sub - kv * p.head_tiles) * HT;
            const int row = SPLIT == kColumns ? g & 3 : g; // columns 4 to 7 are heads 0 to 3 again
            const unsigned short *q = static_cast<const unsigned short *>(a.q) + work.seq * a.q_seq
                                    + (static_cast<long long>(kv) * a.group + head0 + row) * a.q_head;
#pragma unroll
            for (int n = 0; n < NH; ++n) {
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) {
                    q_raw[n][j] = make_uint4(0, 0, 0, 0);
                    if (head0 + row + 8 * n < a.group) {
                        const unsigned short *from = q + 8 * n * a.q_head + 32 * j;
                        if constexpr (BITS == 4) {
                            q_raw[n][j] = *reinterpret_cast<const uint4 *>(from + 8 * t);
                        } else {
                            const uint2 lo = *reinterpret_cast<const uint2 *>(from + 4 * t);
                            const uint2 hi = *reinterpret_cast<const uint2 *>(from + 16 + 4 * t);
                            q_raw[n][j] = make_uint4(lo.x, lo.y, hi.x, hi.y);
                        }
                    }
                }
            }
        };
        loadQ();
        unit();
        look();
        const unsigned ring_addr = smemAddr(ring);
#pragma unroll
        for (int i = 0; i < S - 1; ++i) {
            fetch(ring_addr + i * C::kStage);
        }
        unsigned stage = ring_addr, spare = ring_addr + (S - 1) * C::kStage; // the tile to work on, the slot to fill

        // lane's part of the matrix loads: matrix lane / 8, row lane % 8; matrices are (tokens 0-7 | 8-15) x (chunk, chunk + 1)
        const int m_row = (lane & 7) + ((lane >> 3) & 1) * 8, m_chunk = lane >> 4;
        const int m_swz = CPR % 8 == 0 ? (m_row & 7) : CPR % 4 == 0 ? ((m_row >> 1) & 3) : ((m_row >> 2) & 1);

        while (left > 0) { // a unit, or what of it is in the range
            const int kv = work.sub / p.head_tiles;
            const int head0 = (work.sub - kv * p.head_tiles) * HT; // within the group
            const int heads = min(HT, a.group - head0);
            const long long head_at = static_cast<long long>(kv) * a.group + head0;
            const int len = work.len;

            // q, scaled by a power of two for each head; the scores' factor takes it back
            unsigned qr[NH][HD / 16][2];             // of head g: second operand, [.][k step][.]
            float factor[NH][2], slope[NH][2];       // of the scores' columns, heads 2t and 2t + 1
#pragma unroll
            for (int n = 0; n < NH; ++n) {
                const int h = (SPLIT == kColumns ? g & 3 : g) + 8 * n;
                unsigned largest = 0;
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) {
                    const uint4 &x = q_raw[n][j];
                    const unsigned m = 0x7fff7fffu;
                    const unsigned b = __vmaxu2(__vmaxu2(x.x & m, x.y & m), __vmaxu2(x.z & m, x.w & m));
                    largest = max(largest, max(b & 0xffffu, b >> 16));
                }
                largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                auto wide = [&](unsigned half) {
                    return a.is_bf16 ? __uint_as_float(half << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(half)));
                };
                const int e = static_cast<int>(__float_as_uint(wide(largest)) >> 23); // biased
                const int down = max(253 - e, 1);                                     // 2^(126 - e)
                const float scale_q = __uint_as_float(static_cast<unsigned>(down) << 23);
                const float back = a.scale_log2e * __uint_as_float(static_cast<unsigned>(254 - down) << 23);
                const float bias = a.alibi != nullptr && h < heads ? a.alibi[head_at + h] * 1.4426950408889634f : 0.f;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    factor[n][x] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * x);
                    slope[n][x] = __shfl_sync(0xffffffffu, bias, 8 * t + 4 * x);
                }
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) {
                    const unsigned raw[4] = {q_raw[n][j].x, q_raw[n][j].y, q_raw[n][j].z, q_raw[n][j].w};
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[2 * i] = wide(raw[i] & 0xffffu) * scale_q;
                        x[2 * i + 1] = wide(raw[i] >> 16) * scale_q;
                    }
                    if constexpr (BITS == 4) { // the order of codes4
                        qr[n][2 * j][0] = packHalves(x[0], x[4]);
                        qr[n][2 * j][1] = packHalves(x[1], x[5]);
                        qr[n][2 * j + 1][0] = packHalves(x[2], x[6]);
                        qr[n][2 * j + 1][1] = packHalves(x[3], x[7]);
                    } else {
                        qr[n][2 * j][0] = packHalves(x[0], x[1]);
                        qr[n][2 * j][1] = packHalves(x[2], x[3]);
                        qr[n][2 * j + 1][0] = packHalves(x[4], x[5]);
                        qr[n][2 * j + 1][1] = packHalves(x[6], x[7]);
                    }
                }
            }

            float top[NH][2], sum[NH][2], o[NH][HD / 16][4];
#pragma unroll
            for (int n = 0; n < NH; ++n) {
                top[n][0] = top[n][1] = kLowest;
                sum[n][0] = sum[n][1] = 0.f;
#pragma unroll
                for (int j = 0; j < HD / 16; ++j) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[n][j][i] = 0.f;
                    }
                }
            }

            // exponents of the groups' factors, and the least of a head's, which is in top and counts for all where `even`
            float *const factors = all_factors + warp * (C::kFactors / 4);
            bool even = false, fresh = true;

            int token0 = tile * TILE;
            // from this token on a tile needs more than the plain arithmetic: a distance bias, tokens behind the end
            int special = a.alibi != nullptr ? 0 : max(len - TILE + 1, 0);
            // Beyond 2^20 a score's own rounding is seen in p.  Then scores are rounded before the maximum is taken off, so that the largest
            // is off by nothing; `special` is -1 from there on.
            do {
                waitCopies<S - 2>();
                __syncwarp();
                fetch(spare);
                const unsigned k_addr = stage + m_row * C::kRowBytes, v_addr = k_addr + TILE * C::kRowBytes;

                // scales of the lane's tokens g and g + 8 of each 16, two groups a word (one scale: the low half)
                constexpr int kWords = NG == 1 ? 1 : NG / 2;
                const unsigned char *scales = ring + (stage - ring_addr) + 2 * TILE * C::kRowBytes + g * (2 * NG);
                auto loadScales = [](unsigned (&w)[kWords], const unsigned char *from) {
                    if constexpr (NG == 1) {
                        w[0] = *reinterpret_cast<const unsigned short *>(from);
                    } else if constexpr (kWords == 4) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(from);
                        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
                    } else if constexpr (kWords == 2) {
                        const uint2 x = *reinterpret_cast<const uint2 *>(from);
                        w[0] = x.x, w[1] = x.y;
                    } else {
#pragma unroll
                        for (int i = 0; i < kWords; ++i) {
                            w[i] = reinterpret_cast<const unsigned *>(from)[i];
                        }
                    }
                };
                auto scaleAt = [](const unsigned (&w)[kWords], int j) {
                    return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
                };

                float s[SUBS][NH][4]; // [.][.][token g, heads 2t and 2t + 1 | token g + 8]: scores, p
                unsigned vs[SUBS][2][kWords];
                unsigned weight[SUBS][NG][NH][2];
                float add[NH][2];
#pragma unroll 1
                for (bool settle = fresh || special < 0;; settle = true) {
                    // scores
#pragma unroll
                    for (int u = 0; u < SUBS; ++u) {
                        unsigned ks[2][kWords];
                        loadScales(ks[0], scales + u * (32 * NG));
                        loadScales(ks[1], scales + u * (32 * NG) + 16 * NG);
#pragma unroll
                        for (int n = 0; n < NH; ++n) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                s[u][n][i] = 0.f;
                            }
                        }
#pragma unroll
                        for (int c = 0; c < CPR; c += 2) {
                            unsigned w[4];
                            loadMatrices(w, k_addr + u * (16 * C::kRowBytes) + (((c + m_chunk) ^ m_swz) << 4));
#pragma unroll
                            for (int x = 0; x < 2; ++x) { // the two chunks
                                const int j = c + x;
                                if constexpr (BITS == 4) {
                                    unsigned lo[4], hi[4];
                                    codes4(magic, w[2 * x], lo);
                                    codes4(magic, w[2 * x + 1], hi);
                                    const float s0 = scaleAt(ks[0], j), s1 = scaleAt(ks[1], j);
#pragma unroll
                                    for (int n = 0; n < NH; ++n) {
                                        float d[4];
                                        mmaFirst(d, lo[0], hi[0], lo[1], hi[1], qr[n][2 * j][0], qr[n][2 * j][1]);
                                        mma(d, lo[2], hi[2], lo[3], hi[3], qr[n][2 * j + 1][0], qr[n][2 * j + 1][1]);
                                        s[u][n][0] = fmaf(s0, d[0], s[u][n][0]);
                                        s[u][n][1] = fmaf(s0, d[1], s[u][n][1]);
                                        s[u][n][2] = fmaf(s1, d[2], s[u][n][2]);
                                        s[u][n][3] = fmaf(s1, d[3], s[u][n][3]);
                                    }
                                } else {
                                    const unsigned lo = w[2 * x] ^ 0x80808080u, hi = w[2 * x + 1] ^ 0x80808080u;
                                    const unsigned a0 = codes8<0x4140>(magic, lo), a1 = codes8<0x4140>(magic, hi);
                                    const unsigned a2 = codes8<0x4342>(magic, lo), a3 = codes8<0x4342>(magic, hi);
#pragma unroll
                                    for (int n = 0; n < NH; ++n) {
                                        mma(s[u][n], a0, a1, a2, a3, qr[n][j][0], qr[n][j][1]);
                                    }
                                }
                            }
                        }
                        if constexpr (BITS == 8) {
                            const float s0 = scaleAt(ks[0], 0), s1 = scaleAt(ks[1], 0);
#pragma unroll
                            for (int n = 0; n < NH; ++n) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    s[u][n][i] *= i < 2 ? s0 : s1;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int u = 0; u < SUBS; ++u) {
                        loadScales(vs[u][0], scales + 2 * TILE * NG + u * (32 * NG));
                        loadScales(vs[u][1], scales + 2 * TILE * NG + u * (32 * NG) + 16 * NG);
                    }
                    // scores in the log2 domain are s * f from here on
                    float f[NH][2];
#pragma unroll
                    for (int n = 0; n < NH; ++n) {
                        f[n][0] = factor[n][0];
                        f[n][1] = factor[n][1];
                    }
                    if (token0 >= special) {
#pragma unroll
                        for (int n = 0; n < NH; ++n) {
                            f[n][0] = f[n][1] = 1.f;
                        }
#pragma unroll
                        for (int r = 0; r < 2 * SUBS; ++r) {
                            const int u = r >> 1, i = 2 * (r & 1), token = token0 + 8 * r + g;
                            const float far = static_cast<float>(token - (len - 1));
#pragma unroll
                            for (int n = 0; n < NH; ++n) {
                                s[u][n][i] = fmaf(slope[n][0], far, s[u][n][i] * factor[n][0]);
                                s[u][n][i + 1] = fmaf(slope[n][1], far, s[u][n][i + 1] * factor[n][1]);
                            }
                            if (token >= len) { // no weight, whatever the scales are
#pragma unroll
                                for (int n = 0; n < NH; ++n) {
                                    s[u][n][i] = s[u][n][i + 1] = -INFINITY;
                                }
#pragma unroll
                                for (int k = 0; k < kWords; ++k) {
                                    vs[u][r & 1][k] = 0u;
                                }
                            }
                        }
                    }

                    if (__builtin_expect(settle, 0)) {
                        float *const mine = factors + 2 * t; // of this lane's heads: eight lanes, the same
                        bool far = special < 0;
                        float now[NH][2];
#pragma unroll
                        for (int n = 0; n < NH; ++n) {
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                float m = -INFINITY;
#pragma unroll
                                for (int r = 0; r < 2 * SUBS; ++r) {
                                    m = fmaxf(m, __fmul_rn(s[r >> 1][n][2 * (r & 1) + x], f[n][x]));
                                }
                                m = largestOf(m);
                                far |= fabsf(m) >= 1048576.f && m != -INFINITY;
                                now[n][x] = ceilf(m) + kBelow; // a whole number
                            }
                        }
                        far = __any_sync(0xffffffffu, far);
                        if (far) {
                            special = -1;
#pragma unroll
                            for (int u = 0; u < SUBS; ++u) {
#pragma unroll
                                for (int n = 0; n < NH; ++n) {
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        s[u][n][i] = __fmul_rn(s[u][n][i], f[n][i & 1]);
                                    }
                                }
                            }
#pragma unroll
                            for (int n = 0; n < NH; ++n) {
                                f[n][0] = f[n][1] = 1.f;
                            }
                        }
                        // p of before are smaller by 2^up now, and factors as much larger, up to their limit.  A group whose largest weight of this tile
                        // would be 2^8 or more gets a factor that makes it 2^7.
                        float common[NH][2], up[NH][2], is[NH][2][NG], least[NH][2];
                        bool near = !far;
#pragma unroll
                        for (int n = 0; n < NH; ++n) {
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                common[n][x] = even ? mine[NG * HT + 8 * n + x] : 0.f;
                                top[n][x] += common[n][x];
                                now[n][x] = fmaxf(now[n][x], top[n][x]);
                                up[n][x] = now[n][x] - top[n][x];
                                float most = -INFINITY;
                                least[n][x] = INFINITY;
#pragma unroll
                                for (int j = 0; j < NG; ++j) {
                                    float m = 0.f;
#pragma unroll
                                    for (int r = 0; r < 2 * SUBS; ++r) {
                                        const float p = exp2Fast(fmaf(s[r >> 1][n][2 * (r & 1) + x], f[n][x], -now[n][x]));
                                        m = fmaxf(m, fabsf(p * scaleAt(vs[r >> 1][r & 1], j)));
                                    }
                                    const float high = exponentOf(largestOf(m));
                                    const float was = fresh ? kMostFactor : fminf(mine[j * HT + 8 * n + x] + up[n][x], kMostFactor);
                                    is[n][x][j] = high + was > kLargest ? kLargest - high : was;
                                    least[n][x] = fminf(least[n][x], is[n][x][j]);
                                    most = fmaxf(most, is[n][x][j]);
                                }
                                near = near && most - least[n][x] <= kEven && least[n][x] >= kLeastCommon && least[n][x] <= kMostCommon;
                            }
                        }
                        const bool was_even = even;
                        even = __all_sync(0xffffffffu, near);
                        if (!fresh) {
#pragma unroll
                            for (int n = 0; n < NH; ++n) {
#pragma unroll
                                for (int x = 0; x < 2; ++x) {
#pragma unroll
                                    for (int j = 0; j < NG; ++j) {
                                        const float was = was_even ? common[n][x] : mine[j * HT + 8 * n + x];
                                        scaleGroup<BITS, HD>(o[n], j, x, ((even ? least[n][x] : is[n][x][j]) - was) - up[n][x]);
                                    }
                                    sum[n][x] = shifted(shifted(shifted(sum[n][x], -common[n][x]), -up[n][x]), even ? least[n][x] : 0.f);
                                }
                            }
                        }
                        __syncwarp();
#pragma unroll
                        for (int n = 0; n < NH; ++n) {
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                top[n][x] = now[n][x] - (even ? least[n][x] : 0.f);
#pragma unroll
                                for (int j = 0; j < NG; ++j) {
                                    mine[j * HT + 8 * n + x] = is[n][x][j];
                                }
                                mine[NG * HT + 8 * n + x] = least[n][x];
                            }
                        }
                        __syncwarp();
                        fresh = false;
                    }
                    // p, and the weights p * v_scale * factor in fp16
#pragma unroll
                    for (int n = 0; n < NH; ++n) {
                        add[n][0] = add[n][1] = 0.f;
                    }
#pragma unroll
                    for (int u = 0; u < SUBS; ++u) {
#pragma unroll
                        for (int n = 0; n < NH; ++n) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                s[u][n][i] = exp2Fast(fmaf(s[u][n][i], f[n][i & 1], -top[n][i & 1]));
                            }
                            add[n][0] += s[u][n][0] + s[u][n][2];
                            add[n][1] += s[u][n][1] + s[u][n][3];
                            if constexpr (SPLIT == kColumns) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const float p = leading(s[u][n][i]);
                                    s[u][n][i] = t < 2 ? p : s[u][n][i] - p;
                                }
                            }
                        }
                    }
                    unsigned largest = 0;
                    auto weigh = [&](auto part, auto factor) {
#pragma unroll
                        for (int j = 0; j < NG; ++j) {
#pragma unroll
                            for (int n = 0; n < NH; ++n) {
                                const float by0 = factor(j, n, 0), by1 = factor(j, n, 1);
#pragma unroll
                                for (int u = 0; u < SUBS; ++u) {
                                    const float v0 = scaleAt(vs[u][0], j), v1 = scaleAt(vs[u][1], j);
                                    weight[u][j][n][0] = packHalves(part(s[u][n][0]) * by0 * v0, part(s[u][n][1]) * by1 * v0);
                                    weight[u][j][n][1] = packHalves(part(s[u][n][2]) * by0 * v1, part(s[u][n][3]) * by1 * v1);
                                    largest = __vmaxu2(largest, __vmaxu2(weight[u][j][n][0], weight[u][j][n][1]));
                                }
                            }
                        }
                    };
                    if (even) {
                        weigh([](float p) { return SPLIT == kTwice ? leading(p) : p; }, [](int, int, int) { return 1.f; });
                    } else {
                        weigh([](float p) { return p; }, [&](int j, int n, int x) { return powerOfTwo(factors[j * HT + 8 * n + 2 * t + x]); });
                    }
                    bool again = max(largest & 0xffffu, largest >> 16) >= 0x7c00u; // an infinity, or no number
#pragma unroll
                    for (int n = 0; n < NH; ++n) {
                        again |= fmaxf(add[n][0], add[n][1]) > kMostP;
                    }
                    if (__builtin_expect(settle || !__any_sync(0xffffffffu, again), 1)) {
                        break;
                    }
                }
#pragma unroll
                for (int n = 0; n < NH; ++n) {
                    sum[n][0] += add[n][0];
                    sum[n][1] += add[n][1];
                }

                // outputs
                if constexpr (SPLIT == kTwice) { // what the weights are short of; not even, they were rounded whole
#pragma unroll
                    for (int u = 0; u < SUBS; ++u) {
#pragma unroll
                        for (int n = 0; n < NH; ++n) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                s[u][n][i] = even ? s[u][n][i] - leading(s[u][n][i]) : 0.f;
                            }
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < SUBS; ++u) {
                    [[maybe_unused]] unsigned rest[NH][2];
                    unsigned turned[NH][2];
#pragma unroll
                    for (int c = 0; c < CPR; c += 2) {
                        unsigned w[4];
                        loadMatricesTransposed(w, v_addr + u * (16 * C::kRowBytes) + (((c + m_chunk) ^ m_swz) << 4));
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int j = c + x;
                            if (BITS == 4 || j == 0) { // the weights of this group
#pragma unroll
                                for (int n = 0; n < NH; ++n) {
                                    turned[n][0] = transposed(weight[u][BITS == 4 ? j : 0][n][0]);
                                    turned[n][1] = transposed(weight[u][BITS == 4 ? j : 0][n][1]);
                                    if constexpr (SPLIT == kTwice) {
                                        const float v0 = scaleAt(vs[u][0], BITS == 4 ? j : 0), v1 = scaleAt(vs[u][1], BITS == 4 ? j : 0);
                                        rest[n][0] = transposed(packHalves(s[u][n][0] * v0, s[u][n][1] * v0));
                                        rest[n][1] = transposed(packHalves(s[u][n][2] * v1, s[u][n][3] * v1));
                                    }
                                }
                            }
                            if constexpr (BITS == 4) {
                                unsigned lo[4], hi[4];
                                codes4Odd16(magic, w[2 * x], lo);
                                codes4Odd16(magic, w[2 * x + 1], hi);
#pragma unroll
                                for (int n = 0; n < NH; ++n) {
                                    mma(o[n][2 * j], lo[0], lo[1], hi[0], hi[1], turned[n][0], turned[n][1]);
                                    mma(o[n][2 * j + 1], lo[2], lo[3], hi[2], hi[3], turned[n][0], turned[n][1]);
                                    if constexpr (SPLIT == kTwice) {
                                        mma(o[n][2 * j], lo[0], lo[1], hi[0], hi[1], rest[n][0], rest[n][1]);
                                        mma(o[n][2 * j + 1], lo[2], lo[3], hi[2], hi[3], rest[n][0], rest[n][1]);
                                    }
                                }
                            } else {
                                const unsigned lo = w[2 * x] ^ 0x80808080u, hi = w[2 * x + 1] ^ 0x80808080u;
                                const unsigned a0 = codes8<0x4240>(magic, lo), a1 = codes8<0x4341>(magic, lo);
                                const unsigned a2 = codes8<0x4240>(magic, hi), a3 = codes8<0x4341>(magic, hi);
#pragma unroll
                                for (int n = 0; n < NH; ++n) {
                                    mma(o[n][j], a0, a1, a2, a3, turned[n][0], turned[n][1]);
                                    if constexpr (SPLIT == kTwice) {
                                        mma(o[n][j], a0, a1, a2, a3, rest[n][0], rest[n][1]);
                                    }
                                }
                            }
                        }
                    }
                }
                token0 += TILE;
                spare = stage;
                stage = stage == ring_addr + (S - 1) * C::kStage ? ring_addr : stage + C::kStage;
            } while (--left > 0);

            if constexpr (SPLIT == kColumns) { // the halves together: columns 4 to 7 belong to the lanes with t + 2
#pragma unroll
                for (int n = 0; n < NH; ++n) {
#pragma unroll
                    for (int j = 0; j < HD / 16; ++j) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            o[n][j][i] += __shfl_xor_sync(0xffffffffu, o[n][j][i], 2);
                        }
                    }
                }
            }
            if (!even) { // the factors off
#pragma unroll
                for (int n = 0; n < NH; ++n) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
#pragma unroll
                        for (int j = 0; j < NG; ++j) {
                            scaleGroup<BITS, HD>(o[n], j, x, -factors[j * HT + 8 * n + 2 * t + x]);
                        }
                    }
                }
            }
            // the unit's rows, or this warp's piece of it
            const Walk done = work;
            const long long unit_first = place - tile;
            const bool first = unit_first >= start, last = unit_first + done.tiles <= end;
            {
                Walk w = done;
                left = last ? w.step<TILE>(a, p.subs) : 0;
                __syncwarp();
                work = w;
                __syncwarp();
                if (left > 0) {
                    loadQ();
                }
            }
            place = unit_first + done.tiles + unitCost(TILE); // if the range goes on, it does with the next unit
            tile = 0;
            float inv[NH][2];
#pragma unroll
            for (int n = 0; n < NH; ++n) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    sum[n][x] += __shfl_xor_sync(0xffffffffu, sum[n][x], 4);
                    sum[n][x] += __shfl_xor_sync(0xffffffffu, sum[n][x], 8);
                    sum[n][x] += __shfl_xor_sync(0xffffffffu, sum[n][x], 16);
                    inv[n][x] = 1.f / sum[n][x];
                }
            }
            if (first && last && lane == 0 && p.task_of_unit && !p.unit_of_cta) {
                tasks[done.seq * p.subs + done.sub].pieces = 0;
            }
            if (!(first && last) && lane == 0) {
                pieces[2 * warp + first] = {unit_first, done.seq, done.sub, done.tiles, 1};
            }
            // a piece in front is kept beside the ring, one at the range's end in the ring, which is empty then
            float *mine_o = first ? reinterpret_cast<float *>(ring) : results + warp * HT * C::kStride;
            __syncwarp();
#pragma unroll
            for (int n = 0; n < NH; ++n) {
                constexpr int kPer = BITS == 4 ? 4 : 2; // neighbouring elements of a row that a lane has
                constexpr int kRuns = HD / (8 * kPer);
                if (first && last) {
                    const long long row = done.seq * a.o_seq + (head_at + 8 * n + 2 * t) * a.o_head;
#pragma unroll
                    for (int j = 0; j < kRuns; ++j) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float f = inv[n][x];
                            float v[kPer];
                            v[0] = o[n][BITS == 4 ? 2 * j : j][x] * f;
                            v[1] = o[n][BITS == 4 ? 2 * j : j][2 + x] * (BITS == 4 ? f * 0.0625f : f);
                            if constexpr (BITS == 4) {
                                v[2] = o[n][2 * j + 1][x] * f;
                                v[3] = o[n][2 * j + 1][2 + x] * (f * 0.0625f);
                            }
                            if (8 * n + 2 * t + x < heads) {
                                storeOut(a, p, row + x * a.o_head + 8 * kPer * j + kPer * g, v);
                            }
                        }
                    }
                } else {
                    if (g == 0) {
                        sums[(2 * warp + first) * HT + 8 * n + 2 * t] = make_float2(top[n][0], sum[n][0]);
                        sums[(2 * warp + first) * HT + 8 * n + 2 * t + 1] = make_float2(top[n][1], sum[n][1]);
                    }
                    float *row0 = mine_o + (8 * n + 2 * t) * C::kStride, *row1 = row0 + C::kStride;
#pragma unroll
                    for (int j = 0; j < kRuns; ++j) {
                        if constexpr (BITS == 4) {
                            const float(&x)[4] = o[n][2 * j], (&y)[4] = o[n][2 * j + 1];
                            *reinterpret_cast<float4 *>(row0 + 32 * j + 4 * g) = make_float4(x[0], x[2] * 0.0625f, y[0], y[2] * 0.0625f);
                            *reinterpret_cast<float4 *>(row1 + 32 * j + 4 * g) = make_float4(x[1], x[3] * 0.0625f, y[1], y[3] * 0.0625f);
                        } else {
                            *reinterpret_cast<float2 *>(row0 + 16 * j + 2 * g) = make_float2(o[n][j][0], o[n][j][2]);
                            *reinterpret_cast<float2 *>(row1 + 16 * j + 2 * g) = make_float2(o[n][j][1], o[n][j][3]);
                        }
                    }
                }
            }
        }
    }

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // ---- the pieces that this CTA's warps left: those of one unit are neighbours
    __syncthreads();
    int cut = 0; // the pieces of the CTA's last unit, where that goes on in other CTAs
#pragma unroll 1
    for (int k = 0; k < 2 * kWarps;) {
        const Piece piece = pieces[k];
        if (!piece.used) {
            ++k;
            continue;
        }
        int upto_k = k + 1; // members: used pieces from k on with the same unit
        while (upto_k < 2 * kWarps && (!pieces[upto_k].used || pieces[upto_k].first == piece.first)) {
            ++upto_k;
        }
        const int kv = piece.sub / p.head_tiles, head0 = (piece.sub - kv * p.head_tiles) * HT, heads = min(HT, a.group - head0);
        const long long head_at = static_cast<long long>(kv) * a.group + head0;
        const bool first = piece.first >= cta_start, last = piece.first + piece.tiles <= cta_start + cta_range;
        float *record = reinterpret_cast<float *>(p.workspace + p.tasks_bytes) + (2ll * blockIdx.x + (first ? 1 : 0)) * C::kRecord;
        for (int i = tid; i < heads * (HD / 4); i += kThreads) {
            const int h = i / (HD / 4), d = 4 * (i % (HD / 4));
            float m = kLowest;
            for (int w = k; w < upto_k; ++w) {
                m = pieces[w].used ? fmaxf(m, sums[w * HT + h].x) : m;
            }
            float l = 0.f;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            for (int w = k; w < upto_k; ++w) {
                if (pieces[w].used) {
                    const float2 ml = sums[w * HT + h];
                    const float f = exp2Fast(ml.x - m);
                    const float *from = (w & 1) ? reinterpret_cast<const float *>(smem + (w >> 1) * C::kRing) : results + (w >> 1) * HT * C::kStride;
                    const float4 x = *reinterpret_cast<const float4 *>(from + h * C::kStride + d);
                    l = fmaf(f, ml.y, l);
                    v[0] = fmaf(f, x.x, v[0]);
                    v[1] = fmaf(f, x.y, v[1]);
                    v[2] = fmaf(f, x.z, v[2]);
                    v[3] = fmaf(f, x.w, v[3]);
                }
            }
            if (first && last) {
                const float inv = 1.f / l;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    v[x] *= inv;
                }
                storeOut(a, p, piece.seq * a.o_seq + (head_at + h) * a.o_head + d, v);
            } else {
                *reinterpret_cast<float4 *>(record + h * HD + d) = make_float4(v[0], v[1], v[2], v[3]);
                if (d == 0) {
                    record[HT * HD + h] = m;
                    record[HT * HD + HT + h] = l;
                }
            }
        }
        if (first) {
            cut = last ? 0 : static_cast<int>((piece.first + piece.tiles - 1) / cta_range - blockIdx.x) + 1;
            if (tid == 0 && !p.unit_of_cta && (cut > 0 || p.task_of_unit)) {
                tasks[p.task_of_unit ? piece.seq * p.subs + piece.sub : static_cast<int>(blockIdx.x)] = {piece.seq, piece.sub, cut,
                                                                                                        static_cast<int>(blockIdx.x)};
            }
        }
        k = upto_k;
    }
    if (tid == 0 && cut == 0 && !p.task_of_unit && !p.unit_of_cta) {
        tasks[blockIdx.x].pieces = 0;
    }
}

// Adds the pieces of a cut unit: CTA (task, part of its heads).  A thread has four columns of a head and every kSides-th
// piece, which it adds as they come (maximum, sum, output); the sides meet in shared memory.  Several sides read at a
// time, since a long sequence alone may lie in pieces over the whole grid.
constexpr int kCombineThreads = 512;

template <int HD, int HT>
__global__ void __launch_bounds__(kCombineThreads) quantAttentionCombineKernel(const AttentionArgs a, const TilesArgs p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int kRecord = HT * HD + 2 * HT, kColumns = HD / 4;
    __shared__ float4 part[kCombineThreads];
    __shared__ float2 part_ml[kCombineThreads];
    const Task task = reinterpret_cast<const Task *>(p.workspace)[blockIdx.x];
    if (p.task_of_unit && lengthOf(a, static_cast<int>(blockIdx.x) / p.subs) <= 0) {
        return; // no one wrote this task
    }
    const int kv = task.sub / p.head_tiles, head0 = (task.sub - kv * p.head_tiles) * HT; // within the group
    const int h0 = static_cast<int>(blockIdx.y) * p.combine_heads;
    const int heads = min(p.combine_heads, min(HT, a.group - head0) - h0);
    if (task.pieces == 0 || heads <= 0) {
        return;
    }
    const float *records = reinterpret_cast<const float *>(p.workspace + p.tasks_bytes);
    const int items = p.combine_heads * kColumns; // a multiple or a part of the threads
    const int sides = items < kCombineThreads ? kCombineThreads / items : 1;
    const int side = static_cast<int>(threadIdx.x) / items;
    for (int item = sides > 1 ? static_cast<int>(threadIdx.x) % items : static_cast<int>(threadIdx.x); item < items; item += sides > 1 ? items : kCombineThreads) {
        const int h = h0 + item / kColumns, column = item % kColumns;
        const bool live = item / kColumns < heads;
        float m = kLowest, l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (live && side < sides) {
#pragma unroll 4
            for (int k = side; k < task.pieces; k += sides) {
                // piece 0 is the second record of the CTA that began the unit, piece k the first one of the k-th CTA behind it
                const float *r = records + (2ll * (task.cta + k) + (k == 0 ? 1 : 0)) * kRecord;
                const float mk = r[HT * HD + h], lk = r[HT * HD + HT + h];
                const float4 x = *reinterpret_cast<const float4 *>(r + h * HD + 4 * column);
                const float now = fmaxf(m, mk), f = exp2Fast(m - now), fk = exp2Fast(mk - now);
                m = now;
                l = fmaf(f, l, fk * lk);
                v.x = fmaf(f, v.x, fk * x.x);
                v.y = fmaf(f, v.y, fk * x.y);
                v.z = fmaf(f, v.z, fk * x.z);
                v.w = fmaf(f, v.w, fk * x.w);
            }
        }
        if (sides > 1) {
            part[threadIdx.x] = v;
            part_ml[threadIdx.x] = make_float2(m, l);
            __syncthreads();
            if (side == 0) {
                for (int k = 1; k < sides && k < task.pieces; ++k) {
                    const float2 ml = part_ml[k * items + item];
                    const float4 x = part[k * items + item];
                    const float now = fmaxf(m, ml.x), f = exp2Fast(m - now), fk = exp2Fast(ml.x - now);
                    m = now;
                    l = fmaf(f, l, fk * ml.y);
                    v.x = fmaf(f, v.x, fk * x.x);
                    v.y = fmaf(f, v.y, fk * x.y);
                    v.z = fmaf(f, v.z, fk * x.z);
                    v.w = fmaf(f, v.w, fk * x.w);
                }
            }
        }
        if (live && side == 0) {
            const float inv = 1.f / l;
            const float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
            storeOut(a, p, task.seq * a.o_seq + (static_cast<long long>(kv) * a.group + head0 + h) * a.o_head + 4 * column, y);
        }
    }
}

using TilesKernel = void (*)(AttentionArgs, TilesArgs);

struct Variant {
    TilesKernel tiles[2], combine; // any | dense
    int ctas, smem, record, heads, tile;
};

template <int BITS, int HD, int HT, Split SPLIT>
Variant variant() {
    using C = Cfg<BITS, HD, HT>;
    return {{quantAttentionTilesKernel<BITS, HD, HT, false, SPLIT>, quantAttentionTilesKernel<BITS, HD, HT, true, SPLIT>}, quantAttentionCombineKernel<HD, HT>, C::kCtas, C::kSmem, C::kRecord, HT, C::kTile};
}

template <int BITS, int HD, int HT>
Variant variantFor(bool fp16, size_t group) {
    if constexpr (HT == 8) {
        if (fp16 && group <= 4) {
            return variant<BITS, HD, HT, kColumns>();
        }
    }
    return fp16 ? variant<BITS, HD, HT, kTwice>() : variant<BITS, HD, HT, kWhole>();
}

template <int BITS>
Variant variantFor(size_t head, bool fp16, size_t group) {
    // 16 heads share a pass over the codes where a group has more than 8; at heads of 192 and 256 their outputs would not
    // fit the registers.  Measured at 64/4 heads, 64 x 4096 tokens, bf16 (us, one pass | two of 8 heads): heads of 128 70 | 80 at
    // 4 bits, 72 | 100 at 8; heads of 64 45 | 50, 45 | 58.
    switch (head) {
    case 64:
        return group > 8 ? variantFor<BITS, 64, 16>(fp16, group) : variantFor<BITS, 64, 8>(fp16, group);
    case 128:
        return group > 8 ? variantFor<BITS, 128, 16>(fp16, group) : variantFor<BITS, 128, 8>(fp16, group);
    case 192:
        return variantFor<BITS, 192, 8>(fp16, group);
    default:
        return variantFor<BITS, 256, 8>(fp16, group);
    }
}

Variant variantFor(const AttentionInfo &I) {
    const size_t group = I.num_heads / I.pools.num_kv_heads;
    const bool fp16 = I.dtype == INFINI_DTYPE_F16;
    return I.pools.bits == 4 ? variantFor<4>(I.head_size, fp16, group) : variantFor<8>(I.head_size, fp16, group);
}

} // namespace

TilesPlan planTiles(const AttentionInfo &I, const DeviceProps &props) {
    TilesPlan plan;
    const Pools &P = I.pools;
    const Pool &k = P.k, &v = P.v;
    const ptrdiff_t groups = static_cast<ptrdiff_t>(k.groups);
    auto whole = [](ptrdiff_t stride, ptrdiff_t unit) { return stride % unit == 0; };
    auto narrow = [](ptrdiff_t stride) { return stride >= 0 && stride <= 0x7fffffff; };
    // copies of 16 bytes: 8 tokens of a block at a time, their scales one run; K and V laid out alike; strides of 32 bits
    plan.eligible = P.block_size % 8 == 0 && k.block == v.block && k.kv_head == v.kv_head && k.slot == v.slot && k.s_block == v.s_block
                 && k.s_head == v.s_head && k.s_slot == v.s_slot && k.s_slot == groups && whole(k.block, 16) && whole(k.kv_head, 16)
                 && whole(k.slot, 16) && whole(k.s_block, 8) && whole(k.s_head, 8) && whole(I.q_seq, 8) && whole(I.q_head, 8)
                 && narrow(k.block) && narrow(k.slot) && narrow(k.slot * 8) && narrow(k.s_block);
    if (!plan.eligible || I.num_seqs == 0 || I.num_heads == 0 || I.max_blocks == 0) {
        plan.eligible = false;
        return plan;
    }
    const Variant var = variantFor(I);
    const unsigned long long group = I.num_heads / P.num_kv_heads;
    const unsigned long long head_tiles = (group + var.heads - 1) / var.heads;
    const unsigned long long tokens = static_cast<unsigned long long>(I.max_blocks) * P.block_size; // 31 and 17 bits
    const unsigned long long tiles = (tokens + var.tile - 1) / var.tile;
    const unsigned long long subs = head_tiles * P.num_kv_heads;
    const long double line = static_cast<long double>(tiles + unitCost(var.tile)) * subs * I.num_seqs;
    const unsigned long long at_most = static_cast<unsigned long long>(props.sm_count) * var.ctas;
    if (tokens > static_cast<unsigned long long>(kMostTokensInt) || line > 9e17L || line / at_most > 1e9L) {
        plan.eligible = false; // positions would not fit
        return plan;
    }
    const unsigned long long useful = (static_cast<unsigned long long>(line) + kWarps * minRange(var.tile) - 1) / (kWarps * minRange(var.tile));
    plan.grid = static_cast<int>(useful < at_most ? useful : at_most);
    plan.head_tiles = static_cast<int>(head_tiles);
    plan.subs = static_cast<int>(subs);
    const unsigned long long units = subs * I.num_seqs; // below 2^64: the line is longer
    // A unit to each CTA saves the combine kernel, but lets the longest unit set the time; it is for units that are known to be short
    // and few enough to run at once.  Measured at 32/8 heads of 128 (us, a unit to each CTA | the line): 4 sequences of 256 tokens
    // 7.6 | 13.4 at 4 bits, 8.8 | 14.1 at 8; of 1024 13.1 | 13.6, 18.1 | 14.6; 16 of 1024 14.9 | 18.1, 20.4 | 20.2; 64 of 1024
    // at 8 bits 31 | 39; 256 of 256 (more units than fit) 41.5 | 35.3, 48 | 46.
    const size_t longest = P.block_size * I.max_blocks;
    plan.unit_of_cta = units <= at_most && longest <= (units >= 64 ? 1024u : 512u);
    if (plan.unit_of_cta) {
        plan.grid = static_cast<int>(units);
    }
    plan.task_of_unit = units <= static_cast<unsigned long long>(plan.grid);
    plan.tasks = plan.task_of_unit ? static_cast<int>(units) : plan.grid;
    // all heads of a unit in one CTA of the combine kernel, or each in its own: with few units each has many pieces
    const int heads = static_cast<int>(group < static_cast<unsigned long long>(var.heads) ? group : var.heads);
    plan.combine_heads = static_cast<long long>(plan.tasks) * heads > 8ll * props.sm_count ? heads : 1;
    plan.combine_parts = heads / plan.combine_heads;
    if (!plan.unit_of_cta) {
        plan.tasks_bytes = (sizeof(Task) * plan.tasks + 255) / 256 * 256;
        plan.workspace_bytes = plan.tasks_bytes + sizeof(float) * 2 * plan.grid * static_cast<size_t>(var.record);
    }
    // n / halves for n < 2^31 as mulhi(n, magic) >> shift: magic = floor(2^(32 + shift) / halves) + 1 with 2^shift < halves, which is
    // below 2^32 and off by at most halves, and n * halves < 2^(32 + shift); 2^(31) and one shift less for a power of two
    const unsigned halves = static_cast<unsigned>(P.block_size / 8);
    plan.dense = P.block_size % 16 == 0 && k.slot == static_cast<ptrdiff_t>(I.head_size * P.bits / 8);
    plan.half_self = halves == 1 ? 0xffffffffu : 0u;
    if (halves > 1) {
        while ((2u << plan.half_shift) <= halves) {
            ++plan.half_shift;
        }
        if ((1u << plan.half_shift) == halves) {
            plan.half_magic = 0x80000000u;
            --plan.half_shift;
        } else {
            plan.half_magic = static_cast<unsigned>((1ull << (32 + plan.half_shift)) / halves + 1);
        }
    }
    auto words = [](ptrdiff_t stride) { return stride % 4 == 0; };
    plan.out_words = words(I.o_seq) && words(I.o_head);
    return plan;
}

bool tilesTakePointers(const TilesPlan &plan, const AttentionArgs &a, const void *workspace) {
    return plan.eligible && alignedTo(a.k_codes, 16) && alignedTo(a.v_codes, 16) && alignedTo(a.k_scales, 16) && alignedTo(a.v_scales, 16)
        && alignedTo(a.q, 16) && alignedTo(workspace, 16);
}

infiniStatus_t launchTiles(const AttentionInfo &info, const TilesPlan &plan, const AttentionArgs &a, void *workspace, cudaStream_t stream) {
    const Variant var = variantFor(info);
    TilesArgs p;
    p.workspace = static_cast<unsigned char *>(workspace);
    p.tasks_bytes = static_cast<long long>(plan.tasks_bytes);
    p.combine_heads = plan.combine_heads;
    p.unit_of_cta = plan.unit_of_cta ? 1 : 0;
    p.task_of_unit = plan.task_of_unit ? 1 : 0;
    p.subs = plan.subs;
    p.head_tiles = plan.head_tiles;
    p.half_magic = plan.half_magic;
    p.half_self = plan.half_self;
    p.half_shift = plan.half_shift;
    p.index_shift = a.index_is_64 ? 3 : 2;
    p.halves = static_cast<unsigned>(a.block_size / 8);
    p.out_words = plan.out_words && alignedTo(a.out, 8) ? 1 : 0;
    const TilesKernel kernel = var.tiles[plan.dense];
    // an attribute of the device's function: set by the descriptor's first launch
    if (__atomic_load_n(&plan.ready, __ATOMIC_RELAXED) == 0) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, var.smem) != cudaSuccess) {
            return checkLaunch("quantAttentionTilesKernel: shared memory");
        }
        __atomic_store_n(&plan.ready, 1, __ATOMIC_RELAXED);
    }
    cudaLaunchAttribute pdl;
    pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl.val.programmaticStreamSerializationAllowed = info.use_pdl ? 1 : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(plan.grid));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(var.smem);
    cfg.stream = stream;
    cfg.attrs = &pdl;
    cfg.numAttrs = 1;
    (void)cudaLaunchKernelEx(&cfg, kernel, a, p);
    const infiniStatus_t st = checkLaunch("quantAttentionTilesKernel");
    if (st != INFINI_STATUS_SUCCESS || plan.unit_of_cta) {
        return st;
    }
    cfg.gridDim = dim3(static_cast<unsigned>(plan.tasks), static_cast<unsigned>(plan.combine_parts));
    cfg.blockDim = dim3(kCombineThreads);
    cfg.dynamicSmemBytes = 0;
    (void)cudaLaunchKernelEx(&cfg, var.combine, a, p);
    return checkLaunch("quantAttentionCombineKernel");
}

} // namespace b200::quant_paged_cache
