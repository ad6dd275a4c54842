// Arithmetic on sequence lengths that the quantised paged attention does on the GPU; plain C++, so that it can be tested on
// any machine.
#ifndef INFINIOP_B200_QUANT_LENGTHS_H
#define INFINIOP_B200_QUANT_LENGTHS_H

#ifdef __CUDACC__
#define QUANT_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define QUANT_HOST_DEVICE inline
#endif

namespace b200::quant_paged_cache {

// How a length is stored: I64, I32 or U32.
enum LengthKind : int { kLength64 = 0, kLength32 = 1, kLengthU32 = 2 };

QUANT_HOST_DEVICE long long storedLength(const void *lens, long long i, int kind) {
    return kind == kLength64   ? static_cast<const long long *>(lens)[i]
         : kind == kLengthU32 ? static_cast<long long>(static_cast<const unsigned *>(lens)[i])
                              : static_cast<long long>(static_cast<const int *>(lens)[i]);
}

// Tokens of a sequence whose stored length is n: none where n <= 0, never more than `most`, which its row of the table can
// name.  In 64 bits: a length below -2^31 that were narrowed could come out positive, and a table may name more than 2^31 tokens.
QUANT_HOST_DEVICE long long liveTokens(long long n, long long most) { return n <= 0 ? 0 : n < most ? n : most; }

// What a table may name for a kernel that counts tokens in an int, a whole tile of 64 behind the last one included.
constexpr long long kMostTokensInt = 0x7fffffffLL - 127;

} // namespace b200::quant_paged_cache

#endif
