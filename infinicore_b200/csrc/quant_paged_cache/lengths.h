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
// name.  Compared in 64 bits: a length below -2^31 that were narrowed first could come out positive.
QUANT_HOST_DEVICE int liveTokens(long long n, long long most) {
    if (n <= 0) {
        return 0;
    }
    const long long len = n < most ? n : most;
    return len > 0x7fffffffLL ? 0x7fffffff : static_cast<int>(len);
}

} // namespace b200::quant_paged_cache

#endif
