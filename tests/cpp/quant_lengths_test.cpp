// The functions of csrc/quant_paged_cache/lengths.h:
//
//     quant_lengths_test <n> <most> [<n> <most> ...]     liveTokens of every pair
//     quant_lengths_test i64|i32|u32 <n> [<n> ...]       storedLength of every number, as that type
#include "quant_paged_cache/lengths.h"

#include <cstdio>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <vector>

namespace qc = b200::quant_paged_cache;

int main(int argc, char **argv) {
    if (argc > 1 && (argv[1][0] == 'i' || argv[1][0] == 'u')) {
        const bool wide = std::strcmp(argv[1], "i64") == 0;
        std::vector<int64_t> n64;
        std::vector<int32_t> n32;
        for (int i = 2; i < argc; ++i) {
            n64.push_back(std::strtoll(argv[i], nullptr, 10));
            n32.push_back(static_cast<int32_t>(static_cast<uint32_t>(n64.back())));
        }
        const int kind = wide ? qc::kLength64 : argv[1][0] == 'u' ? qc::kLengthU32 : qc::kLength32;
        for (int i = 0; i < argc - 2; ++i) {
            std::printf("%lld\n", qc::storedLength(wide ? static_cast<const void *>(n64.data()) : n32.data(), i, kind));
        }
        return 0;
    }
    for (int i = 1; i + 1 < argc; i += 2) {
        std::printf("%lld\n", static_cast<long long>(qc::liveTokens(std::strtoll(argv[i], nullptr, 10), std::strtoll(argv[i + 1], nullptr, 10))));
    }
    return 0;
}
