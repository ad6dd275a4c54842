// liveTokens (csrc/quant_paged_cache/lengths.h) of every pair of arguments:
//
//     quant_lengths_test <n> <most> [<n> <most> ...]
#include "quant_paged_cache/lengths.h"

#include <cstdio>
#include <cstdlib>

int main(int argc, char **argv) {
    for (int i = 1; i + 1 < argc; i += 2) {
        std::printf("%lld\n", static_cast<long long>(b200::quant_paged_cache::liveTokens(std::strtoll(argv[i], nullptr, 10), std::strtoll(argv[i + 1], nullptr, 10))));
    }
    return 0;
}
