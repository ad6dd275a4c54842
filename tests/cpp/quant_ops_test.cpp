// The C++ wrappers of the operators over quantised pools, on inputs a Python test wrote:
//
//     quant_ops_test <dir> <bits> <tokens> <kv_heads> <head> <blocks> <block> <seqs> <heads> <max_blocks>
//
// reads k, v, slots, q, tables, lens (raw bytes, .bin), writes the rows into zeroed pools, reads them back as F32, attends, does
// all of it a second time from the descriptor cache, and writes k_back, v_back and out (.out.bin).
#include "infinicore_b200/ops.hpp"

#include <cstdio>
#include <cstdlib>
#include <fstream>
#include <iterator>
#include <string>
#include <vector>

namespace ib = infinicore_b200;

namespace {

std::string g_dir;

void *upload(const std::vector<char> &host) {
    void *p = nullptr;
    ib::check(infinirtMalloc(&p, host.size()), "infinirtMalloc");
    ib::check(infinirtMemcpy(p, host.data(), host.size(), INFINIRT_MEMCPY_H2D), "infinirtMemcpy");
    return p;
}

ib::Tensor load(const char *name, infiniDtype_t dtype, std::vector<size_t> shape) {
    std::ifstream in(g_dir + "/" + name + ".bin", std::ios::binary);
    std::vector<char> host((std::istreambuf_iterator<char>(in)), std::istreambuf_iterator<char>());
    return ib::Tensor(upload(host), dtype, std::move(shape));
}

ib::Tensor zeros(infiniDtype_t dtype, size_t elem, std::vector<size_t> shape) {
    size_t n = elem;
    for (size_t d : shape) {
        n *= d;
    }
    return ib::Tensor(upload(std::vector<char>(n, 0)), dtype, std::move(shape));
}

void save(const char *name, const ib::Tensor &t, size_t elem) {
    size_t n = elem;
    for (size_t d : t.shape) {
        n *= d;
    }
    std::vector<char> host(n);
    ib::check(infinirtMemcpy(host.data(), t.data, n, INFINIRT_MEMCPY_D2H), "infinirtMemcpy");
    std::ofstream(g_dir + "/" + name + ".out.bin", std::ios::binary).write(host.data(), static_cast<std::streamsize>(n));
}

} // namespace

int main(int argc, char **argv) {
    if (argc != 11) {
        std::fprintf(stderr, "usage: quant_ops_test dir bits tokens kv_heads head blocks block seqs heads max_blocks\n");
        return 2;
    }
    g_dir = argv[1];
    size_t n[9];
    for (int i = 0; i < 9; ++i) {
        n[i] = std::strtoull(argv[2 + i], nullptr, 10);
    }
    const size_t bits = n[0], tokens = n[1], kvh = n[2], hd = n[3], blocks = n[4], bs = n[5], seqs = n[6], heads = n[7], width = n[8];
    try {
        ib::check(infinirtSetDevice(INFINI_DEVICE_NVIDIA, 0), "infinirtSetDevice");
        const infiniDtype_t codes = bits == 8 ? INFINI_DTYPE_I8 : INFINI_DTYPE_U8;
        const std::vector<size_t> cache = {blocks, kvh, bs, bits == 8 ? hd : hd / 2}, scales = {blocks, kvh, bs, bits == 8 ? 1 : hd / 32};
        const ib::op::QuantPools pools = {zeros(codes, 1, cache), zeros(codes, 1, cache), zeros(INFINI_DTYPE_BF16, 2, scales),
                                          zeros(INFINI_DTYPE_BF16, 2, scales)};
        const ib::Tensor k = load("k", INFINI_DTYPE_BF16, {tokens, kvh, hd}), v = load("v", INFINI_DTYPE_BF16, {tokens, kvh, hd});
        const ib::Tensor slots = load("slots", INFINI_DTYPE_I64, {tokens});
        const ib::Tensor q = load("q", INFINI_DTYPE_BF16, {seqs, heads, hd});
        const ib::Tensor tables = load("tables", INFINI_DTYPE_I64, {seqs, width}), lens = load("lens", INFINI_DTYPE_I64, {seqs});
        const ib::Tensor k_back = zeros(INFINI_DTYPE_F32, 4, {tokens, kvh, hd}), v_back = zeros(INFINI_DTYPE_F32, 4, {tokens, kvh, hd});
        const ib::Tensor out = zeros(INFINI_DTYPE_BF16, 2, {seqs, heads, hd});
        for (int turn = 0; turn < 2; ++turn) {
            ib::op::quant_paged_caching_(pools, k, v, slots);
            ib::op::quant_paged_cache_read_(k_back, v_back, pools, slots);
            ib::op::quant_paged_attention_(out, q, pools, tables, lens, std::nullopt, 0.1f);
        }
        const ib::CacheStats stats = ib::cache_stats();
        if (stats.misses != 3 || stats.hits != 3) {
            std::fprintf(stderr, "descriptor cache: %zu misses, %zu hits\n", stats.misses, stats.hits);
            return 1;
        }
        bool refused = false;
        try {
            ib::op::quant_paged_caching_(pools, k_back, v, slots);
        } catch (const ib::StatusError &e) {
            refused = e.status == INFINI_STATUS_BAD_TENSOR_DTYPE;
        }
        if (!refused || ib::kernel_status() != 0) {
            std::fprintf(stderr, "a bad dtype was not refused, or a kernel raised a flag\n");
            return 1;
        }
        save("k_back", k_back, 4);
        save("v_back", v_back, 4);
        save("out", out, 2);
    } catch (const std::exception &e) {
        std::fprintf(stderr, "%s\n", e.what());
        return 1;
    }
    return 0;
}
