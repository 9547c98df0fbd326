// Range and share lengths of attention over a cache (csrc/attention_cache_ranges.h) on the
// host, for sums as batches make them: one line a case. Compiled twice by its test, with
// products and sums contracted wherever the compiler may and without: the lines have to be
// the same, as the kernels that each work a length out have to come to the same one.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>
#include <random>

#include "attention_cache_ranges.h"

int main() {
    std::mt19937_64 rng(7);
    const auto log_uniform = [&](double lo, double hi) {
        return lo * std::exp(std::uniform_real_distribution<double>(0, std::log(hi / lo))(rng));
    };
    uint64_t hash = 1469598103934665603ull;
    for (int i = 0; i < 2000000; ++i) {
        const int rows = i % 3 == 0 ? 16 : i % 3 == 1 ? 32 : 128;
        const int seqs = static_cast<int>(log_uniform(1, 64));
        qimg::RangeSums s = {0.0f, 0.0f, 0.0f, 1, 0};
        for (int b = 0; b < seqs; ++b) {
            const int tiles = static_cast<int>(log_uniform(1, 3000)), n = static_cast<int>(log_uniform(1, 200000));
            const int fewer = i & 1 ? static_cast<int>(log_uniform(1, n + 1)) : 0;
            s.work += qimg::seen_steps(static_cast<float>(tiles), n, fewer);
            s.all += qimg::seen_steps(static_cast<float>(tiles), n, 0);
            s.tiles += static_cast<float>(tiles);
            s.longest = n > s.longest ? n : s.longest;
        }
        s.least = (s.longest + 31) / 32;
        qimg::times_heads(s, 1 + i % 7);
        const int len = rows == 128 ? qimg::share_length(s, i & 1) : qimg::few_length(s, rows);
        const bool pays = qimg::shares_pay(s.all / 512, s.tiles, s.work / 300);
        hash = (hash ^ static_cast<uint32_t>(len) ^ (pays ? 1ull << 40 : 0)) * 1099511628211ull;
        if (i % 1000 == 999) std::printf("%016llx\n", static_cast<unsigned long long>(hash));
    }
    return 0;
}
