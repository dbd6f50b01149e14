// scored_index.cc -- mlk_paged_index.h's masks on the host: the positions a token
// sees, against the definition, for random and wrong windows, prefixes and starts.
#include <cstdio>
#include <random>

#include "mlk_paged_index.h"

using namespace mlk;

int main() {
    std::mt19937 rng(7);
    auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    for (int n = 0; n < 20000; ++n) {
        const int32_t len = pick(1, 40), pos = pick(0, len - 1);
        int32_t prefix[3] = {-7, pick(-3, 50), 99}, first[2] = {99, pick(-5, 50)};
        if (n % 100 == 0) prefix[1] = 2147483647;
        if (n % 100 == 1) first[1] = -2147483647 - 1;
        Scores m{nullptr, pick(0, 2) ? prefix : nullptr, pick(0, 2) ? first : nullptr, 0.0f,
                 pick(0, 1) ? pick(1, 45) : 0};
        if (n % 50 == 0) m.window = 1 << 30;
        const Seen v = SeenBy(m, 1, 1, pos, len);
        if (v.lo < 0 || v.hi >= len || v.hi < pos) {
            std::printf("outside: %d..%d of %d\n", v.lo, v.hi, len);
            return 1;
        }
        for (int64_t j = 0; j < len; ++j) {
            bool seen = j <= pos || (m.prefix != nullptr && j < prefix[1] && pos < prefix[1]);
            if (m.window > 0) seen = seen && j > static_cast<int64_t>(pos) - m.window;
            if (m.first != nullptr) seen = seen && j >= first[1];
            if (seen != (j >= v.lo && j <= v.hi)) {
                std::printf("len %d pos %d j %lld: %d..%d\n", len, pos, static_cast<long long>(j), v.lo, v.hi);
                return 1;
            }
        }
    }
    return 0;
}
