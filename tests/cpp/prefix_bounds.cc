// prefix_bounds.cc -- mlk_paged_index.h's SeenBy on the host for prefix lengths of any value
// at all: what a token sees stays within its sequence and is what the definition says.
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "mlk_paged_index.h"

using namespace mlk;

int main() {
    const int32_t low = INT32_MIN, high = INT32_MAX;
    const int32_t prefixes[] = {low, low + 1, low / 2, -9, -1, 0, 1, 2, 16, 39, 40, 41, 1 << 30, high - 1, high};
    const int32_t lens[] = {1, 2, 17, 40, 1 << 30};
    for (const int32_t len : lens) {
        const int32_t places[] = {0, len / 2, len - 1};
        for (const int32_t pos : places) {
            for (const int32_t prefix : prefixes) {
                for (const int32_t window : {0, 1, 5, 1 << 30}) {
                    const Scores m{nullptr, &prefix, nullptr, 0.0f, window};
                    const Seen v = SeenBy(m, 0, 0, pos, len);
                    const int64_t lo = window > 0 && pos - int64_t{window} + 1 > 0 ? pos - int64_t{window} + 1 : 0;
                    const int64_t end = prefix < len ? prefix : len;
                    const int64_t hi = end - 1 > pos ? end - 1 : pos;
                    if (v.lo != lo || v.hi != hi || v.hi >= len) {
                        std::printf("len %d pos %d prefix %d window %d: %d..%d, not %lld..%lld\n", len, pos, prefix, window,
                                    v.lo, v.hi, static_cast<long long>(lo), static_cast<long long>(hi));
                        return 1;
                    }
                }
            }
        }
    }
    return 0;
}
