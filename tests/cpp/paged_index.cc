// Host run of the index arithmetic that the paged kernels use
// (mlk_paged_index.h): what it accepts stays inside the buffers, and what is
// wrong is refused or clamped.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "mlk_paged_index.h"

namespace {
void Check(bool ok, const char* what) {
    if (!ok) {
        std::printf("FAILED: %s\n", what);
        std::exit(1);
    }
}
}  // namespace

int main() {
    std::mt19937 rng(1);
    auto pick = [&](int64_t lo, int64_t hi) {
        return std::uniform_int_distribution<int64_t>(lo, hi)(rng);
    };
    for (int round = 0; round < 20000; ++round) {
        const int n_seqs = static_cast<int>(pick(1, 9));
        const int shift = static_cast<int>(pick(0, 6));
        const int64_t stride = pick(1, 12);
        const int32_t cap = static_cast<int32_t>(stride << shift);
        mlk::Ragged r{};
        r.n_seqs = n_seqs;
        r.n_tokens = static_cast<int32_t>(pick(1, 200));
        r.max_new = static_cast<int32_t>(pick(1, 60));
        r.max_len = static_cast<int32_t>(pick(1, cap));
        r.table_stride = stride;
        const bool wild = round % 2;
        std::vector<int32_t> start(n_seqs + 1), len(n_seqs), table(n_seqs * stride);
        for (int s = 0; s <= n_seqs; ++s) {
            start[s] = wild ? static_cast<int32_t>(pick(INT32_MIN, INT32_MAX))
                            : (s ? start[s - 1] : 0) + static_cast<int32_t>(pick(0, 30));
        }
        for (auto& v : len) v = static_cast<int32_t>(wild ? pick(INT32_MIN, INT32_MAX) : pick(0, 99));
        for (auto& v : table) v = static_cast<int32_t>(wild ? pick(INT32_MIN, INT32_MAX) : pick(-2, 12));
        r.start = start.data();
        r.len = len.data();
        r.table = table.data();
        mlk::RowsAt at{};
        at.page_shift = shift;
        at.n_pages = 10;
        at.k_row = at.v_row = 24;
        at.page_stride = (int64_t{24} << shift) + 5;
        for (int s = 0; s < n_seqs; ++s) {
            mlk::Seq q{};
            const bool ok = mlk::LoadSeq(r, s, &q);
            const int64_t a = start[s], n = int64_t{start[s + 1]} - a;
            const bool want = a >= 0 && n >= 0 && a + n <= r.n_tokens && n <= r.max_new &&
                              n <= len[s] && len[s] <= r.max_len;
            Check(ok == want, "LoadSeq accepts exactly the sequences within the bounds");
            if (!ok) continue;
            Check(q.t0 == a && q.n == n && q.len == len[s], "LoadSeq's values");
            for (int32_t j = 0; j < q.len; ++j) {
                bool bad = false;
                const int32_t g = mlk::PageOf(at, table.data() + s * stride, j, &bad);
                const int32_t raw = table[s * stride + (j >> shift)];
                Check(bad == (raw < 0 || raw >= 10) && g == (bad ? 0 : raw), "PageOf");
                const int64_t o = mlk::PagedRow(at, g, j);
                Check(o >= 0 && o + 24 <= 9 * at.page_stride + (int64_t{24} << shift), "PagedRow");
            }
        }
    }
    std::printf("ok\n");
    return 0;
}
