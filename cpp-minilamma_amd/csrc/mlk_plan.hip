// mlk_plan.hip -- the pages and token rows of a server's step from its requests'
// lengths, and the pages given back.
//
// Plan: with need_s = ceil((len_s + n_s) / P) - ceil(len_s / P), A and B the
// inclusive sums of need and n over the sequences, s is taken in where (need_s == 0
// or A_s <= free) and B_s <= n_tokens.  Both sums never fall, so what is refused for
// pages is every later sequence that starts one, and what is refused for rows every
// later one with tokens: the pages of those taken in are the stack's first A_s, and
// every sequence knows its own from A_(s-1) alone.  Release: the sum of the pages
// given back says where each goes.
//
// Each is a scan over the sequences by one workgroup, then independent work for
// each token row (or page): which sequence it belongs to (a search in the starts),
// its position and slot.  The row at a page's first position enters it in the
// table; the pages a sequence held before are read there, the new ones popped by
// index, so no row waits for another.  Integer work; what it costs is latency: plan and
// release of 262144 rows of 4096 sequences (4.4 MB, 0.9 us at a copy's rate) take 23.4 to 24.0 us,
// their four kernels 7.9, 5.8, 3.2 and 6.6; of 6 rows of one sequence 9.5, two launches.
#include "mlk_paged.h"

#include <climits>

namespace mlk {
namespace {

constexpr int kPer = 4;  // sequences a thread takes of a step of the scan
constexpr int kRowThreads = 256;
constexpr int64_t kMaxPages = 1 << 30;
// A step of up to kOwnRows rows (or pages) for each of a workgroup's threads is that one
// workgroup's whole work: the smallest of few waves, which wait less for each other (a prompt of
// 6: 3.8 us, with 16 waves 5.5).  A larger one's rows have a launch of their own (8186 rows
// of 256 sequences, in one 6.2 us, in two 8.7 and what lies between two launches).
constexpr int kOwnThreads = 256, kScanThreads = 1024;
constexpr int64_t kOwnRows = 8;
inline bool IsOwn(int threads, int64_t n_seqs, int64_t rows) {
    return n_seqs <= threads * kPer && rows <= threads * kOwnRows;
}

struct Pool {
    int32_t *table, *len, *free_pages, *n_free;
    int64_t table_stride;
    int32_t n_seqs, n_pages, page_shift;
};

struct PlanArgs {
    Pool pool;
    const int32_t* fresh;  // new tokens
    int32_t n_tokens, max_len;
    int32_t *start, *positions, *seq;
    int64_t* slots;
    int32_t* base;  // [n_seqs + 1]: pages popped before each sequence's; last: *n_free before
    bool wide;      // len, fresh and start are 16-byte aligned
    int32_t* err;
};

struct ReleaseArgs {
    Pool pool;
    const int32_t* keep;
    int32_t* before;  // [n_seqs + 2]: pages given back before each sequence's, in all; *n_free
    bool wide;        // len and keep are 16-byte aligned
    int32_t* err;
};

// A thread's kPer neighbouring elements of an array of n, from s on, as one load or store where
// the array is 16-byte aligned (`wide`) and has them all; `none` past its end.
static_assert(kPer == 4, "an int4");
__device__ inline void Load4(const int32_t* p, int s, int n, bool wide, int32_t none, int32_t (&v)[kPer]) {
    if (wide && s + kPer <= n) {
        const int4 x = *reinterpret_cast<const int4*>(p + s);
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
        return;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = s + i < n ? p[s + i] : none;
}
__device__ inline void Store4(int32_t* p, int s, int n, bool wide, const int32_t (&v)[kPer]) {
    if (wide && s + kPer <= n) {
        *reinterpret_cast<int4*>(p + s) = make_int4(v[0], v[1], v[2], v[3]);
        return;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (s + i < n) p[s + i] = v[i];
    }
}

__device__ inline int32_t PagesOf(int64_t len, int32_t shift) {
    return static_cast<int32_t>((len + (int64_t{1} << shift) - 1) >> shift);
}

__device__ inline int32_t FreePages(const Pool& p, bool* bad) {
    const int32_t f = *p.n_free;
    if (f < 0 || f > p.n_pages) *bad = true;
    return f < 0 ? 0 : f > p.n_pages ? p.n_pages : f;
}

// Sums of at most 2^31 - 1, which stands for all beyond.
__device__ inline uint32_t Sum(uint32_t a, uint32_t b) {
    const uint32_t c = a + b;
    return c < 0x7FFFFFFFu ? c : 0x7FFFFFFFu;
}

// Sums over the workgroup's earlier threads; *total: over all.  `scratch` holds a pair a wave and
// is reused after the caller's next barrier.
template <int kThreads>
__device__ inline uint2 ScanBefore(uint2 v, uint2* scratch, uint2* total) {
    constexpr int kWaves = kThreads / kWave;
    const int lane = static_cast<int>(threadIdx.x) % kWave, wave = static_cast<int>(threadIdx.x) / kWave;
    uint2 sum = v;
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) {
        const uint32_t x = __shfl_up(sum.x, off, kWave), y = __shfl_up(sum.y, off, kWave);
        if (lane >= off) sum = make_uint2(Sum(sum.x, x), Sum(sum.y, y));
    }
    if (lane == kWave - 1) scratch[wave] = sum;
    uint2 up = make_uint2(__shfl_up(sum.x, 1, kWave), __shfl_up(sum.y, 1, kWave));
    if (lane == 0) up = make_uint2(0, 0);
    __syncthreads();
    uint2 before = make_uint2(0, 0), all = make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i == wave) before = all;
        all = make_uint2(Sum(all.x, scratch[i].x), Sum(all.y, scratch[i].y));
    }
    *total = all;
    return make_uint2(Sum(before.x, up.x), Sum(before.y, up.y));
}

// Largest s of 0 .. n - 1 with start[s] <= x (start[0] <= x, non-decreasing).
__device__ inline int Find(const int32_t* start, int n, int32_t x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (start[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The same by a whole wave, which looks at 64 places at once: a load for each 64-th part.
__device__ inline int FindByWave(const int32_t* start, int n, int32_t x) {
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    int from = 0;
    for (;;) {
        const int step = (n + kWave - 1) / kWave, at = lane * step;
        const int c = __popcll(__ballot(at < n && start[from + at] <= x));
        from += (c - 1) * step;  // (lane 0's place is one)
        if (step == 1) return __builtin_amdgcn_readfirstlane(from);
        n = n - (c - 1) * step < step ? n - (c - 1) * step : step;
    }
}

// Token row t, the k-th of sequence s, which held `len` positions; its new pages
// are those below the stack's `top`-th.
__device__ inline bool PutRow(const PlanArgs& p, int32_t t, int s, int32_t len, int32_t k, int32_t top) {
    const Pool& o = p.pool;
    const int32_t pos = len + k, j = pos >> o.page_shift, held = PagesOf(len, o.page_shift);
    const int32_t in_page = pos & ((1 << o.page_shift) - 1);
    int32_t* entry = o.table + s * o.table_stride + j;
    int32_t page;
    if (j >= held) {
        page = o.free_pages[top - 1 - (j - held)];
        if (in_page == 0) *entry = page;
    } else {
        page = *entry;
    }
    const bool in = page >= 0 && page < o.n_pages;
    if (p.positions != nullptr) p.positions[t] = pos;
    if (p.seq != nullptr) p.seq[t] = s;
    if (p.slots != nullptr) {
        p.slots[t] = in ? (static_cast<int64_t>(page) << o.page_shift) + in_page : -1;
    }
    return in;
}

template <int kThreads, bool kOwn>
__global__ __launch_bounds__(kThreads) void PlanScan(const PlanArgs p) {
    constexpr int kSeqs = kThreads * kPer;
    __shared__ uint2 sums[2][kThreads / kWave];
    __shared__ int32_t s_start[kOwn ? kSeqs + 1 : 1], s_len[kOwn ? kSeqs : 1], s_base[kOwn ? kSeqs : 1];
    __shared__ uint32_t taken;
    const Pool& o = p.pool;
    const int tid = static_cast<int>(threadIdx.x);
    bool bad = false;
    const int32_t free = FreePages(o, &bad);
    if (tid == 0) taken = 0;
    uint32_t pages = 0, asked = 0, rows = 0;  // of earlier steps of the scan
    for (int s0 = 0; s0 < o.n_seqs; s0 += kSeqs) {
        int32_t len[kPer], n[kPer], need[kPer];
        uint2 mine = make_uint2(0, 0);
        const int my_s = s0 + tid * kPer;
        Load4(o.len, my_s, o.n_seqs, p.wide, 0, len);
        Load4(p.fresh, my_s, o.n_seqs, p.wide, 0, n);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int64_t to = static_cast<int64_t>(len[i]) + n[i];
            need[i] = 0;
            if (len[i] < 0 || n[i] < 0 || to > p.max_len) {
                bad = true;
                n[i] = 0;
            } else {
                need[i] = PagesOf(to, o.page_shift) - PagesOf(len[i], o.page_shift);
            }
            mine = make_uint2(Sum(mine.x, need[i]), Sum(mine.y, n[i]));
        }
        uint2 all;
        const uint2 before = ScanBefore<kThreads>(mine, sums[0], &all);
        uint32_t a = Sum(pages, before.x), b = Sum(asked, before.y), r = b;
        int32_t base[kPer];
        uint32_t my_rows = 0, top = 0;
        bool refused = false;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            base[i] = static_cast<int32_t>(a);
            a = Sum(a, need[i]);
            b = Sum(b, n[i]);
            if ((need[i] != 0 && a > static_cast<uint32_t>(free)) || b > static_cast<uint32_t>(p.n_tokens)) {
                refused |= n[i] != 0;
                n[i] = need[i] = 0;
            }
            if (need[i] != 0) top = a;
            my_rows += n[i];
        }
        if (top != 0) atomicMax(&taken, top);
        // (where all are taken in, here and before, their rows are what was asked for)
        if (__syncthreads_or(refused || rows != asked)) {
            r = rows + ScanBefore<kThreads>(make_uint2(my_rows, 0), sums[1], &mine).x;
            rows += mine.x;
        } else {
            rows = Sum(rows, all.y);
        }
        int32_t start[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            start[i] = static_cast<int32_t>(r);
            r += n[i];
            if constexpr (kOwn) {
                s_start[my_s + i] = start[i];
                s_len[my_s + i] = len[i];
                s_base[my_s + i] = base[i];
            }
            len[i] += n[i];
        }
        Store4(p.start, my_s, o.n_seqs, p.wide, start);
        Store4(o.len, my_s, o.n_seqs, p.wide, len);
        if constexpr (!kOwn) Store4(p.base, my_s, o.n_seqs, true, base);
        pages = Sum(pages, all.x);
        asked = Sum(asked, all.y);
        __syncthreads();
    }
    if (tid == 0) {
        p.start[o.n_seqs] = static_cast<int32_t>(rows);
        *o.n_free = free - static_cast<int32_t>(taken);
        if constexpr (!kOwn) p.base[o.n_seqs] = free;
    }
    if constexpr (kOwn) {
        for (int t = tid; t < static_cast<int>(rows); t += kThreads) {
            const int s = Find(s_start, o.n_seqs, t);
            if (!PutRow(p, t, s, s_len[s], t - s_start[s], free - s_base[s])) bad = true;
        }
    }
    if (bad) RaiseFlag(p.err, 1);
}

// Token rows of a step, one a thread; the starts of as many sequences from its first row's on
// lie in shared memory.
__global__ __launch_bounds__(kRowThreads) void PlanRows(const PlanArgs p) {
    __shared__ int32_t s_start[kRowThreads + 1];
    const Pool& o = p.pool;
    const int tid = static_cast<int>(threadIdx.x);
    const int32_t t0 = static_cast<int32_t>(blockIdx.x) * kRowThreads, t = t0 + tid;
    const int32_t rows = p.start[o.n_seqs], free = p.base[o.n_seqs];
    if (t0 >= rows) return;
    const int first = FindByWave(p.start, o.n_seqs, t0);
    const int here = o.n_seqs - first < kRowThreads ? o.n_seqs - first : kRowThreads;
    for (int i = tid; i <= here; i += kRowThreads) s_start[i] = p.start[first + i];
    __syncthreads();
    if (t >= rows) return;
    // (sequences without rows can lie between: then it is further on)
    int s;
    int32_t from, to;
    if (t < s_start[here]) {
        const int i = Find(s_start, here, t);
        s = first + i;
        from = s_start[i];
        to = s_start[i + 1];
    } else {
        s = first + here + Find(p.start + first + here, o.n_seqs - first - here, t);
        from = p.start[s];
        to = p.start[s + 1];
    }
    if (!PutRow(p, t, s, o.len[s] - (to - from), t - from, free - p.base[s])) RaiseFlag(p.err, 1);
}

// The i-th of `total` pages given back, sequence s's k-th; `kept` pages stay.
// (An entry that is no page goes back too: every page has its place by the lengths alone.)
__device__ inline bool PutPage(const ReleaseArgs& p, int32_t i, int s, int32_t kept, int32_t k,
                               int32_t free, int32_t total) {
    const Pool& o = p.pool;
    int32_t* entry = o.table + s * o.table_stride + kept + k;
    const int32_t page = *entry;
    const int64_t at = static_cast<int64_t>(free) + total - 1 - i;
    *entry = -1;
    if (at < o.n_pages) o.free_pages[at] = page;
    return at < o.n_pages && page >= 0 && page < o.n_pages;
}

template <int kThreads, bool kOwn>
__global__ __launch_bounds__(kThreads) void ReleaseScan(const ReleaseArgs p) {
    constexpr int kSeqs = kThreads * kPer;
    __shared__ uint2 sums[kThreads / kWave];
    __shared__ int32_t s_before[kOwn ? kSeqs : 1], s_kept[kOwn ? kSeqs : 1];
    const Pool& o = p.pool;
    const int tid = static_cast<int>(threadIdx.x);
    bool bad = false;
    const int32_t free = FreePages(o, &bad);
    uint32_t pages = 0;
    for (int s0 = 0; s0 < o.n_seqs; s0 += kSeqs) {
        int32_t gone[kPer], kept[kPer], keep[kPer], len[kPer];
        uint32_t mine = 0;
        const int my_s = s0 + tid * kPer;
        Load4(p.keep, my_s, o.n_seqs, p.wide, -1, keep);
        Load4(o.len, my_s, o.n_seqs, p.wide, 0, len);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            gone[i] = kept[i] = 0;
            if (keep[i] >= 0) {
                if (keep[i] > len[i] || len[i] > o.table_stride << o.page_shift) {
                    bad = true;
                } else {
                    kept[i] = PagesOf(keep[i], o.page_shift);
                    gone[i] = PagesOf(len[i], o.page_shift) - kept[i];
                    len[i] = keep[i];
                }
            }
            mine += gone[i];
        }
        uint2 all;
        uint32_t at = pages + ScanBefore<kThreads>(make_uint2(mine, 0), sums, &all).x;
        int32_t before[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            before[i] = static_cast<int32_t>(at);
            at += gone[i];
            if constexpr (kOwn) {
                s_before[my_s + i] = before[i];
                s_kept[my_s + i] = kept[i];
            }
        }
        Store4(o.len, my_s, o.n_seqs, p.wide, len);
        if constexpr (!kOwn) Store4(p.before, my_s, o.n_seqs, true, before);
        pages += all.x;
        __syncthreads();
    }
    const int32_t total = static_cast<int32_t>(pages);
    if (tid == 0) {
        const int64_t now = static_cast<int64_t>(free) + total;
        *o.n_free = now < o.n_pages ? static_cast<int32_t>(now) : o.n_pages;
        if constexpr (!kOwn) {
            p.before[o.n_seqs] = total;
            p.before[o.n_seqs + 1] = free;
        }
    }
    if constexpr (kOwn) {
        for (int i = tid; i < total; i += kThreads) {
            const int s = Find(s_before, o.n_seqs, i);
            if (!PutPage(p, i, s, s_kept[s], i - s_before[s], free, total)) bad = true;
        }
    }
    if (bad) RaiseFlag(p.err, 1);
}

// Pages given back, one a thread at a time; the sums of as many sequences from the first page's
// on lie in shared memory.
__global__ __launch_bounds__(kRowThreads) void ReleasePages(const ReleaseArgs p) {
    __shared__ int32_t s_before[kRowThreads];
    const Pool& o = p.pool;
    const int tid = static_cast<int>(threadIdx.x);
    const int32_t total = p.before[o.n_seqs], free = p.before[o.n_seqs + 1];
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRowThreads;
    bool bad = false;
    for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * kRowThreads; i0 < total; i0 += step) {
        const int first = FindByWave(p.before, o.n_seqs, static_cast<int32_t>(i0));
        const int here = o.n_seqs - first < kRowThreads ? o.n_seqs - first : kRowThreads;
        __syncthreads();
        if (tid < here) s_before[tid] = p.before[first + tid];
        __syncthreads();
        const int64_t i = i0 + tid;
        if (i >= total) continue;
        const int32_t x = static_cast<int32_t>(i);
        const int at = Find(s_before, here, x);
        int s = first + at;
        int32_t before = s_before[at];
        if (at == here - 1) {  // (sequences that gave none back can lie between: then further on)
            s += Find(p.before + s, o.n_seqs - s, x);
            before = p.before[s];
        }
        // (a sequence that gave pages back now has the length it kept)
        if (!PutPage(p, x, s, PagesOf(o.len[s], o.page_shift), x - before, free, total)) bad = true;
    }
    if (bad) RaiseFlag(p.err, 1);
}

mlk_status CheckPool(const char* fn, const mlk_paged_pool* pool, Pool* out) {
    if (pool == nullptr) return Fail(MLK_ERR_INVALID, "%s: pool must not be null", fn);
    const mlk_paged_pool& p = *pool;
    const void* ptrs[4] = {p.page_table, p.seq_len, p.free_pages, p.n_free};
    for (int i = 0; i < 4; ++i) {
        if (ptrs[i] == nullptr || !Aligned(ptrs[i], 4)) {
            return Fail(MLK_ERR_INVALID, "%s: page_table, seq_len, free_pages and n_free must be "
                                         "4-byte aligned device arrays", fn);
        }
        for (int j = 0; j < i; ++j) {
            if (ptrs[i] == ptrs[j]) return Fail(MLK_ERR_INVALID, "%s: the pool's arrays must be distinct", fn);
        }
    }
    if (p.page_size < 1 || (p.page_size & (p.page_size - 1)) != 0) {
        return Fail(MLK_ERR_INVALID, "%s: page_size must be a power of two", fn);
    }
    if (p.n_pages < 1 || p.n_pages > kMaxPages) {
        return Fail(MLK_ERR_INVALID, "%s: n_pages must be in 1..2^30", fn);
    }
    if (p.n_seqs < 0 || p.n_seqs > kMaxSeqs) {
        return Fail(MLK_ERR_INVALID, "%s: n_seqs must be in 0..2^20", fn);
    }
    if (p.table_stride < 1 || p.table_stride > INT32_MAX || p.table_stride * p.n_seqs > INT32_MAX) {
        return Fail(MLK_ERR_INVALID, "%s: table_stride must be positive and the table have fewer "
                                     "than 2^31 entries", fn);
    }
    *out = {p.page_table, p.seq_len, p.free_pages, p.n_free, p.table_stride,
            static_cast<int32_t>(p.n_seqs), static_cast<int32_t>(p.n_pages),
            __builtin_ctz(static_cast<unsigned>(p.page_size))};
    return MLK_OK;
}

mlk_status CheckWorkspace(const char* fn, const void* ws, size_t bytes, int64_t n_seqs) {
    if (ws == nullptr || !Aligned(ws, 16)) {
        return Fail(MLK_ERR_INVALID, "%s: workspace must be a 16-byte aligned device buffer", fn);
    }
    const int64_t need = mlk_paged_plan_workspace_bytes(n_seqs);
    if (bytes < static_cast<size_t>(need)) {
        return Fail(MLK_ERR_INVALID, "%s: workspace of %zu bytes, %lld are needed", fn, bytes,
                    static_cast<long long>(need));
    }
    return MLK_OK;
}

}  // namespace
}  // namespace mlk

using namespace mlk;

extern "C" {

int64_t mlk_paged_plan_workspace_bytes(int64_t n_seqs) {
    if (n_seqs <= 0 || n_seqs > kMaxSeqs) return 0;
    return (4 * (n_seqs + 2) + 15) / 16 * 16;
}

mlk_status mlk_paged_plan(const mlk_paged_pool* pool, const int32_t* new_tokens, int64_t n_tokens,
                          int64_t max_seq_len, int32_t* token_start, int32_t* positions,
                          int32_t* token_seq, int64_t* slots, void* workspace,
                          size_t workspace_bytes, int32_t* err, void* stream) {
    const char* fn = "mlk_paged_plan";
    PlanArgs p{};
    mlk_status st = CheckPool(fn, pool, &p.pool);
    if (st != MLK_OK) return st;
    if (n_tokens < 0 || n_tokens > kMaxTokens) {
        return Fail(MLK_ERR_INVALID, "%s: n_tokens must be in 0..2^23", fn);
    }
    if (max_seq_len < 1 || max_seq_len > (1 << 30) ||
        max_seq_len > pool->table_stride * pool->page_size) {
        return Fail(MLK_ERR_INVALID, "%s: max_seq_len must be in 1..2^30 and at most table_stride "
                                     "* page_size", fn);
    }
    // (no sequences: of the outputs only token_start[0] is written, where it is given)
    const bool none = pool->n_seqs == 0;
    if (none && token_start == nullptr) return MLK_OK;
    if ((new_tokens == nullptr && !none) || token_start == nullptr || !Aligned(new_tokens, 4) ||
        !Aligned(token_start, 4) || !Aligned(positions, 4) || !Aligned(token_seq, 4)) {
        return Fail(MLK_ERR_INVALID, "%s: new_tokens and token_start must be 4-byte aligned device "
                                     "arrays, as positions and token_seq where given", fn);
    }
    if (!Aligned(slots, 8)) return Fail(MLK_ERR_INVALID, "%s: slots must be 8-byte aligned", fn);
    const void* outs[4] = {token_start, positions, token_seq, slots};
    const void* ins[5] = {pool->page_table, pool->seq_len, pool->free_pages, pool->n_free, new_tokens};
    for (int i = 0; i < 4; ++i) {
        bool same = false;
        for (int j = 0; j < 5; ++j) same |= outs[i] != nullptr && outs[i] == ins[j];
        for (int j = 0; j < i; ++j) same |= outs[i] != nullptr && outs[i] == outs[j];
        if (same) return Fail(MLK_ERR_INVALID, "%s: an output may not alias another or the pool", fn);
    }
    if (new_tokens == pool->seq_len) return Fail(MLK_ERR_INVALID, "%s: new_tokens may not alias seq_len", fn);
    if (!none) st = CheckWorkspace(fn, workspace, workspace_bytes, pool->n_seqs);
    if (st != MLK_OK) return st;
    p.fresh = new_tokens;
    p.n_tokens = static_cast<int32_t>(n_tokens);
    p.max_len = static_cast<int32_t>(max_seq_len);
    p.start = token_start;
    p.positions = positions;
    p.seq = token_seq;
    p.slots = slots;
    p.base = static_cast<int32_t*>(workspace);
    p.wide = Aligned(pool->seq_len, 16) && Aligned(new_tokens, 16) && Aligned(token_start, 16);
    p.err = err;
    const hipStream_t s = AsStream(stream);
    if (none || IsOwn(kOwnThreads, p.pool.n_seqs, n_tokens)) {
        hipLaunchKernelGGL((PlanScan<kOwnThreads, true>), dim3(1), dim3(kOwnThreads), 0, s, p);
        return CheckLaunch("PlanScan");
    }
    if (IsOwn(kScanThreads, p.pool.n_seqs, n_tokens)) {
        hipLaunchKernelGGL((PlanScan<kScanThreads, true>), dim3(1), dim3(kScanThreads), 0, s, p);
        return CheckLaunch("PlanScan");
    }
    hipLaunchKernelGGL((PlanScan<kScanThreads, false>), dim3(1), dim3(kScanThreads), 0, s, p);
    st = CheckLaunch("PlanScan");
    if (st != MLK_OK || n_tokens == 0) return st;
    const dim3 grid(static_cast<unsigned>((n_tokens + kRowThreads - 1) / kRowThreads));
    hipLaunchKernelGGL(PlanRows, grid, dim3(kRowThreads), 0, s, p);
    return CheckLaunch("PlanRows");
}

mlk_status mlk_paged_release(const mlk_paged_pool* pool, const int32_t* keep, void* workspace,
                             size_t workspace_bytes, int32_t* err, void* stream) {
    const char* fn = "mlk_paged_release";
    ReleaseArgs p{};
    mlk_status st = CheckPool(fn, pool, &p.pool);
    if (st != MLK_OK) return st;
    if (pool->n_seqs == 0) return MLK_OK;
    if (keep == nullptr || !Aligned(keep, 4)) {
        return Fail(MLK_ERR_INVALID, "%s: keep must be a 4-byte aligned device array", fn);
    }
    if (keep == pool->seq_len || keep == pool->page_table || keep == pool->free_pages || keep == pool->n_free) {
        return Fail(MLK_ERR_INVALID, "%s: keep may not alias the pool", fn);
    }
    st = CheckWorkspace(fn, workspace, workspace_bytes, pool->n_seqs);
    if (st != MLK_OK) return st;
    p.keep = keep;
    p.before = static_cast<int32_t*>(workspace);
    p.wide = Aligned(pool->seq_len, 16) && Aligned(keep, 16);
    p.err = err;
    const hipStream_t s = AsStream(stream);
    // pages that can come back at once
    const int64_t entries = pool->n_seqs * pool->table_stride;
    const int64_t most = entries < pool->n_pages ? entries : pool->n_pages;
    if (IsOwn(kOwnThreads, p.pool.n_seqs, most)) {
        hipLaunchKernelGGL((ReleaseScan<kOwnThreads, true>), dim3(1), dim3(kOwnThreads), 0, s, p);
        return CheckLaunch("ReleaseScan");
    }
    if (IsOwn(kScanThreads, p.pool.n_seqs, most)) {
        hipLaunchKernelGGL((ReleaseScan<kScanThreads, true>), dim3(1), dim3(kScanThreads), 0, s, p);
        return CheckLaunch("ReleaseScan");
    }
    hipLaunchKernelGGL((ReleaseScan<kScanThreads, false>), dim3(1), dim3(kScanThreads), 0, s, p);
    st = CheckLaunch("ReleaseScan");
    if (st != MLK_OK) return st;
    hipLaunchKernelGGL(ReleasePages, dim3(GridFor(most, kRowThreads, 8)), dim3(kRowThreads), 0, s, p);
    return CheckLaunch("ReleasePages");
}

}  // extern "C"
