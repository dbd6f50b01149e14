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
// index, so no row waits for another.  Integer work; what it costs is latency.
#include "mlk_paged.h"

#include <climits>

namespace mlk {
namespace {

constexpr int kScanThreads = 1024, kPer = 4;        // sequences a thread takes
constexpr int kScanSeqs = kScanThreads * kPer;      // of a step of the scan
constexpr int kRowThreads = 256, kRowsEach = 1024;  // rows of a workgroup
constexpr int64_t kMaxPages = 1 << 30;
// Rows that the scanning workgroup works out itself, without a second launch.
constexpr int64_t kOwnRows = 16384;

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
    int32_t* err;
};

struct ReleaseArgs {
    Pool pool;
    const int32_t* keep;
    int32_t* before;  // [n_seqs + 2]: pages given back before each sequence's, in all; *n_free
    int32_t* err;
};

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

// Sum over the workgroup's earlier threads; *total: over all.  `scratch` is reused
// after the caller's next barrier.
__device__ inline uint32_t ScanBefore(uint32_t v, uint32_t* scratch, uint32_t* total) {
    constexpr int kWaves = kScanThreads / kWave;
    const int lane = static_cast<int>(threadIdx.x) % kWave, wave = static_cast<int>(threadIdx.x) / kWave;
    uint32_t sum = v;
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) {
        const uint32_t o = __shfl_up(sum, off, kWave);
        if (lane >= off) sum = Sum(sum, o);
    }
    if (lane == kWave - 1) scratch[wave] = sum;
    uint32_t up = __shfl_up(sum, 1, kWave);
    if (lane == 0) up = 0;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i == wave) before = all;
        all = Sum(all, scratch[i]);
    }
    *total = all;
    return Sum(before, up);
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

template <bool kOwn>
__global__ __launch_bounds__(kScanThreads) void PlanScan(const PlanArgs p) {
    __shared__ uint32_t sums[3][kScanThreads / kWave];
    __shared__ int32_t s_start[kOwn ? kScanSeqs + 1 : 1], s_len[kOwn ? kScanSeqs : 1],
        s_base[kOwn ? kScanSeqs : 1];
    __shared__ uint32_t taken;
    const Pool& o = p.pool;
    const int tid = static_cast<int>(threadIdx.x);
    bool bad = false;
    const int32_t free = FreePages(o, &bad);
    if (tid == 0) taken = 0;
    uint32_t pages = 0, asked = 0, rows = 0;  // of earlier steps of the scan
    for (int s0 = 0; s0 < o.n_seqs; s0 += kScanSeqs) {
        int32_t len[kPer], n[kPer], need[kPer];
        uint32_t my_pages = 0, my_asked = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int s = s0 + tid * kPer + i;
            len[i] = n[i] = need[i] = 0;
            if (s < o.n_seqs) {
                len[i] = o.len[s];
                n[i] = p.fresh[s];
            }
            const int64_t to = static_cast<int64_t>(len[i]) + n[i];
            if (len[i] < 0 || n[i] < 0 || to > p.max_len) {
                bad = true;
                n[i] = 0;
            } else {
                need[i] = PagesOf(to, o.page_shift) - PagesOf(len[i], o.page_shift);
            }
            my_pages = Sum(my_pages, need[i]);
            my_asked = Sum(my_asked, n[i]);
        }
        uint32_t all_pages, all_asked, all_rows;
        uint32_t a = Sum(pages, ScanBefore(my_pages, sums[0], &all_pages));
        uint32_t b = Sum(asked, ScanBefore(my_asked, sums[1], &all_asked));
        int32_t base[kPer];
        uint32_t my_rows = 0, top = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            base[i] = static_cast<int32_t>(a);
            a = Sum(a, need[i]);
            b = Sum(b, n[i]);
            if ((need[i] != 0 && a > static_cast<uint32_t>(free)) || b > static_cast<uint32_t>(p.n_tokens)) {
                n[i] = need[i] = 0;
            }
            if (need[i] != 0) top = a;
            my_rows += n[i];
        }
        if (top != 0) atomicMax(&taken, top);
        uint32_t r = rows + ScanBefore(my_rows, sums[2], &all_rows);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int s = s0 + tid * kPer + i;
            if (s < o.n_seqs) {
                p.start[s] = static_cast<int32_t>(r);
                if (n[i] != 0) o.len[s] = len[i] + n[i];
                if constexpr (kOwn) {
                    s_start[s] = static_cast<int32_t>(r);
                    s_len[s] = len[i];
                    s_base[s] = base[i];
                } else {
                    p.base[s] = base[i];
                }
            }
            r += n[i];
        }
        pages = Sum(pages, all_pages);
        asked = Sum(asked, all_asked);
        rows += all_rows;
        __syncthreads();
    }
    if (tid == 0) {
        p.start[o.n_seqs] = static_cast<int32_t>(rows);
        *o.n_free = free - static_cast<int32_t>(taken);
        if constexpr (!kOwn) p.base[o.n_seqs] = free;
    }
    if constexpr (kOwn) {
        for (int t = tid; t < static_cast<int>(rows); t += kScanThreads) {
            const int s = Find(s_start, o.n_seqs, t);
            if (!PutRow(p, t, s, s_len[s], t - s_start[s], free - s_base[s])) bad = true;
        }
    }
    if (bad) RaiseFlag(p.err, 1);
}

// Token rows of a step, kRowsEach a workgroup; the starts of as many sequences from
// its first row's on lie in shared memory.
__global__ __launch_bounds__(kRowThreads) void PlanRows(const PlanArgs p) {
    __shared__ int32_t s_start[kRowsEach + 1];
    const Pool& o = p.pool;
    const int tid = static_cast<int>(threadIdx.x);
    const int32_t t0 = static_cast<int32_t>(blockIdx.x) * kRowsEach, rows = p.start[o.n_seqs];
    if (t0 >= rows) return;
    const int first = Find(p.start, o.n_seqs, t0);
    const int here = o.n_seqs - first < kRowsEach ? o.n_seqs - first : kRowsEach;
    for (int i = tid; i <= here; i += kRowThreads) s_start[i] = p.start[first + i];
    __syncthreads();
    const int32_t free = p.base[o.n_seqs];
    bool bad = false;
    for (int i = tid; i < kRowsEach && t0 + i < rows; i += kRowThreads) {
        const int32_t t = t0 + i;
        // (sequences without rows can lie between: then it is further on)
        const int s = t < s_start[here] ? first + Find(s_start, here, t)
                                        : first + here + Find(p.start + first + here, o.n_seqs - first - here, t);
        const int32_t from = p.start[s], len = o.len[s] - (p.start[s + 1] - from);
        if (!PutRow(p, t, s, len, t - from, free - p.base[s])) bad = true;
    }
    if (bad) RaiseFlag(p.err, 1);
}

// The i-th of `total` pages given back, sequence s's k-th; `kept` pages stay.
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

template <bool kOwn>
__global__ __launch_bounds__(kScanThreads) void ReleaseScan(const ReleaseArgs p) {
    __shared__ uint32_t sums[kScanThreads / kWave];
    __shared__ int32_t s_before[kOwn ? kScanSeqs : 1], s_kept[kOwn ? kScanSeqs : 1];
    const Pool& o = p.pool;
    const int tid = static_cast<int>(threadIdx.x);
    bool bad = false;
    const int32_t free = FreePages(o, &bad);
    uint32_t pages = 0;
    for (int s0 = 0; s0 < o.n_seqs; s0 += kScanSeqs) {
        int32_t gone[kPer], kept[kPer];
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int s = s0 + tid * kPer + i;
            gone[i] = kept[i] = 0;
            if (s < o.n_seqs) {
                const int32_t keep = p.keep[s], len = o.len[s];
                if (keep >= 0) {
                    if (keep > len || len > o.table_stride << o.page_shift) {
                        bad = true;
                    } else {
                        kept[i] = PagesOf(keep, o.page_shift);
                        gone[i] = PagesOf(len, o.page_shift) - kept[i];
                        o.len[s] = keep;
                    }
                }
            }
            mine += gone[i];
        }
        uint32_t all, at = pages + ScanBefore(mine, sums, &all);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int s = s0 + tid * kPer + i;
            if (s < o.n_seqs) {
                if constexpr (kOwn) {
                    s_before[s] = static_cast<int32_t>(at);
                    s_kept[s] = kept[i];
                } else {
                    p.before[s] = static_cast<int32_t>(at);
                }
            }
            at += gone[i];
        }
        pages += all;
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
        for (int i = tid; i < total; i += kScanThreads) {
            const int s = Find(s_before, o.n_seqs, i);
            if (!PutPage(p, i, s, s_kept[s], i - s_before[s], free, total)) bad = true;
        }
    }
    if (bad) RaiseFlag(p.err, 1);
}

__global__ __launch_bounds__(kRowThreads) void ReleasePages(const ReleaseArgs p) {
    const Pool& o = p.pool;
    const int32_t total = p.before[o.n_seqs], free = p.before[o.n_seqs + 1];
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRowThreads;
    bool bad = false;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x; i < total; i += step) {
        const int s = Find(p.before, o.n_seqs, static_cast<int32_t>(i));
        // (a sequence that gave pages back now has the length it kept)
        const int32_t kept = PagesOf(o.len[s], o.page_shift);
        if (!PutPage(p, static_cast<int32_t>(i), s, kept, static_cast<int32_t>(i) - p.before[s], free, total)) bad = true;
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
    if (pool->n_seqs == 0) return MLK_OK;
    if (new_tokens == nullptr || token_start == nullptr || !Aligned(new_tokens, 4) ||
        !Aligned(token_start, 4) || !Aligned(positions, 4) || !Aligned(token_seq, 4)) {
        return Fail(MLK_ERR_INVALID, "%s: new_tokens and token_start must be 4-byte aligned device "
                                     "arrays, as positions and token_seq where given", fn);
    }
    if (!Aligned(slots, 8)) return Fail(MLK_ERR_INVALID, "%s: slots must be 8-byte aligned", fn);
    const void* outs[4] = {token_start, positions, token_seq, slots};
    const void* ins[5] = {pool->page_table, pool->seq_len, pool->free_pages, pool->n_free, new_tokens};
    for (int i = 0; i < 4; ++i) {
        bool same = false;
        for (int j = 0; j < 5; ++j) same |= outs[i] == ins[j];
        for (int j = 0; j < i; ++j) same |= outs[i] != nullptr && outs[i] == outs[j];
        if (same) return Fail(MLK_ERR_INVALID, "%s: an output may not alias another or the pool", fn);
    }
    if (new_tokens == pool->seq_len) return Fail(MLK_ERR_INVALID, "%s: new_tokens may not alias seq_len", fn);
    st = CheckWorkspace(fn, workspace, workspace_bytes, pool->n_seqs);
    if (st != MLK_OK) return st;
    p.fresh = new_tokens;
    p.n_tokens = static_cast<int32_t>(n_tokens);
    p.max_len = static_cast<int32_t>(max_seq_len);
    p.start = token_start;
    p.positions = positions;
    p.seq = token_seq;
    p.slots = slots;
    p.base = static_cast<int32_t*>(workspace);
    p.err = err;
    const hipStream_t s = AsStream(stream);
    if (p.pool.n_seqs <= kScanSeqs && n_tokens <= kOwnRows) {
        hipLaunchKernelGGL(PlanScan<true>, dim3(1), dim3(kScanThreads), 0, s, p);
        return CheckLaunch("PlanScan");
    }
    hipLaunchKernelGGL(PlanScan<false>, dim3(1), dim3(kScanThreads), 0, s, p);
    st = CheckLaunch("PlanScan");
    if (st != MLK_OK || n_tokens == 0) return st;
    const dim3 grid(static_cast<unsigned>((n_tokens + kRowsEach - 1) / kRowsEach));
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
    p.err = err;
    const hipStream_t s = AsStream(stream);
    // pages that can come back at once
    const int64_t entries = pool->n_seqs * pool->table_stride;
    const int64_t most = entries < pool->n_pages ? entries : pool->n_pages;
    if (p.pool.n_seqs <= kScanSeqs && most <= kOwnRows) {
        hipLaunchKernelGGL(ReleaseScan<true>, dim3(1), dim3(kScanThreads), 0, s, p);
        return CheckLaunch("ReleaseScan");
    }
    hipLaunchKernelGGL(ReleaseScan<false>, dim3(1), dim3(kScanThreads), 0, s, p);
    st = CheckLaunch("ReleaseScan");
    if (st != MLK_OK) return st;
    hipLaunchKernelGGL(ReleasePages, dim3(GridFor(most, kRowThreads, 8)), dim3(kRowThreads), 0, s, p);
    return CheckLaunch("ReleasePages");
}

}  // extern "C"
