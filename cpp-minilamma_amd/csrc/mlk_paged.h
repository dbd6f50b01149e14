// mlk_paged.h -- what the kernels for many sequences at once share: element
// types, the search for a row's sequence and the arguments' checks (the index
// arithmetic itself: mlk_paged_index.h).
#pragma once

#include "mlk_common.h"
#include "mlk_paged_index.h"

namespace mlk {

// ------------------------------------------------------------ element types
// 16-bit elements are handled as their bits; arithmetic is fp32.

struct F32 {
    typedef float Bits;
    static constexpr int kType = MLK_F32;
    static __device__ float Get(float v) { return v; }
    static __device__ float Put(float v) { return v; }
};
struct F16 {
    typedef uint16_t Bits;
    static constexpr int kType = MLK_F16;
    static __device__ float Get(uint16_t v) {
        return static_cast<float>(__builtin_bit_cast(_Float16, v));
    }
    static __device__ uint16_t Put(float v) {
        return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
    }
};
struct BF16 {
    typedef uint16_t Bits;
    static constexpr int kType = MLK_BF16;
    static __device__ float Get(uint16_t v) { return __uint_as_float(uint32_t{v} << 16); }
    static __device__ uint16_t Put(float v) {
        return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
    }
};

// Raises *err for sequences out of bounds; every thread of one workgroup.
__device__ inline void CheckSeqs(const Ragged& r, int32_t* err) {
    if (err == nullptr) return;
    bool bad = false;
    for (int s = static_cast<int>(threadIdx.x); s < r.n_seqs; s += static_cast<int>(blockDim.x)) {
        Seq q;
        if (!LoadSeq(r, s, &q)) bad = true;
    }
    if (bad) RaiseFlag(err, 1);
}

// Largest s of 0 .. n_seqs - 1 with f(start[s], s) <= x (f non-decreasing in s;
// n_seqs >= 1; 0 where none).  The lanes of the wave look at 64 sequences at once,
// evenly apart until 64 are left: one load each time, n_seqs / 64 left after it.
// (Append of one bf16 token each of 65536 sequences, 8B heads: 0.35 ms; looking at
// 64 neighbours at a time 4.7.)
// (Whatever the device holds, `left` shrinks and s stays below n_seqs.)
template <typename F>
__device__ inline int LastSeq(const Ragged& r, int64_t x, F f) {
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    int from = 0, left = r.n_seqs;
    for (;;) {
        const int step = (left + kWave - 1) / kWave, at = lane * step;
        const bool in = at < left && f(ReadIndex(r.start + from + at), from + at) <= x;
        const int c = __popcll(__ballot(in));
        if (c > 0) from += (c - 1) * step;
        if (c == 0 || step == 1) return __builtin_amdgcn_readfirstlane(from);
        left = left - (c - 1) * step < step ? left - (c - 1) * step : step;
    }
}

// ------------------------------------------------------------ host checks

// Bounds that keep grids below 2^32 threads and the offsets of a few rows, from
// one of them on, below 2^32 elements.
constexpr int64_t kMaxSeqs = 1 << 20, kMaxTokens = 1 << 23, kMaxRow = 1 << 27;

struct PagedArgs {
    Ragged batch;
    RowsAt rows;
};

// Checks cache and batch and fills *args; `type` is the activations' type.
mlk_status CheckPaged(const char* fn, const mlk_paged_cache* cache, const mlk_paged_batch* batch,
                      int32_t type, PagedArgs* args);
// n_heads, scale and types of an attention call.
mlk_status CheckHeads(const char* fn, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                      float scale);
// A buffer of `type` elements.
mlk_status CheckElements(const char* fn, const char* name, const void* p, int32_t type);

inline int TypeBytes(int32_t type) { return type == MLK_F32 ? 4 : 2; }

// ------------------------------------------------------------ attention

// One launch of ragged attention (mlk_ragged.hip).
struct AttendArgs {
    Ragged batch;
    RowsAt rows;
    int32_t type, cache_type;
    const void* q;
    int64_t q_row;
    void* out;
    int32_t n_heads, n_kv_heads;
    float scale;
    void* workspace;
    size_t workspace_bytes;
    int32_t* err;
    hipStream_t stream;
    Scores scores;
};
mlk_status Attend(const AttendArgs& a);
// With a.scores.
mlk_status AttendScored(const AttendArgs& a);
int64_t AttendWorkspace(int64_t n_seqs, int64_t n_tokens, int64_t max_new, int64_t max_len,
                        int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, bool packed,
                        const Scores& scores, bool scored);

}  // namespace mlk
