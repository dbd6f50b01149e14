// mlk_paged_index.h -- the index arithmetic of ragged batches and paged caches:
// which token rows and positions a sequence has and where a position's K and V
// rows lie.  Device arrays are not trusted: everything read from them is checked
// or clamped here before it becomes an address.  Plain C++ as well as device
// code, so that the CPU tests run the same functions.
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define MLK_HD __host__ __device__
#else
#define MLK_HD
#endif

namespace mlk {

// A ragged batch as the kernels see it.  Paged: sequence s's new tokens are its
// last positions.  Packed (table == nullptr): its tokens are the sequence.
struct Ragged {
    const int32_t* start;  // [n_seqs + 1]
    const int32_t* len;    // [n_seqs]; packed: nullptr
    const int32_t* table;  // [n_seqs, table_stride]; packed: nullptr
    int64_t table_stride;
    int32_t n_seqs, n_tokens, max_new, max_len;
};

struct Seq {
    int32_t t0, n, len;  // first token row, new tokens, length with them
};

// An element of an array that no kernel writes while it is read here.  On the
// device the load is from constant memory: with a uniform index it takes the
// scalar path, and does not queue behind the wave's loads of K and V.
MLK_HD inline int32_t ReadIndex(const int32_t* p) {
#ifdef __HIP_DEVICE_COMPILE__
    return *(const __attribute__((address_space(4))) int32_t*)(p);
#else
    return *p;
#endif
}

// Sequence s, checked against the host's bounds; false: out of bounds, to be
// left alone.
MLK_HD inline bool LoadSeq(const Ragged& r, int s, Seq* q) {
    const int32_t a = ReadIndex(r.start + s), b = ReadIndex(r.start + s + 1);
    if (a < 0 || b < a || b > r.n_tokens) return false;
    const int32_t n = b - a;
    const int32_t len = r.len != nullptr ? ReadIndex(r.len + s) : n;
    *q = {a, n, len};
    return n <= r.max_new && len >= n && len <= r.max_len;
}

// Score functions and masks (mlk_attention_scores); all zero: plain causal attention.
struct Scores {
    const float* slopes;          // [n_heads] or nullptr
    const int32_t *prefix, *first;  // [n_seqs], [n_tokens] or nullptr
    float softcap;
    int32_t window;               // 0: none
};

// The positions that token row t, at position pos of sequence s of length len, sees:
// lo .. hi, none where lo > hi.
struct Seen {
    int32_t lo, hi;
};
MLK_HD inline Seen SeenBy(const Scores& m, int s, int32_t t, int32_t pos, int32_t len) {
    Seen v{0, pos};
    if (m.window > 0 && pos - m.window + 1 > 0) v.lo = pos - m.window + 1;
    if (m.first != nullptr) {
        const int32_t f = ReadIndex(m.first + t);
        if (f > v.lo) v.lo = f;
    }
    if (m.prefix != nullptr) {
        // (compared before one is taken off: it may be of any value)
        const int32_t n = ReadIndex(m.prefix + s), end = n < len ? n : len;
        if (end > v.hi) v.hi = end - 1;
    }
    return v;
}

// Where K and V rows lie: position j's row of KV head g starts at element
//   paged:  page * page_stride + (j % page_size) * k_row + g * head_dim
//   packed: (t0 + j) * k_row + g * head_dim      (v_row for V)
struct RowsAt {
    const void *k, *v;
    int64_t page_stride;
    int64_t k_row, v_row;  // elements between positions
    int32_t page_shift;    // log2 of the page size
    int32_t n_pages;
    int32_t head_dim;
};

// The page of position j, 0 in place of one outside the cache (*bad set).
MLK_HD inline int32_t PageOf(const RowsAt& a, const int32_t* table_row, int32_t j, bool* bad) {
    const int32_t g = ReadIndex(table_row + (j >> a.page_shift));
    const bool in = g >= 0 && g < a.n_pages;
    if (!in) *bad = true;
    return in ? g : 0;
}

// Element offset of position j's K row (KV head 0) in page `page`.
MLK_HD inline int64_t PagedRow(const RowsAt& a, int32_t page, int32_t j) {
    return static_cast<int64_t>(page) * a.page_stride +
           static_cast<int64_t>(j & ((1 << a.page_shift) - 1)) * a.k_row;
}

}  // namespace mlk
