// mlk_paged.hip -- new tokens of many sequences into a paged KV cache, RoPE on
// the way, and the C entries of the attention over it (kernels: mlk_ragged.hip).
//
// Append: token row t of sequence s is position p = seq_len[s] - (start[s + 1]
// - t).  Pair i of a head of q or k turns by p * theta^(-2i / head_dim)
// (float64 angle, cos, sin and rotation, rounded to float as mlk_rope_f32
// does, then to the type stored); k and v rows go to page table[s][p /
// page_size], row p % page_size.  Bound by bytes: it reads q, k and v and
// writes q and the two cache rows once.
//
// One workgroup per token: its first threads evaluate the token's angles into
// shared memory (every head of q and k turns by the same ones), all threads move
// units of PV pairs.  A unit's elements are one run of 16 bytes (normal pairs: PV
// neighbouring ones) or two (NeoX: half a head apart), so that every load and
// store of a wave is contiguous, which the non-temporal stores need: with runs of
// 32 bytes in two halves they cost 15% instead of gaining 10%.  The first
// kBatch units' loads are issued before the angles.
//
// 4096 fp32 tokens of 8B heads into an fp16 cache (185 MB) take 34 us, 8191 bf16
// tokens of 70B heads (336 MB) 61 us: 5.5 TB/s, where torch's 4 GiB copy reaches
// 4.8.  64 decode tokens take 6 us, a launch.
#include "mlk_paged.h"

#include <climits>
#include <cmath>

namespace mlk {
namespace {

constexpr int kAppendThreads = 256;

struct AppendArgs {
    Ragged batch;
    RowsAt rows;
    const void *k, *v, *q;
    void* q_out;
    int64_t k_row, v_row, q_row, q_out_row;
    int32_t n_heads, n_kv_heads;  // n_heads 0: no q
    bool rope;
    int32_t* err;
};

constexpr int kBatch = 3;  // units a thread loads before it rotates the first

// N elements of T from / to memory, through fp32.
template <typename T, int N>
__device__ inline void LoadN(const typename T::Bits* p, float* x) {
    if constexpr (N == 1) {
        x[0] = T::Get(*p);
    } else {
        typedef typename T::Bits Vec __attribute__((ext_vector_type(N)));
        const Vec v = __builtin_nontemporal_load(reinterpret_cast<const Vec*>(p));
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = T::Get(v[i]);
    }
}
template <typename T, int N>
__device__ inline void StoreN(typename T::Bits* p, const float* x) {
    if constexpr (N == 1) {
        *p = T::Put(x[0]);
    } else {
        typedef typename T::Bits Vec __attribute__((ext_vector_type(N)));
        Vec v;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = T::Put(x[i]);
        __builtin_nontemporal_store(v, reinterpret_cast<Vec*>(p));
    }
}

// One unit in fp32: x[2 i], x[2 i + 1] are pair i.
template <typename A, int PV, bool kNeox>
struct Unit {
    float x[2 * PV];
    int64_t o;   // element offset of the head in its row
    int g, to;   // group of pairs in the head; 0: q, 1: k, 2: v, -1: none
    template <typename T>
    __device__ void Load(const T* row, int half, int hd) {
        const T* src = row + o;
        if constexpr (PV == 1) {
            const int e1 = kNeox ? g + half : 2 * g + 1;
            x[0] = A::Get(src[kNeox ? g : 2 * g]);
            x[1] = e1 < hd ? A::Get(src[e1]) : 0.0f;
        } else if constexpr (kNeox) {
            float a[PV], b[PV];
            LoadN<A, PV>(src + PV * g, a);
            LoadN<A, PV>(src + PV * g + half, b);
#pragma unroll
            for (int i = 0; i < PV; ++i) {
                x[2 * i] = a[i];
                x[2 * i + 1] = b[i];
            }
        } else {
            LoadN<A, 2 * PV>(src + 2 * PV * g, x);
        }
    }
    template <typename C, typename T>
    __device__ void Store(T* row, int half, int hd) const {
        T* dst = row + o;
        if constexpr (PV == 1) {
            const int e1 = kNeox ? g + half : 2 * g + 1;
            dst[kNeox ? g : 2 * g] = C::Put(x[0]);
            if (e1 < hd) dst[e1] = C::Put(x[1]);
        } else if constexpr (kNeox) {
            float a[PV], b[PV];
#pragma unroll
            for (int i = 0; i < PV; ++i) {
                a[i] = x[2 * i];
                b[i] = x[2 * i + 1];
            }
            StoreN<C, PV>(dst + PV * g, a);
            StoreN<C, PV>(dst + PV * g + half, b);
        } else {
            StoreN<C, 2 * PV>(dst + 2 * PV * g, x);
        }
    }
};

template <typename A, typename C, int PV, bool kNeox>
__global__ __launch_bounds__(kAppendThreads) void PagedAppend(AppendArgs p, const RopeFreqs f) {
    __shared__ double2 turn[kRopePairs];  // cos, sin of the token's pairs
    const int tid = static_cast<int>(threadIdx.x);
    const int32_t t = static_cast<int32_t>(blockIdx.x);
    const int hd = p.rows.head_dim, half = (hd + 1) / 2;
    if (t == 0) CheckSeqs(p.batch, p.err);
    const int s = LastSeq(p.batch, t, [](int32_t a, int) { return a; });
    Seq q;
    if (!LoadSeq(p.batch, s, &q) || t < q.t0 || t >= q.t0 + q.n) return;
    const int32_t pos = q.len - q.n + (t - q.t0);
    bool bad = false;
    const int32_t page = PageOf(p.rows, p.batch.table + s * p.batch.table_stride, pos, &bad);
    if (bad && tid == 0) RaiseFlag(p.err, 1);
    const int64_t at = PagedRow(p.rows, page, pos);
    typedef typename A::Bits AB;
    typedef typename C::Bits CB;
    const AB* rq = static_cast<const AB*>(p.q) + t * p.q_row;
    const AB* rk = static_cast<const AB*>(p.k) + t * p.k_row;
    const AB* rv = static_cast<const AB*>(p.v) + t * p.v_row;
    AB* oq = static_cast<AB*>(p.q_out) + t * p.q_out_row;
    CB* ok = static_cast<CB*>(const_cast<void*>(p.rows.k)) + at;
    CB* ov = static_cast<CB*>(const_cast<void*>(p.rows.v)) + at;
    const int groups = half / PV;
    const int units = (p.n_heads + 2 * p.n_kv_heads) * groups;
    Unit<A, PV, kNeox> u[kBatch];
    auto load = [&](int first) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int i = first + b * kAppendThreads;
            u[b].to = -1;
            if (i >= units) continue;
            const int h = i / groups;
            u[b].g = i % groups;
            u[b].to = h < p.n_heads ? 0 : h < p.n_heads + p.n_kv_heads ? 1 : 2;
            const int in = u[b].to == 0 ? h
                           : u[b].to == 1 ? h - p.n_heads : h - p.n_heads - p.n_kv_heads;
            u[b].o = static_cast<int64_t>(in) * hd;
            u[b].Load(u[b].to == 0 ? rq : u[b].to == 1 ? rk : rv, half, hd);
        }
    };
    load(tid);
    if (p.rope) {
        for (int i = tid; i < half; i += kAppendThreads) {
            RopeCosSin(pos, f.inv[i], &turn[i].x, &turn[i].y);
        }
        __syncthreads();
    }
    for (int first = tid; first < units; first += kBatch * kAppendThreads) {
        if (first != tid) load(first);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (u[b].to < 0) continue;
            if (p.rope && u[b].to != 2) {
#pragma unroll
                for (int i = 0; i < PV; ++i) {
                    const double2 c = turn[u[b].g * PV + i];
                    RopeRotate(u[b].x[2 * i], u[b].x[2 * i + 1], c.x, c.y, &u[b].x[2 * i],
                               &u[b].x[2 * i + 1]);
                }
            }
            if (u[b].to == 0) u[b].template Store<A>(oq, half, hd);
            else if (!bad) u[b].template Store<C>(u[b].to == 1 ? ok : ov, half, hd);
        }
    }
}

// Pairs of a 16-byte unit.
template <typename A>
constexpr int UnitPairs(bool neox) {
    return (neox ? 16 : 8) / static_cast<int>(sizeof(typename A::Bits));
}

template <typename A, typename C>
void LaunchAppend(const AppendArgs& p, const RopeFreqs& f, bool neox, bool wide, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(p.batch.n_tokens)), block(kAppendThreads);
    if (neox) {
        if (wide) hipLaunchKernelGGL((PagedAppend<A, C, UnitPairs<A>(true), true>), grid, block, 0, s, p, f);
        else hipLaunchKernelGGL((PagedAppend<A, C, 1, true>), grid, block, 0, s, p, f);
    } else {
        if (wide) hipLaunchKernelGGL((PagedAppend<A, C, UnitPairs<A>(false), false>), grid, block, 0, s, p, f);
        else hipLaunchKernelGGL((PagedAppend<A, C, 1, false>), grid, block, 0, s, p, f);
    }
}

bool KnownType(int32_t t) { return t == MLK_F32 || t == MLK_F16 || t == MLK_BF16; }

}  // namespace

mlk_status CheckElements(const char* fn, const char* name, const void* p, int32_t type) {
    if (p == nullptr) return Fail(MLK_ERR_INVALID, "%s: %s must not be null", fn, name);
    if (!Aligned(p, TypeBytes(type))) {
        return Fail(MLK_ERR_INVALID, "%s: %s must be %d-byte aligned", fn, name, TypeBytes(type));
    }
    return MLK_OK;
}

mlk_status CheckHeads(const char* fn, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                      float scale) {
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0) {
        return Fail(MLK_ERR_INVALID, "%s: n_heads must be a positive multiple of n_kv_heads", fn);
    }
    if (n_heads > 65536) {
        return Fail(MLK_ERR_INVALID, "%s: more than 65536 heads", fn);
    }
    if (head_dim < 1 || head_dim > 256) {
        return Fail(MLK_ERR_INVALID, "%s: head_dim must be in 1..256", fn);
    }
    if (!std::isfinite(scale) || scale <= 0.0f) {
        return Fail(MLK_ERR_INVALID, "%s: scale must be finite and positive", fn);
    }
    return MLK_OK;
}

static mlk_status CheckCounts(const char* fn, int64_t n_seqs, int64_t n_tokens) {
    if (n_seqs < 0 || n_seqs > kMaxSeqs || n_tokens < 0 || n_tokens > kMaxTokens) {
        return Fail(MLK_ERR_INVALID, "%s: n_seqs must be in 0..2^20 and n_tokens in 0..2^23", fn);
    }
    return MLK_OK;
}

mlk_status CheckPaged(const char* fn, const mlk_paged_cache* cache, const mlk_paged_batch* batch,
                      int32_t type, PagedArgs* args) {
    if (cache == nullptr || batch == nullptr) {
        return Fail(MLK_ERR_INVALID, "%s: cache and batch must not be null", fn);
    }
    const mlk_paged_cache& c = *cache;
    const mlk_paged_batch& b = *batch;
    if (!KnownType(type) || !KnownType(c.type)) {
        return Fail(MLK_ERR_INVALID, "%s: unknown element type", fn);
    }
    if (type != MLK_F32 && type != c.type) {
        return Fail(MLK_ERR_INVALID, "%s: 16-bit activations need a cache of their own type", fn);
    }
    if (c.n_kv_heads <= 0 || c.n_kv_heads > 65536) {
        return Fail(MLK_ERR_INVALID, "%s: n_kv_heads must be in 1..65536", fn);
    }
    if (c.head_dim < 1 || c.head_dim > 256) {
        return Fail(MLK_ERR_INVALID, "%s: head_dim must be in 1..256", fn);
    }
    if (c.page_size < 1 || c.page_size > (1 << 20) || (c.page_size & (c.page_size - 1)) != 0) {
        return Fail(MLK_ERR_INVALID, "%s: page_size must be a power of two up to 2^20", fn);
    }
    if (c.n_pages < 1 || c.n_pages > INT32_MAX) {
        return Fail(MLK_ERR_INVALID, "%s: n_pages must be in 1..2^31 - 1", fn);
    }
    const int64_t slot = static_cast<int64_t>(c.n_kv_heads) * c.head_dim;
    if (c.page_stride < c.page_size * slot || c.page_stride > INT64_MAX / 4 / c.n_pages) {
        return Fail(MLK_ERR_INVALID,
                    "%s: page_stride must cover page_size * n_kv_heads * head_dim elements", fn);
    }
    mlk_status st = CheckElements(fn, "k pages", c.k, c.type);
    if (st != MLK_OK) return st;
    st = CheckElements(fn, "v pages", c.v, c.type);
    if (st != MLK_OK) return st;
    if (c.k == c.v) return Fail(MLK_ERR_INVALID, "%s: k and v pages must be distinct", fn);
    st = CheckCounts(fn, b.n_seqs, b.n_tokens);
    if (st != MLK_OK) return st;
    int shift = 0;
    while ((1 << shift) < c.page_size) ++shift;
    *args = {};
    args->rows = {c.k, c.v, c.page_stride, slot, slot, shift, static_cast<int32_t>(c.n_pages),
                  c.head_dim};
    if (b.n_seqs == 0 || b.n_tokens == 0) return MLK_OK;  // nothing to do
    if (b.token_start == nullptr || b.seq_len == nullptr || b.page_table == nullptr) {
        return Fail(MLK_ERR_INVALID, "%s: token_start, seq_len and page_table must not be null",
                    fn);
    }
    if (!Aligned(b.token_start, 4) || !Aligned(b.seq_len, 4) || !Aligned(b.page_table, 4)) {
        return Fail(MLK_ERR_INVALID,
                    "%s: token_start, seq_len and page_table must be 4-byte aligned", fn);
    }
    if (b.max_new_tokens < 1 || b.max_seq_len < 1 || b.max_seq_len > (1 << 30)) {
        return Fail(MLK_ERR_INVALID,
                    "%s: max_new_tokens must be positive and max_seq_len in 1..2^30", fn);
    }
    if (b.table_stride < 1 || b.table_stride > INT32_MAX ||
        b.max_seq_len > b.table_stride * c.page_size) {
        return Fail(MLK_ERR_INVALID, "%s: max_seq_len exceeds table_stride * page_size", fn);
    }
    int64_t max_new = b.max_new_tokens < b.max_seq_len ? b.max_new_tokens : b.max_seq_len;
    if (max_new > b.n_tokens) max_new = b.n_tokens;
    args->batch = {b.token_start, b.seq_len, b.page_table, b.table_stride,
                   static_cast<int32_t>(b.n_seqs), static_cast<int32_t>(b.n_tokens),
                   static_cast<int32_t>(max_new), static_cast<int32_t>(b.max_seq_len)};
    return MLK_OK;
}

}  // namespace mlk

using namespace mlk;

extern "C" {

mlk_status mlk_paged_kv_append(const mlk_paged_cache* cache, const mlk_paged_batch* batch,
                               int32_t type, const void* k, int64_t k_row_stride, const void* v,
                               int64_t v_row_stride, const void* q, int64_t q_row_stride,
                               void* q_out, int64_t q_out_row_stride, int32_t n_heads,
                               float theta, int32_t rope_type, int32_t* err, void* stream) {
    const char* fn = "mlk_paged_kv_append";
    PagedArgs a;
    mlk_status st = CheckPaged(fn, cache, batch, type, &a);
    if (st != MLK_OK) return st;
    const int32_t hd = cache->head_dim, KV = cache->n_kv_heads;
    const int64_t slot = static_cast<int64_t>(KV) * hd;
    st = CheckElements(fn, "k", k, type);
    if (st != MLK_OK) return st;
    st = CheckElements(fn, "v", v, type);
    if (st != MLK_OK) return st;
    if (k_row_stride < slot || v_row_stride < slot) {
        return Fail(MLK_ERR_INVALID, "%s: row strides must be at least n_kv_heads * head_dim", fn);
    }
    if (!std::isfinite(theta) || theta < 0.0f) {
        return Fail(MLK_ERR_INVALID, "%s: theta must be finite and not negative", fn);
    }
    if (theta != 0.0f) {
        if (rope_type != MLK_ROPE_NORMAL && rope_type != MLK_ROPE_NEOX) {
            return Fail(MLK_ERR_INVALID, "%s: unknown rope type %d", fn, rope_type);
        }
        if (hd % 2 != 0) return Fail(MLK_ERR_INVALID, "%s: head_dim must be even", fn);
    } else if (q != nullptr) {
        return Fail(MLK_ERR_INVALID, "%s: theta 0 rotates nothing: q must be null", fn);
    }
    if (q != nullptr) {
        st = CheckElements(fn, "q", q, type);
        if (st != MLK_OK) return st;
        st = CheckElements(fn, "q_out", q_out, type);
        if (st != MLK_OK) return st;
        if (n_heads <= 0 || n_heads > 65536) {
            return Fail(MLK_ERR_INVALID, "%s: n_heads must be in 1..65536", fn);
        }
        const int64_t width = static_cast<int64_t>(n_heads) * hd;
        if (q_row_stride < width || q_out_row_stride < width) {
            return Fail(MLK_ERR_INVALID, "%s: row strides must be at least n_heads * head_dim",
                        fn);
        }
        if (q_out == q && q_out_row_stride != q_row_stride) {
            return Fail(MLK_ERR_INVALID, "%s: q in place needs equal row strides", fn);
        }
        if (q_out == k || q_out == v || q_out == cache->k || q_out == cache->v) {
            return Fail(MLK_ERR_INVALID, "%s: q_out may not alias k, v or the pages", fn);
        }
    }
    if (k == cache->k || k == cache->v || v == cache->k || v == cache->v) {
        return Fail(MLK_ERR_INVALID, "%s: k and v may not alias the pages", fn);
    }
    if (a.batch.n_seqs == 0) return MLK_OK;
    const bool neox = theta != 0.0f && rope_type == MLK_ROPE_NEOX;
    AppendArgs p{};
    p.batch = a.batch;
    p.rows = a.rows;
    p.k = k;
    p.v = v;
    p.q = q;
    p.q_out = q != nullptr ? q_out : nullptr;
    p.k_row = k_row_stride;
    p.v_row = v_row_stride;
    p.q_row = q != nullptr ? q_row_stride : 0;
    p.q_out_row = q != nullptr ? q_out_row_stride : 0;
    p.n_heads = q != nullptr ? n_heads : 0;
    p.n_kv_heads = KV;
    p.rope = theta != 0.0f;
    p.err = err;
    // 16-byte units: `run` neighbouring elements everywhere
    const int ab = TypeBytes(type), cb = TypeBytes(cache->type), run = 16 / ab;
    const bool wide = hd % (neox ? 2 * run : run) == 0 && k_row_stride % run == 0 &&
                      v_row_stride % run == 0 && cache->page_stride % run == 0 &&
                      p.q_row % run == 0 && p.q_out_row % run == 0 && Aligned(k, 16) &&
                      Aligned(v, 16) && Aligned(q, 16) && Aligned(p.q_out, 16) &&
                      Aligned(cache->k, run * cb) && Aligned(cache->v, run * cb);
    const RopeFreqs f = p.rope ? MakeRopeFreqs(theta, hd) : RopeFreqs{};
    const hipStream_t s = AsStream(stream);
    if (type == MLK_F32) {
        if (cache->type == MLK_F32) LaunchAppend<F32, F32>(p, f, neox, wide, s);
        else if (cache->type == MLK_F16) LaunchAppend<F32, F16>(p, f, neox, wide, s);
        else LaunchAppend<F32, BF16>(p, f, neox, wide, s);
    } else if (type == MLK_F16) {
        LaunchAppend<F16, F16>(p, f, neox, wide, s);
    } else {
        LaunchAppend<BF16, BF16>(p, f, neox, wide, s);
    }
    return CheckLaunch("PagedAppend");
}

mlk_status mlk_attention_paged(const mlk_paged_cache* cache, const mlk_paged_batch* batch,
                               int32_t type, const void* q, int64_t q_row_stride, void* out,
                               int32_t n_heads, float scale, void* workspace,
                               size_t workspace_bytes, int32_t* err, void* stream) {
    const char* fn = "mlk_attention_paged";
    PagedArgs a;
    mlk_status st = CheckPaged(fn, cache, batch, type, &a);
    if (st != MLK_OK) return st;
    st = CheckHeads(fn, n_heads, cache->n_kv_heads, cache->head_dim, scale);
    if (st != MLK_OK) return st;
    st = CheckElements(fn, "q", q, type);
    if (st != MLK_OK) return st;
    st = CheckElements(fn, "out", out, type);
    if (st != MLK_OK) return st;
    if (q_row_stride < static_cast<int64_t>(n_heads) * cache->head_dim) {
        return Fail(MLK_ERR_INVALID, "%s: q_row_stride must be at least n_heads * head_dim", fn);
    }
    if (out == q || out == cache->k || out == cache->v) {
        return Fail(MLK_ERR_INVALID, "%s: out may not alias q or the pages", fn);
    }
    if (workspace != nullptr && !Aligned(workspace, 16)) {
        return Fail(MLK_ERR_INVALID, "%s: workspace must be 16-byte aligned", fn);
    }
    if (a.batch.n_seqs == 0) return MLK_OK;
    return Attend({a.batch, a.rows, type, cache->type, q, q_row_stride, out, n_heads,
                   cache->n_kv_heads, scale, workspace, workspace == nullptr ? 0 : workspace_bytes,
                   err, AsStream(stream)});
}

int64_t mlk_attention_paged_workspace_bytes(int64_t n_seqs, int64_t n_tokens,
                                            int64_t max_new_tokens, int64_t max_seq_len,
                                            int32_t n_heads, int32_t n_kv_heads,
                                            int32_t head_dim) {
    return AttendWorkspace(n_seqs, n_tokens, max_new_tokens, max_seq_len, n_heads, n_kv_heads,
                           head_dim, false);
}

mlk_status mlk_attention_packed(int32_t type, const void* q, int64_t q_row_stride, const void* k,
                                int64_t k_row_stride, const void* v, int64_t v_row_stride,
                                const int32_t* seq_start, int64_t n_seqs, int64_t n_tokens,
                                int64_t max_seq_len, int32_t n_heads, int32_t n_kv_heads,
                                int32_t head_dim, float scale, void* out, void* workspace,
                                size_t workspace_bytes, int32_t* err, void* stream) {
    const char* fn = "mlk_attention_packed";
    if (!KnownType(type)) return Fail(MLK_ERR_INVALID, "%s: unknown element type", fn);
    mlk_status st = CheckHeads(fn, n_heads, n_kv_heads, head_dim, scale);
    if (st != MLK_OK) return st;
    const char* names[4] = {"q", "k", "v", "out"};
    const void* ptrs[4] = {q, k, v, out};
    for (int i = 0; i < 4; ++i) {
        st = CheckElements(fn, names[i], ptrs[i], type);
        if (st != MLK_OK) return st;
    }
    const int64_t slot = static_cast<int64_t>(n_kv_heads) * head_dim;
    if (q_row_stride < static_cast<int64_t>(n_heads) * head_dim || k_row_stride < slot ||
        v_row_stride < slot) {
        return Fail(MLK_ERR_INVALID, "%s: row strides must be at least heads * head_dim", fn);
    }
    if (out == q || out == k || out == v) {
        return Fail(MLK_ERR_INVALID, "%s: out may not alias q, k or v", fn);
    }
    if (k_row_stride > kMaxRow || v_row_stride > kMaxRow) {
        return Fail(MLK_ERR_INVALID, "%s: k and v row strides must be at most 2^27 elements", fn);
    }
    st = CheckCounts(fn, n_seqs, n_tokens);
    if (st != MLK_OK) return st;
    if (workspace != nullptr && !Aligned(workspace, 16)) {
        return Fail(MLK_ERR_INVALID, "%s: workspace must be 16-byte aligned", fn);
    }
    if (n_seqs == 0 || n_tokens == 0) return MLK_OK;
    if (seq_start == nullptr || !Aligned(seq_start, 4)) {
        return Fail(MLK_ERR_INVALID, "%s: seq_start must be a 4-byte aligned device array", fn);
    }
    if (max_seq_len < 1) return Fail(MLK_ERR_INVALID, "%s: max_seq_len must be positive", fn);
    const int32_t T = static_cast<int32_t>(n_tokens);
    const int32_t most = max_seq_len < n_tokens ? static_cast<int32_t>(max_seq_len) : T;
    const Ragged b{seq_start, nullptr, nullptr, 0, static_cast<int32_t>(n_seqs), T, most, most};
    const RowsAt r{k, v, 0, k_row_stride, v_row_stride, 0, 0, head_dim};
    return Attend({b, r, type, type, q, q_row_stride, out, n_heads, n_kv_heads, scale, workspace,
                   workspace == nullptr ? 0 : workspace_bytes, err, AsStream(stream)});
}

int64_t mlk_attention_packed_workspace_bytes(int64_t n_seqs, int64_t n_tokens,
                                             int64_t max_seq_len, int32_t n_heads,
                                             int32_t n_kv_heads, int32_t head_dim) {
    return AttendWorkspace(n_seqs, n_tokens, max_seq_len, max_seq_len, n_heads, n_kv_heads,
                           head_dim, true);
}

}  // extern "C"
