// mlk_ragged.h -- what the two kernels of ragged attention share: the matrix
// instructions over 16-bit elements, the split of fp32 values into 16-bit
// pieces, and the launch parameters.
//
// Pieces.  fp32 q and softmax weights w meet 16-bit (or fp32) K and V on the
// 16-bit matrix cores as sums of 16-bit pieces:
//   fp16 K, V: 2 fp16 pieces (11 + 11 bits, truncated: within 2^-21 of the value).
//     q is first scaled by a power of two per row, its largest element to
//     2^14 .. 2^15, and w by 2^14, so that the second piece of all but tiny
//     elements is a normal fp16 number; the scales go into the exponent's factor
//     and cancel in the division by the sum.
//   bf16 K, V: 3 bf16 pieces, exact (8 + 8 + 8 bits).
//   fp32 K, V: 3 x 3 bf16 pieces, the 6 products above 2^-21 of q k (the three
//     dropped ones are below 2^-20).
// 16-bit q needs no split.  Its w (fp16: scaled as above) is two pieces of its type in
// the few-row kernel, within 2^-15 of it (fp16 2^-20): bound by bytes, that costs
// nothing there (64 bf16 decode rows of the 8B heads 190 us either way).  In the tile
// kernel w is rounded to q's type: the second piece's products would take 657 to 836 us
// (9001 packed bf16 tokens of the 70B heads), and over values of either sign the
// weights' roundings add about a quarter to the error of the result's own.
#pragma once

#include "mlk_paged.h"

#include <cmath>
#include <type_traits>

namespace mlk {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f;

struct MmaBf {
    static __device__ f32x16 Mma32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ f32x4 Mma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ uint32_t Round2(float a, float b) {
        const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
        return __builtin_bit_cast(uint32_t, v);
    }
    // 2 values into N pieces each
    template <int N>
    static __device__ void Split2(float a, float b, uint32_t (&o)[N]) {
        if constexpr (N == 1) {
            o[0] = Round2(a, b);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                o[i] = i + 1 < N ? PackBf(a, b) : Round2(a, b);
                if (i + 1 < N) {
                    a -= __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
                    b -= __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
                }
            }
        }
    }
};

struct MmaF16 {
    static __device__ f32x16 Mma32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ f32x4 Mma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ uint32_t Round2(float a, float b) {
        const f16x2 v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
        return __builtin_bit_cast(uint32_t, v);
    }
    template <int N>
    static __device__ void Split2(float a, float b, uint32_t (&o)[N]) {
        if constexpr (N == 1) {
            o[0] = Round2(a, b);
        } else {
            static_assert(N == 2);
            const auto hi = __builtin_amdgcn_cvt_pkrtz(a, b);
            o[0] = __builtin_bit_cast(uint32_t, hi);
            o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(
                                                    a - static_cast<float>(hi[0]),
                                                    b - static_cast<float>(hi[1])));
        }
    }
};

// How activations of type A meet a cache of type C: NQ pieces of q (and of w in the
// tile kernel), NK of K and V, NW of w in the few-row kernel; W: w's scale, a power
// of two; kScaleQ: q scaled per row.
template <typename A, typename C>
struct Pieces;
template <>
struct Pieces<BF16, BF16> {
    typedef MmaBf M;
    static constexpr int NQ = 1, NK = 1, NW = 2, W = 0;
    static constexpr bool kScaleQ = false;
};
template <>
struct Pieces<F16, F16> {
    typedef MmaF16 M;
    static constexpr int NQ = 1, NK = 1, NW = 2, W = 14;
    static constexpr bool kScaleQ = false;
};
template <>
struct Pieces<F32, F16> {
    typedef MmaF16 M;
    static constexpr int NQ = 2, NK = 1, NW = 2, W = 14;
    static constexpr bool kScaleQ = true;
};
template <>
struct Pieces<F32, BF16> {
    typedef MmaBf M;
    static constexpr int NQ = 3, NK = 1, NW = 3, W = 0;
    static constexpr bool kScaleQ = false;
};
template <>
struct Pieces<F32, F32> {
    typedef MmaBf M;
    static constexpr int NQ = 3, NK = 3, NW = 3, W = 0;
    static constexpr bool kScaleQ = false;
};

// Eight fp32 values into N operands.
template <typename M, int N>
__device__ inline void Split8(const float* x, u32x4 (&o)[N]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w[N];
        M::template Split2<N>(x[2 * i], x[2 * i + 1], w);
#pragma unroll
        for (int p = 0; p < N; ++p) o[p][i] = w[p];
    }
}

// Power-of-two exponent that brings a row's largest |q| to 2^14 .. 2^15 (0 for
// a row of zeros or with a non-finite element).
__device__ inline int RowExponent(float amax) {
    const int e = static_cast<int>(__float_as_uint(amax) >> 23);  // amax >= 0; subnormal: 0
    if (amax == 0.0f || e == 255) return 0;
    const int s = 14 - (e - 127);
    return s < 100 ? s : 100;
}

// The scores' factor for a row scaled by 2^e, kept a normal number: 0 or infinity times
// a difference of infinity or 0 would be NaN.  Below the least one every weight is 1
// (scores are below 2^40 in size), above the largest only the maximum's is not 0.
__device__ inline float RowFactor(float factor, int e) {
    return fminf(fmaxf(ldexpf(factor, -e), 0x1p-126f), 0x1.fffffep127f);
}

// Maximum / sum over the lanes l, l ^ 32 (every lane gets it).
__device__ inline float Max32(float v) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                     false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float Sum32(float v) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                     false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The same over l, l ^ 16.
__device__ inline float Max16(float v) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                     false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float Sum16(float v) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                     false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---------------------------------------------------- non-finite V, masked tiles
// A weight of 0 does not hide an infinity or NaN in a matrix product.  Where a
// tile has positions that some row does not attend to, V is looked through for
// non-finite values as it lies in registers, and they are replaced by zeros; a
// workgroup that met any adds them to the results of the rows that do attend to
// them, element by element, at its end (adding one twice changes nothing).

// Replaces the non-finite of N dwords' elements by zeros; whether there was one.
// An exponent of all ones is found by the carry of its lowest bit into the sign's
// place: integer work in vector registers, no lane masks.
template <typename C, int N>
__device__ inline bool OnlyFinite(uint32_t* v) {
    constexpr uint32_t kExp = C::kType == MLK_F32 ? 0x7F800000u
                              : C::kType == MLK_F16 ? 0x7C007C00u : 0x7F807F80u;
    constexpr uint32_t kLow = C::kType == MLK_F32 ? 0x00800000u
                              : C::kType == MLK_F16 ? 0x04000400u : 0x00800080u;
    constexpr uint32_t kSign = C::kType == MLK_F32 ? 0x80000000u : 0x80008000u;
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) any |= (v[i] & kExp) + kLow;
    any &= kSign;
    if (any != 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t hit = ((v[i] & kExp) + kLow) & kSign;
            if constexpr (C::kType == MLK_F32) {
                v[i] &= ~static_cast<uint32_t>(static_cast<int32_t>(hit) >> 31);
            } else {
                v[i] &= ~((hit >> 15) * 0xFFFFu);
            }
        }
    }
    return any != 0;
}

// The sum of the non-finite elements at dim d of positions first .. last of a
// sequence (0: none); `v` is the KV head's first element.
template <typename C>
__device__ inline float NonFiniteSum(const RowsAt& at, const int32_t* table, int64_t t0,
                                     const typename C::Bits* v, int32_t first, int32_t last,
                                     int d) {
    float sum = 0.0f;
    bool bad = false;
    for (int32_t j = first; j <= last; ++j) {
        const int64_t o = table != nullptr ? PagedRow(at, PageOf(at, table, j, &bad), j)
                                           : (t0 + j) * at.v_row;
        const float x = C::Get(v[o + d]);
        if (!__builtin_isfinite(x)) sum += x;
    }
    return sum;
}

// ------------------------------------------------------------ launches

struct RaggedParams {
    Ragged batch;
    RowsAt rows;
    const void* q;
    int64_t q_row;
    void* out;
    int32_t n_heads, n_kv_heads, group;
    float factor;  // scale * log2 e
    int32_t vec;   // rows of q, K and V 16-byte aligned, head_dim % 8 == 0
    // tile kernel: chunk c of a row is positions c * chunk .. of it
    int32_t chunk, n_chunks;
    // few-row kernel: workgroups (0: one per sequence and KV head), and the most KV
    // heads a workgroup's waves may take side by side
    int32_t workers, few_heads;
    // sequences or row tiles that earlier launches of the call have taken
    int64_t taken;
    // partial results (maximum and sum of a row's part, then its weighted rows)
    // where a row has more than one part
    float2* part_ml;
    float* part_o;
    // sequences of at most this many rows (new tokens * group) are the few-row
    // kernel's, the others the tile kernel's
    int32_t few_rows;
    int32_t* err;
};

// Rows of a KV head that the few-row kernel takes: two blocks of 16, one where
// two would not leave registers for the tile in flight.
inline int FewMost(int head_dim) { return head_dim <= 128 ? 32 : 16; }
constexpr int kFewKeys = 32;   // positions of its unit of work
constexpr int kFewHeads = 8;   // most KV heads of its workgroup

// Launches on `stream`; type and cache_type choose the instance.
// Waves of a few-row workgroup: 8, or 4 where the registers of 8 would not do.
inline int FewWaves(int head_dim, int few_rows) { return head_dim <= 128 && few_rows <= 16 ? 8 : 4; }
// Most workgroups of a launch (512 threads each, below 2^32 in all), and of a call:
// what is not split goes over as many launches as it takes.
constexpr int64_t kMaxBlocks = 1 << 22, kMaxCallBlocks = int64_t{1} << 35;
int64_t TileBlocks(const RaggedParams& p);
mlk_status LaunchFew(const RaggedParams& p, int32_t type, int32_t cache_type, hipStream_t stream);
// Rows of a tile: 8 waves' 32 each, 4 waves' where a row's results take twice the
// registers.
__host__ __device__ constexpr int TileRows(int head_dim) { return head_dim <= 128 ? 256 : 128; }
mlk_status LaunchTile(const RaggedParams& p, int32_t type, int32_t cache_type, hipStream_t stream);

// f.template Run<A, C>() for the types.
template <typename F>
mlk_status ByType(int32_t type, int32_t cache_type, const F& f) {
    if (type == MLK_F16) return f.template Run<F16, F16>();
    if (type == MLK_BF16) return f.template Run<BF16, BF16>();
    if (cache_type == MLK_F16) return f.template Run<F32, F16>();
    if (cache_type == MLK_BF16) return f.template Run<F32, BF16>();
    return f.template Run<F32, F32>();
}

// The few-row kernel's work: units of kFewKeys positions, sequence by sequence,
// block of KV heads by block.  Worker w takes units w * share .. + share - 1,
// whatever sequences they belong to, so lengths of all kinds load the device
// evenly; of the (sequence, block) pairs in its range only the first and the last
// can be other workers' too, so it leaves at most two partial results a row.
// Everything follows from the lengths on the device: a captured call divides
// what it finds at its replay.
struct FewWork {
    int64_t share;
    int32_t heads;  // KV heads of a block, a power of two up to kFewHeads
    // the sequence looked for: its units and those of the sequences before it
    int64_t before;
    int32_t s, units;
};

// (A short sequence counts kFewRun units, what it costs; those past its length
// hold nothing.)
constexpr int kFewRun = 8;
__device__ inline int32_t FewUnits(const RaggedParams& p, int s) {
    Seq q;
    if (s >= p.batch.n_seqs || !LoadSeq(p.batch, s, &q)) return 0;
    if (q.n == 0 || static_cast<int64_t>(q.n) * p.group > p.few_rows) return 0;
    const int32_t units = (q.len + kFewKeys - 1) / kFewKeys;
    return units > kFewRun ? units : kFewRun;
}

// Units of all sequences, and of those before sequence `upto` (a whole wave;
// every lane gets them).
__device__ inline int64_t CountFewUnits(const RaggedParams& p, int upto, int64_t* before) {
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    int64_t total = 0;
    *before = 0;
    for (int s0 = 0; s0 < p.batch.n_seqs; s0 += kWave) {
        int64_t u = FewUnits(p, s0 + lane), b = s0 + lane < upto ? u : 0;
        for (int off = kWave / 2; off > 0; off /= 2) {
            u += __shfl_xor(u, off, kWave);
            b += __shfl_xor(b, off, kWave);
        }
        total += u;
        *before += b;
    }
    return total;
}

// How `total` units are divided.  A workgroup's waves take neighbouring heads of
// the same positions (whole rows of the cache, read once and together) where
// that leaves every worker kFewRun units or more; else fewer heads and more
// waves per head, down to one head's positions spread over all waves.
__device__ inline void DivideFew(const RaggedParams& p, int64_t total, FewWork* w) {
    int heads = p.few_heads;
    while (heads > 1 && total * (p.n_kv_heads / heads) < static_cast<int64_t>(p.workers) * kFewRun) {
        heads /= 2;
    }
    const int64_t share = (total * (p.n_kv_heads / heads) + p.workers - 1) / p.workers;
    w->heads = heads;
    w->share = share > kFewRun ? share : kFewRun;
}

// The sequence of a worker's first unit (a whole wave; false: nothing to do).
__device__ inline bool FindFewWork(const RaggedParams& p, int64_t worker, FewWork* w) {
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    if (p.batch.n_seqs == 1) {
        w->s = 0;
        w->before = 0;
        w->units = FewUnits(p, 0);
        DivideFew(p, w->units, w);
        return worker * w->share < static_cast<int64_t>(w->units) * (p.n_kv_heads / w->heads);
    }
    int64_t before = 0, total = 0;
    if (p.batch.n_seqs > kWave) total = CountFewUnits(p, 0, &before);
    for (int s0 = 0; s0 < p.batch.n_seqs; s0 += kWave) {
        const int32_t mine = FewUnits(p, s0 + lane);
        int64_t sum = mine;  // of lanes 0 .. lane
        for (int off = 1; off < kWave; off *= 2) {
            const int64_t v = __shfl_up(sum, off, kWave);
            if (lane >= off) sum += v;
        }
        const int64_t here = __shfl(sum, kWave - 1, kWave);
        if (s0 == 0) {
            if (p.batch.n_seqs <= kWave) total = here;
            DivideFew(p, total, w);
        }
        const int64_t blocks = p.n_kv_heads / w->heads, target = worker * w->share;
        if (target >= total * blocks) return false;
        const uint64_t past = __ballot((before + sum) * blocks > target);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            w->s = s0 + at;
            w->units = __builtin_amdgcn_readlane(mine, at);
            w->before = before + __shfl(sum, at, kWave) - w->units;
            return true;
        }
        before += here;
    }
    return false;
}

// Where the partial of row m lies: few-row kernel, by worker, place in its range
// (0: its first pair, 1: its last) and head of the block; tile kernel, by token row.
__device__ inline int64_t FewPartial(const RaggedParams& p, int64_t worker, int place, int head,
                                     int m) {
    return ((worker * 2 + place) * kFewHeads + head) * p.few_rows + m;
}
__device__ inline int64_t TilePartial(const RaggedParams& p, int32_t t, int h) {
    return (static_cast<int64_t>(t) * p.n_heads + h) * p.n_chunks;
}

// How rows lie.  kFull: head_dim is the instance's and rows are 16-byte aligned.
// kPadded: aligned, head_dim a smaller multiple of 8; runs past it read the row's
// first elements instead (K's meet q's zeros, V's results are not kept).  kScalar:
// anything else, element by element.
enum Lie { kScalar = 0, kPadded = 1, kFull = 2 };
inline Lie LieOf(const RaggedParams& p, int head_dim) {
    return !p.vec ? kScalar : p.rows.head_dim == head_dim ? kFull : kPadded;
}

// Elements d .. d + N - 1 of a K, V or q row, as raw bits; kOnce: no other workgroup
// reads them (a non-temporal load); kZero: zeros past hd.
template <typename C, int N, Lie kLie, bool kOnce, bool kZero = false>
__device__ inline void LoadRun(const typename C::Bits* row, int d, int hd, uint32_t* o) {
    constexpr int W = N * static_cast<int>(sizeof(typename C::Bits)) / 4;
    if constexpr (kLie == kScalar) {
#pragma unroll
        for (int i = 0; i < W; ++i) o[i] = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (d + i < hd) {
                if constexpr (sizeof(typename C::Bits) == 4) o[i] = __float_as_uint(row[d + i]);
                else o[i / 2] |= static_cast<uint32_t>(row[d + i]) << (16 * (i % 2));
            }
        }
    } else {
        const bool in = kLie == kFull || d < hd;
        const typename C::Bits* p = row + (in ? d : 0);
        constexpr int V = W < 4 ? W : 4;
        typedef uint32_t Vec __attribute__((ext_vector_type(V)));
#pragma unroll
        for (int i = 0; i < W / V; ++i) {
            const Vec v = kOnce ? __builtin_nontemporal_load(reinterpret_cast<const Vec*>(p) + i)
                                : reinterpret_cast<const Vec*>(p)[i];
#pragma unroll
            for (int e = 0; e < V; ++e) o[V * i + e] = kZero && !in ? 0u : v[e];
        }
    }
}

}  // namespace mlk
