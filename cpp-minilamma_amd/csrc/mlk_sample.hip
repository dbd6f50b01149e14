// mlk_sample.hip -- the next token of each row of logits: temperature, top-k,
// top-p and min-p, from given uniform numbers.
//
// In descending order of the logits (the lower index first where they are equal),
// with w_i = exp((x_i - x_1) / T) and C_n = w_1 + .. + w_n, the tokens kept are the
// first n = max(1, min(n_k, n_p, n_m)), and the one chosen is the first with C_i >
// u C_n.  Each cut, and the choice itself, is the place in that order where a count
// or a sum crosses a bound.  A row is not sorted for it: bins of 1/32 of a
// temperature (b = rint(32 x / T), whatever the row's maximum is) say in which bin
// each bound is crossed, and only the elements of those bins are looked at again.
//
// SampleBins (the one read of all logits, up to kMaxParts workgroups a row): every wave
// has a histogram of its own in shared memory, a ring of the 1024 bins up to the largest
// it has met (32 temperatures; what drops out weighs below 2^-45 of the row's largest), so
// nothing waits for the maximum.  A weight is kept relative to its bin's middle, exp(f / 32)
// with |f| <= 1/2: a polynomial of degree 5 in float64 (Taylor's, within 2^-45), as a
// whole number of 2^-42.  Sums of whole numbers depend on no order: a row's bins, and so its
// token, are the same for every division of the work and every batch.  Rows with a top-k
// count instead, and evaluate no weights.  The largest of every 128 bytes is noted.
//
// SampleChoose, kCuts (a workgroup a row): the parts' bins are added and scanned, which gives
// the bins where the bounds are crossed.  SampleGather (many a row): the logits of those bins
// into a list; 128 bytes are read again only if their largest reaches the lowest bin looked
// for.  SampleChoose, kFinish (a workgroup a row, of twice the threads where rows are few): where the list is all that can be kept and
// no longer than kFewAll, it is put in order by comparison and every cut is a count; else
// the crossing is found in its bin by 1024 equal ranges of the bin, then (equal logits) of the
// keys.  A bin of more elements than the list holds (nearly equal logits, high temperatures)
// is narrowed by the digits of the order's key (logit bits, then index), pass by pass over
// the row.  Of few rows the three are one launch, kOneLaunch, in which every workgroup of the
// gathering adds up the bins for itself and the one that ends last finishes.  Rows of up to
// kList logits are one launch alone, kSmall, with everything in the list.
//
// What bounds it: 512 fp32 rows of 128256 of mixed settings (263 MB, 56 us at a copy's rate)
// 123 to 130 us: SampleBins 67 to 70 (with a top-k, or at temperature 0, 55: the bytes; weights cost
// the rest, float64 and additions in shared memory), cuts 8, gather 28, finish 20, as each takes
// by itself.  64 bf16 rows 54 us, one fp32 row 28, 6 fp32 rows of 131 7: a few launches, each a
// chain of loads, scans and barriers.
#include "mlk_paged.h"

#include <cmath>
#include <type_traits>

namespace mlk {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / kWave;  // first pass
constexpr int kChooseThreads = 256, kChooseWaves = kChooseThreads / kWave;  // the later ones
constexpr int kBins = 1024;     // of a histogram, a power of two
constexpr int kPerUnit = 32;    // bins of a temperature
constexpr int kList = 4096;     // elements gathered at once
constexpr int kFewAll = kChooseThreads;  // of a list that is put in order as a whole
constexpr int kChunk = 1024;    // segments looked at at once
constexpr int kWideThreads = 512, kMostWaves = kWideThreads / kWave;  // of kFinish where rows are few
constexpr int kMaxParts = 48;   // workgroups of a row
constexpr int64_t kMaxVocab = 1 << 20, kMaxRows = 1 << 20;
constexpr double kOne = 0x1p42;  // a weight of 1
constexpr int kAhead = 4;       // 16-byte loads a lane has in flight
constexpr int kSegment = 8;     // lanes (16 bytes each) whose largest is noted together

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long ull;

// What a workgroup of the first pass leaves behind, then kBins masses (or counts),
// from its largest bin down.
struct Part {
    int32_t top;     // its largest bin
    uint32_t flags;  // kSome, kNan
    uint64_t best;   // temperature 0: the order's first
    float largest;   // logit
    int32_t unused[3];
};
constexpr uint32_t kSome = 1, kNan = 2;
constexpr int64_t kPartBytes = sizeof(Part) + kBins * 8;

// What the second pass leaves of a row for the two that follow, then the kBins masses (or
// counts) of its bins, then kList keys.
struct RowState {  // 48 bytes
    int32_t top;     // its largest bin
    float largest;   // logit
    float al, ah, bl, bh;  // logits to gather: al .. ah and bl .. bh
    uint32_t live;   // kChosen: its token is; kAll: what is gathered is all that can be kept
    uint32_t n;      // how many were gathered
    uint64_t reach;  // the sum that top-p asks for; with a top-k, 0: it follows from that
    uint32_t done;   // kOneLaunch: workgroups of the row that have gathered theirs
    uint32_t unused;  // (whole 16 bytes)
};
constexpr uint32_t kChosen = 0, kLive = 1, kAll = 2;
constexpr int64_t kStateBytes = sizeof(RowState) + kBins * 8 + kList * 8;

struct SampleArgs {
    const void* x;
    int64_t row;  // elements
    int32_t vocab, parts, segments;
    mlk_sampling how;
    const float* u;
    int32_t* tokens;
    float* prob;
    char* part;      // [rows][parts] of kPartBytes
    char* state;     // [rows] of kStateBytes
    float* largest;  // [rows][segments]
    int32_t* err;
};

// A row's settings.
struct How {
    double c;      // bins per unit of a logit
    float limit;   // of a logit's size
    float t, p, m, u;
    int32_t k;     // 0: all
    bool bad;
};

__device__ inline How HowOf(const SampleArgs& a, int64_t row) {
    How h;
    h.t = a.how.temperature != nullptr ? a.how.temperature[row] : 1.0f;
    h.k = a.how.top_k != nullptr ? a.how.top_k[row] : 0;
    h.p = a.how.top_p != nullptr ? a.how.top_p[row] : 1.0f;
    h.m = a.how.min_p != nullptr ? a.how.min_p[row] : 0.0f;
    h.u = h.t == 0.0f ? 0.0f : a.u[row];
    h.bad = !(h.t >= 0.0f) || !(h.u >= 0.0f && h.u < 1.0f) || h.p != h.p || h.m != h.m;
    if (h.m > 1.0f) {  // none weighs as much: the first alone
        h.k = 1;
        h.m = 0.0f;
    }
    if (h.k <= 0 || h.k >= a.vocab) h.k = 0;
    const float t = fmaxf(h.t, 0x1p-14f);
    h.c = kPerUnit / static_cast<double>(t);
    h.limit = fminf(t * 0x1p24f, 0x1.fffffep127f);
    return h;
}

// Bin of a logit (at most 2^29 in size by the limit) and its place f in it.
__device__ inline int32_t BinOf(const How& h, float x, double* f) {
    const double v = __builtin_amdgcn_fmed3f(x, -h.limit, h.limit);
    constexpr double kRound = 0x1.8p52;
    const double t = fma(v, h.c, kRound);
    *f = fma(v, h.c, -(t - kRound));
    return static_cast<int32_t>(__double2loint(t));
}
__device__ inline int32_t BinOf(const How& h, float x) {
    double f;
    return BinOf(h, x, &f);
}

// exp(f / kPerUnit) 2^42 as a whole number.
__device__ inline uint64_t Weight(double f) {
    constexpr double z = 1.0 / kPerUnit;
    double e = z * z * z * z * z / 120 * kOne;
    e = fma(e, f, z * z * z * z / 24 * kOne);
    e = fma(e, f, z * z * z / 6 * kOne);
    e = fma(e, f, z * z / 2 * kOne);
    e = fma(e, f, z * kOne);
    e = fma(e, f, kOne + 0x1p52);  // the sum's last bit is 1: rounded to a whole number
    return static_cast<uint64_t>(__double_as_longlong(e)) & 0xFFFFFFFFFFFFFull;
}

// Descending order of logits as ascending whole numbers; equal for +0 and -0.
__device__ inline uint32_t Descending(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b >> 31 ? b : ~b & 0x7FFFFFFFu;
}
__device__ inline float Logit(uint32_t key) {
    return __uint_as_float(key >> 31 ? key : ~key & 0x7FFFFFFFu);
}
__device__ inline uint64_t Key(float x, int32_t i) {
    return (static_cast<uint64_t>(Descending(x)) << 32) | static_cast<uint32_t>(i);
}

constexpr uint64_t kNoKey = ~uint64_t{0}, kLastKey = kNoKey - 1;  // past every element's

// The least logit that weighs anything beside a row's (or a part's) largest: all numbers do as
// far as their bins say, but beside infinity only its equals.
__device__ inline float LeastOf(float largest) {
    return largest < INFINITY ? -0x1.fffffep127f : INFINITY;
}

// A row as units of 16 bytes from the last 16-byte boundary at or before it.
template <typename T>
struct RowUnits {
    static constexpr int E = 16 / sizeof(typename T::Bits);
    const typename T::Bits* x;
    int32_t vocab, skip;  // elements of the first unit that are before the row
    __device__ RowUnits(const SampleArgs& a, int64_t row) {
        x = static_cast<const typename T::Bits*>(a.x) + row * a.row;
        vocab = a.vocab;
        skip = static_cast<int32_t>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(typename T::Bits));
    }
    __device__ int32_t Units() const { return (skip + vocab + E - 1) / E; }
    __device__ int32_t Index(int32_t unit, int e) const { return unit * E - skip + e; }
    static constexpr uint32_t kNone = E == 4 ? 0xFF800000u : T::kType == MLK_F16 ? 0xFC00FC00u : 0xFF80FF80u;
    // A unit's bits, -infinity where it reaches out of the row or is not `there`.
    __device__ u32x4 Load(int32_t unit, bool there) const {
        const int32_t i = Index(unit, 0);
        u32x4 raw = {kNone, kNone, kNone, kNone};
        if (there && i >= 0 && i + E <= vocab) {
            raw = *reinterpret_cast<const u32x4*>(x + i);
        } else if (there) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (i + e >= 0 && i + e < vocab) {
                    if constexpr (E == 4) {
                        raw[e] = __float_as_uint(x[i + e]);
                    } else {
                        const uint32_t b = x[i + e];
                        raw[e / 2] = e % 2 ? (raw[e / 2] & 0xFFFFu) | b << 16 : (raw[e / 2] & 0xFFFF0000u) | b;
                    }
                }
            }
        }
        return raw;
    }
    static __device__ float Get(const u32x4& raw, int e) {
        if constexpr (E == 4) return __uint_as_float(raw[e]);
        else return T::Get(static_cast<uint16_t>(raw[e / 2] >> (16 * (e % 2))));
    }
};

template <int kCtrl>
__device__ inline float MaxDpp(float v) {
    const int o = __builtin_amdgcn_update_dpp(0, static_cast<int>(__float_as_uint(v)), kCtrl, 0xF, 0xF, true);
    return fmaxf(v, __uint_as_float(static_cast<uint32_t>(o)));
}
// Largest of the 8 lanes of a segment, and of the wave from there.
__device__ inline float Max8(float v) {
    v = MaxDpp<0xB1>(v);         // lanes l ^ 1
    v = MaxDpp<0x4E>(v);         // l ^ 2
    return MaxDpp<0x141>(v);     // mirrored within 8
}
__device__ inline float MaxFrom8(float v) {
    v = MaxDpp<0x140>(v);        // mirrored within 16
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}

// ------------------------------------------------------------ first pass

template <typename T>
__global__ __launch_bounds__(kThreads) void SampleBins(const SampleArgs p) {
    constexpr int E = RowUnits<T>::E;
    __shared__ uint64_t hist[kWaves][kBins];  // sums; counts in the low halves of the first
    __shared__ int32_t tops[kWaves];
    __shared__ uint32_t flags_of[kWaves];
    __shared__ uint64_t best_of[kWaves];
    __shared__ float largest_of[kWaves];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int64_t row = blockIdx.x / p.parts;
    const int part = static_cast<int>(blockIdx.x % p.parts);
    const How h = HowOf(p, row);
    if (h.bad) return;  // the second pass sees that too
    if (part == 0 && tid == 0) {
        RowState* state = reinterpret_cast<RowState*>(p.state + row * kStateBytes);
        state->n = 0;
        state->done = 0;
    }
    const RowUnits<T> r(p, row);
    const int32_t units = r.Units(), blocks = (units + kWave - 1) / kWave;
    const int32_t b0 = static_cast<int32_t>(static_cast<int64_t>(blocks) * part / p.parts);
    const int32_t b1 = static_cast<int32_t>(static_cast<int64_t>(blocks) * (part + 1) / p.parts);
    uint64_t* mass = hist[wave];
    uint32_t* count = reinterpret_cast<uint32_t*>(mass);
    for (int i = lane; i < kBins; i += kWave) mass[i] = 0;
    bool some = false, nan = false;
    int32_t top = 0;
    float so_far = -INFINITY;
    uint64_t best = ~uint64_t{0};
    float* largest = p.largest + row * p.segments;

    // neighbouring blocks for each wave, the same number or one less
    const int32_t w0 = b0 + (b1 - b0) * wave / kWaves, w1 = b0 + (b1 - b0) * (wave + 1) / kWaves;
    for (int32_t b = w0; b < w1; b += kAhead) {
        u32x4 raw[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int32_t unit = (b + a) * kWave + lane;
            raw[a] = r.Load(unit, b + a < w1 && unit < units);
        }
        float v[kAhead][E];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[a][e] = r.Get(raw[a], e);
        }
        float all = -INFINITY;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            float m = v[a][0];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                nan |= v[a][e] != v[a][e];
                m = fmaxf(m, v[a][e]);
            }
            m = Max8(m);
            if (b + a < w1 && lane % kSegment == 0) {
                const int32_t seg = ((b + a) * kWave + lane) / kSegment;
                if (seg < p.segments) largest[seg] = m;
            }
            all = fmaxf(all, m);
        }
        all = MaxFrom8(all);
        if (h.t == 0.0f) {
            if (all < so_far) continue;
            so_far = all;
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const uint64_t k = v[a][e] > -INFINITY
                                           ? Key(v[a][e], r.Index((b + a) * kWave + lane, e)) : ~uint64_t{0};
                    best = k < best ? k : best;
                }
            }
            continue;
        }
        if (all > so_far) {  // (uniform) the ring moves on: what it now holds anew was far below
            so_far = all;
            const int32_t to = BinOf(h, all);
            if (some) {
                // (beside infinity all that was before is)
                const int32_t fresh = all < INFINITY && to - top < kBins ? to - top : kBins;
                for (int32_t i = lane; i < fresh; i += kWave) mass[(to - i) & (kBins - 1)] = 0;
            }
            top = to;
            some = true;
        }
        if (!some) continue;
        if (so_far == INFINITY) {  // its equals count alone, each the same
            uint32_t n = 0;
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
#pragma unroll
                for (int e = 0; e < E; ++e) n += v[a][e] == INFINITY ? 1 : 0;
            }
            double f;
            const int32_t at = BinOf(h, INFINITY, &f) & (kBins - 1);
            if (n != 0) atomicAdd(reinterpret_cast<ull*>(&mass[at]), static_cast<ull>(h.k != 0 ? n : n * Weight(f)));
            continue;
        }
        auto add = [&](auto counts) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                if (b + a >= w1) break;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    double f;
                    const int32_t at = BinOf(h, v[a][e], &f);
                    if (!(v[a][e] > -INFINITY) || static_cast<uint32_t>(top - at) >= kBins) continue;
                    if constexpr (decltype(counts)::value) atomicAdd(&count[2 * (at & (kBins - 1))], 1u);
                    else atomicAdd(reinterpret_cast<ull*>(&mass[at & (kBins - 1)]), static_cast<ull>(Weight(f)));
                }
            }
        };
        if (h.k != 0) add(std::true_type{});
        else add(std::false_type{});
    }
    nan = __ballot(nan) != 0;
    if (h.t == 0.0f) {
#pragma unroll
        for (int off = kWave / 2; off > 0; off /= 2) {
            const uint64_t o = __shfl_xor(static_cast<ull>(best), off, kWave);
            best = o < best ? o : best;
        }
        some = best != ~uint64_t{0};
    }
    if (lane == 0) {
        tops[wave] = top;
        flags_of[wave] = (some ? kSome : 0) | (nan ? kNan : 0);
        best_of[wave] = best;
        largest_of[wave] = so_far;
    }
    __syncthreads();
    uint32_t flags = 0;
    int32_t all_top = INT32_MIN;
    float most = -INFINITY;
    for (int w = 0; w < kWaves; ++w) {
        flags |= flags_of[w];
        if ((flags_of[w] & kSome) && tops[w] > all_top) all_top = tops[w];
        if (best_of[w] < best) best = best_of[w];
        most = fmaxf(most, largest_of[w]);
    }
    // (a wave that met an infinity has the largest bin; those that met none count for nothing then)
    const float least = LeastOf(most);
    Part* out = reinterpret_cast<Part*>(p.part + blockIdx.x * kPartBytes);
    if (tid == 0) *out = {all_top, flags, best, most, {}};
    if (h.t == 0.0f || !(flags & kSome)) return;
    uint64_t* bins = reinterpret_cast<uint64_t*>(out + 1);
    for (int i = tid; i < kBins; i += kThreads) {
        const int32_t at = all_top - i;
        uint64_t sum = 0;
        for (int w = 0; w < kWaves; ++w) {
            if ((flags_of[w] & kSome) && largest_of[w] >= least && static_cast<uint32_t>(tops[w] - at) < kBins) {
                sum += hist[w][at & (kBins - 1)];
            }
        }
        bins[i] = sum;
    }
}

// ------------------------------------------------------------ second pass

// Inclusive sums over the workgroup's threads, in a fixed order; *total over all.
template <int kWaves, typename V>
__device__ inline V ScanBlock(V v, V* scratch, V* total) {
    const int lane = static_cast<int>(threadIdx.x) % kWave, wave = static_cast<int>(threadIdx.x) / kWave;
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) {
        const V o = __shfl_up(v, off, kWave);
        if (lane >= off) v += o;
    }
    __syncthreads();
    if (lane == kWave - 1) scratch[wave] = v;
    __syncthreads();
    V before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i == wave) before = all;
        all += scratch[i];
    }
    *total = all;
    return before + v;
}

struct Choice {
    uint64_t list[kList];  // keys of gathered elements
    uint32_t code[kList];  // their bins, and where in them: CodeOf
    uint64_t bin[kBins];   // masses or counts of the bins; of a search's ranges
    uint64_t sum[kBins];   // of the weights up to and with bin i, of the largest bin's middle
    uint16_t some[kList];  // segments to look through; places in the list that a search is left with
    uint64_t few[kWave];
    double edge[2 * kPerUnit];  // exp(-i / kPerUnit), and exp(-i)
    uint64_t scan_u[kMostWaves], scan_v[kMostWaves];
    int32_t found[2];
    uint32_t n_list, n_segments, n_few;
    uint64_t word[3];
};

enum Bound { kCount, kReach, kPass };  // count >= bound, sum >= bound, sum > bound

// The first place in a bin's order that meets a bound: its key, the sum before it and its
// own weight (whole numbers).
struct Place {
    uint64_t key, before, own;
};

// Bins lo .. hi.
struct Span {
    int lo, hi;
    __device__ bool Has(int b) const { return b >= lo && b <= hi; }
};

template <typename T, int kT>  // kT threads
struct Chooser {
    static constexpr int kW = kT / kWave, kEach = kBins / kT;  // neighbouring bins a thread has
    const SampleArgs& p;
    const How& h;
    Choice& s;
    RowUnits<T> r;
    const float* largest;
    int32_t top;
    float least;     // of the row's logits, what is smaller weighs nothing
    uint64_t limit;  // keys past it are cut off by top-k

    __device__ int Tid() const { return static_cast<int>(threadIdx.x); }
    __device__ int Lane() const { return Tid() % kWave; }
    __device__ int Wave() const { return __builtin_amdgcn_readfirstlane(Tid() / kWave); }
    __device__ int BinOfKey(uint64_t key, double* f) const {
        return top - BinOf(h, Logit(static_cast<uint32_t>(key >> 32)), f);
    }
    // A bin's middle, of the largest bin's: exp(-bin / kPerUnit), as a product of two.
    static_assert(kBins == kPerUnit * kPerUnit, "two tables of kPerUnit");
    __device__ double Edge(int bin) const { return s.edge[bin % kPerUnit] * s.edge[kPerUnit + bin / kPerUnit]; }
    __device__ void MakeEdges() {  // (a barrier follows)
        if (Tid() < 2 * kPerUnit) s.edge[Tid()] = exp(Tid() < kPerUnit ? Tid() * (-1.0 / kPerUnit) : static_cast<double>(kPerUnit - Tid()));
    }
    __device__ double WeightOf(float x) const {
        double f;
        const int32_t b = top - BinOf(h, x, &f);
        return static_cast<double>(Weight(f)) * Edge(b);
    }
    // Which of kBins equal ranges of its bin an element lies in, from the largest down.
    static __device__ int RangeOf(double place) {
        const int i = static_cast<int>((0.5 - place) * kBins);
        return i < 0 ? 0 : i < kBins ? i : kBins - 1;
    }
    __device__ uint32_t CodeOf(uint64_t key) const {
        double place;
        const int b = BinOfKey(key, &place);
        return key <= kLastKey && b >= 0 && b < kBins ? static_cast<uint32_t>(b * kBins + RangeOf(place)) : ~0u;
    }
    __device__ void PutInList(int at, uint64_t key) {
        s.list[at] = key;
        s.code[at] = CodeOf(key);
    }
    __device__ uint64_t Below(int bin) const { return bin > 0 ? s.sum[bin - 1] : 0; }
    // Whole weights of a bin as those of the largest bin's middle; of that bin itself they stay as
    // they are (float64 holds no sum of over 2^53: of equal logits all bounds are exact).
    __device__ uint64_t Scaled(uint64_t w, int bin) {
        return bin == 0 ? w : static_cast<uint64_t>(rint(static_cast<double>(w) * Edge(bin)));
    }

    // Logits no smaller (larger) than any of bin `bin`, to within a thousandth of a bin and a
    // rounding; -infinity is below all (bins of the highest temperatures reach past the numbers).
    __device__ float Lowest(int bin) const {
        const double b = static_cast<double>(top) - bin;
        if (!(h.c > 0.0) || b <= -0x1p28) return least;
        const double x = (b - 0.501) / h.c;
        return fmaxf(static_cast<float>(x - fabs(x) * 0x1p-23), least);
    }
    __device__ float Highest(int bin) const {
        const double b = static_cast<double>(top) - bin;
        if (!(h.c > 0.0) || bin == 0 || b >= 0x1p28) return INFINITY;
        const double x = (b + 0.501) / h.c;
        return static_cast<float>(x + fabs(x) * 0x1p-23);
    }

    // The segments c0 .. c0 + kChunk - 1 whose largest is at least `low` into s.segment; how many.
    __device__ int Segments(int32_t c0, int32_t segments, float low) {
        __syncthreads();
        if (Tid() == 0) s.n_segments = 0;
        __syncthreads();
        float m[kChunk / kT];
#pragma unroll
        for (int i = 0; i < kChunk / kT; ++i) {
            const int32_t seg = c0 + i * kT + Tid();
            m[i] = seg < segments ? largest[seg] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < kChunk / kT; ++i) {
            const bool hit = m[i] >= low;
            const uint64_t mask = __ballot(hit);
            if (mask == 0) continue;
            uint32_t at = 0;
            if (Lane() == 0) at = atomicAdd(&s.n_segments, static_cast<uint32_t>(__popcll(mask)));
            at = __builtin_amdgcn_readfirstlane(at) + __popcll(mask & ((uint64_t{1} << Lane()) - 1));
            if (hit) s.some[at] = static_cast<uint16_t>(i * kT + Tid());
        }
        __syncthreads();
        return static_cast<int>(s.n_segments);
    }

    // The elements of a bin (and a few of its neighbours) into s.list; how many there are (of
    // more than kList, not all are there).
    __device__ int Gather(int bin) {
        if (Tid() == 0) s.n_list = 0;  // (a barrier follows in Segments)
        Near({bin, bin}, [&](float x, int32_t i) {
            const uint32_t at = atomicAdd(&s.n_list, 1u);
            if (at < kList) PutInList(static_cast<int>(at), Key(x, i));
        });
        return static_cast<int>(s.n_list);
    }

    // f(logit, index) over the row's elements near a span of bins: of each 128 bytes whose
    // largest is no lower than those.
    template <typename F>
    __device__ void Near(const Span& span, const F& f) {
        constexpr int kElements = kSegment * RowUnits<T>::E;  // of a segment
        const float low = Lowest(span.hi), high = Highest(span.lo);
        const int32_t segments = (r.Units() + kSegment - 1) / kSegment;
        for (int32_t c0 = 0; c0 < segments; c0 += kChunk) {
            const int n = Segments(c0, segments, low);
#pragma unroll 1
            for (int j = Tid(); j < n * kElements; j += kT) {
                const int32_t i = r.Index((c0 + s.some[j / kElements]) * kSegment, j % kElements);
                const float x = i >= 0 && i < r.vocab ? T::Get(r.x[i]) : -INFINITY;
                if (x >= low && x <= high) f(x, i);
            }
        }
        __syncthreads();
    }
    // f(bin, place in it, key) over the row's elements of a span of bins, up to the limit.
    template <typename F>
    __device__ void Visit(const Span& span, const F& f) {
        Near(span, [&](float x, int32_t i) {
            double place;
            const uint64_t key = Key(x, i);
            const int b = BinOfKey(key, &place);
            if (span.Has(b) && key <= limit) f(b, place, key);
        });
    }
    // The same over the first n of s.list; f(bin, place, key, code).
    template <typename F>
    __device__ void InList(int n, const Span& span, const F& f) {
#pragma unroll 2
        for (int i = Tid(); i < n; i += kT) {
            const uint32_t code = s.code[i];
            if (!span.Has(static_cast<int>(code / kBins))) continue;
            const uint64_t key = s.list[i];
            double place;
            const int b = BinOfKey(key, &place);
            if (key <= limit) f(b, place, key, code);
        }
        __syncthreads();
    }

    // Least and largest over the workgroup.
    __device__ void MinMax(uint64_t* lo, uint64_t* hi) {
#pragma unroll
        for (int off = kWave / 2; off > 0; off /= 2) {
            const uint64_t a = __shfl_xor(static_cast<ull>(*lo), off, kWave), b = __shfl_xor(static_cast<ull>(*hi), off, kWave);
            *lo = a < *lo ? a : *lo;
            *hi = b > *hi ? b : *hi;
        }
        __syncthreads();
        if (Lane() == 0) {
            s.scan_u[Wave()] = *lo;
            s.scan_v[Wave()] = *hi;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kW; ++i) {
            *lo = s.scan_u[i] < *lo ? s.scan_u[i] : *lo;
            *hi = s.scan_v[i] > *hi ? s.scan_v[i] : *hi;
        }
    }

    __device__ void ClearBins() {
        for (int i = Tid(); i < kBins; i += kT) s.bin[i] = 0;
    }
    __device__ void AddTo(int range, uint64_t w) {
        atomicAdd(reinterpret_cast<ull*>(&s.bin[range]), static_cast<ull>(w));
    }
    // A step of a search: s.bin holds what lies in kBins ranges of the order (counts or
    // sums); the first range where the bound is met after *before, or the last that holds
    // any.  *before: with what lies before that range; *held: what it holds.
    __device__ int Narrow(Bound what, uint64_t bound, uint64_t* before, uint64_t* held) {
        uint64_t w[kEach], mine = 0, all;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            w[i] = s.bin[Tid() * kEach + i];
            mine += w[i];
        }
        uint64_t sum = *before + ScanBlock<kW>(mine, s.scan_u, &all) - mine;
        all += *before;
        // (a bound past the end: the last place)
        if (what == kPass ? bound >= all : bound > all) bound = what == kPass ? all - 1 : all;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint64_t upto = sum + w[i];
            if (what == kPass ? upto > bound && sum <= bound : upto >= bound && sum < bound) {
                s.found[0] = Tid() * kEach + i;
                s.word[0] = sum;
                s.word[1] = w[i];
            }
            sum = upto;
        }
        __syncthreads();
        *before = s.word[0];
        *held = s.word[1];
        const int at = s.found[0];
        __syncthreads();
        return at;
    }

    // The first place of bin `bin`, all of whose elements are in the list of n, to meet the
    // bound: by equal ranges of the bin, then (equal logits) by ranges of the keys that are
    // left, until a wave holds them.
    __device__ Place Select(int n, int bin, Bound what, uint64_t bound) {
        uint64_t before = 0, held, least = kNoKey, most = 0;
        ClearBins();
        if (Tid() == 0) s.n_few = 0;
        __syncthreads();
        if (n > kWave) {
            InList(n, {bin, bin}, [&](int, double place, uint64_t, uint32_t code) {
                AddTo(static_cast<int>(code % kBins), what == kCount ? 1 : Weight(place));
            });
        }
        const uint32_t code = static_cast<uint32_t>(bin) * kBins + (n > kWave ? Narrow(what, bound, &before, &held) : 0);
        // that range's (of a short list, the bin's) places
        for (int i0 = 0; i0 < n; i0 += kT) {
            const int i = i0 + Tid();
            bool in = i < n && (n > kWave ? s.code[i] == code : s.code[i] / kBins == static_cast<uint32_t>(bin));
            uint64_t mask = __ballot(in);
            if (mask == 0) continue;
            const uint64_t key = in ? s.list[i] : kNoKey;
            in = in && key <= limit;
            mask = __ballot(in);
            uint32_t at = 0;
            if (Lane() == 0) at = atomicAdd(&s.n_few, static_cast<uint32_t>(__popcll(mask)));
            at = __builtin_amdgcn_readfirstlane(at) + __popcll(mask & ((uint64_t{1} << Lane()) - 1));
            if (in) {
                s.some[at] = static_cast<uint16_t>(i);
                least = key < least ? key : least;
                most = key > most ? key : most;
            }
        }
        __syncthreads();
        int m = static_cast<int>(s.n_few);
        uint64_t lo = 0, hi = kLastKey;
        while (m > kWave) {
            MinMax(&least, &most);
            int shift = 0;
            while ((most - least) >> shift >= kBins) ++shift;
            ClearBins();
            __syncthreads();
            for (int i = Tid(); i < m; i += kT) {
                double place;
                const uint64_t key = s.list[s.some[i]];
                BinOfKey(key, &place);
                AddTo(static_cast<int>((key - least) >> shift), what == kCount ? 1 : Weight(place));
            }
            __syncthreads();
            const int at = Narrow(what, bound, &before, &held);
            lo = least + (static_cast<uint64_t>(at) << shift);
            hi = lo + ((uint64_t{1} << shift) - 1);
            least = kNoKey;
            most = 0;
            // what is left, in place: all have read theirs before any writes
            uint16_t mine[kList / kT];
            int count = 0;
            for (int i = Tid(); i < m; i += kT) {
                const uint16_t index = s.some[i];
                const uint64_t key = s.list[index];
                if (key < lo || key > hi) continue;
                least = key < least ? key : least;
                most = key > most ? key : most;
#pragma unroll
                for (int j = 0; j < kList / kT; ++j) mine[j] = j == count ? index : mine[j];
                ++count;
            }
            if (Tid() == 0) s.n_few = 0;
            __syncthreads();
            if (count > 0) {
                const uint32_t to = atomicAdd(&s.n_few, static_cast<uint32_t>(count));
#pragma unroll
                for (int j = 0; j < kList / kT; ++j) {
                    if (j < count) s.some[to + j] = mine[j];
                }
            }
            __syncthreads();
            m = static_cast<int>(s.n_few);
        }
        // one wave: every lane an element, its place by comparison with all others
        if (Tid() < kWave) {
            const bool real = Tid() < m;
            const uint64_t key = s.list[m > 0 ? s.some[real ? Tid() : 0] : 0];
            s.few[Tid()] = key;
            double place;
            BinOfKey(key, &place);
            const uint64_t own = Weight(place), one = what == kCount ? 1 : own;
            s.bin[Tid()] = one;  // (this wave alone is here)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            uint64_t sum = before;
#pragma unroll 4
            for (int i = 0; i < m; ++i) sum += s.few[i] <= key ? s.bin[i] : 0;
            const bool ok = real && (what == kPass ? sum > bound : sum >= bound);
            // the first that is ok; none: the last of all
            uint64_t best = __ballot(ok) != 0 ? (ok ? key : ~uint64_t{0}) : (real ? ~key : ~uint64_t{0});
#pragma unroll
            for (int off = kWave / 2; off > 0; off /= 2) {
                const uint64_t o = __shfl_xor(static_cast<ull>(best), off, kWave);
                best = o < best ? o : best;
            }
            if (__ballot(ok) == 0) best = ~best;
            if (real && key == best) {
                s.word[0] = key;
                s.word[1] = sum - one;
                s.word[2] = own;
            }
        }
        __syncthreads();
        const Place at{s.word[0], s.word[1], s.word[2]};
        __syncthreads();
        return at;
    }

    // The same for a bin of more elements than the list holds (nearly equal logits): by the
    // digits of their keys, pass by pass over the row.
    __device__ Place Search(int bin, Bound what, uint64_t bound) {
        uint64_t high = 0, before = 0, held;
        constexpr int kDigit = 10;
        for (int shift = 60; shift >= 0; shift -= kDigit) {
            __syncthreads();
            ClearBins();
            Visit({bin, bin}, [&](int, double place, uint64_t key) {
                if (shift < 60 && key >> (shift + kDigit) != high) return;
                AddTo(static_cast<int>(key >> shift) & (kBins - 1), what == kCount ? 1 : Weight(place));
            });
            high = (high << kDigit) | static_cast<uint64_t>(Narrow(what, bound, &before, &held));
        }
        double place;
        BinOfKey(high, &place);
        return {high, before, Weight(place)};
    }

    // A bound on the sum over all as one on whole weights within bin `bin`.
    __device__ uint64_t InBin(uint64_t bound, int bin, bool reach) const {
        if (bin == 0) return bound;
        const uint64_t below = Below(bin);
        const double in = bound > below ? static_cast<double>(bound - below) / Edge(bin) : 0.0;
        return static_cast<uint64_t>(reach ? ceil(in) : in);
    }

    // Sums over the bins from their masses.
    __device__ void SumBins() {
        uint64_t w[kEach], mine = 0, all;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            w[i] = Scaled(s.bin[Tid() * kEach + i], Tid() * kEach + i);
            mine += w[i];
        }
        uint64_t sum = ScanBlock<kW>(mine, s.scan_u, &all) - mine;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            sum += w[i];
            s.sum[Tid() * kEach + i] = sum;
        }
        __syncthreads();
    }
    // First bins up to `last` whose sum is past (reach: at least) each bound; `last` if none.
    __device__ Span FirstBins(int last, bool reach, uint64_t x, uint64_t y) {
        if (Tid() < 2) s.found[Tid()] = last;
        __syncthreads();
        for (int i = Tid(); i < last; i += kT) {
            const uint64_t sum = s.sum[i], before = Below(i);
            if (reach ? sum >= x && before < x : sum > x && (i == 0 || before <= x)) s.found[0] = i;
            if (reach ? sum >= y && before < y : sum > y && (i == 0 || before <= y)) s.found[1] = i;
        }
        __syncthreads();
        const Span at{s.found[0], s.found[1]};
        __syncthreads();
        return at;
    }
};

// The largest whole number of at most a * sum for a in [0, 1), exactly; *rest: whether it is less.
// (The arguments are all lanes' the same: scalar work.)
__device__ inline uint64_t Times(float a, uint64_t all_sum, bool* rest) {
    const uint32_t bits = __builtin_amdgcn_readfirstlane(__float_as_uint(a)) & 0x7FFFFFFFu;  // -0 is 0
    const uint64_t sum = static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(all_sum >> 32))) << 32 |
                         static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(all_sum)));
    const uint32_t e = bits >> 23;  // a = m 2^-shift
    const uint32_t m = e == 0 ? bits : (bits & 0x7FFFFFu) | 0x800000u;
    const uint32_t shift = 149 - (e == 0 ? 0 : e - 1);  // 24 .. 149
    // m * sum = high 2^32 + low
    const uint64_t p = uint64_t{m} * static_cast<uint32_t>(sum), high = uint64_t{m} * (sum >> 32) + (p >> 32);
    const uint32_t low = static_cast<uint32_t>(p);
    if (shift < 32) {
        *rest = low << (32 - shift) != 0;
        return high << (32 - shift) | low >> shift;
    }
    const uint32_t s = shift - 32;
    const uint64_t x = s < 64 ? high >> s : 0;
    *rest = low != 0 || (s < 64 ? x << s : 0) != high;
    return x;
}

__device__ inline uint64_t Share(float u, uint64_t sum) {
    bool rest;
    return Times(u, sum, &rest);
}

// The least whole sum that is at least p (below 1) of `sum`, 1 or more.
__device__ inline uint64_t Reach(float p, uint64_t sum) {
    if (!(p > 0.0f)) return 1;
    bool rest;
    const uint64_t x = Times(p, sum, &rest);
    return rest || x == 0 ? x + 1 : x;
}

// The row's logits in the two spans of `at`, in any order, into `found` (of more than kList not
// all); *n_found: how many.  8 lanes to each 128 bytes whose largest is no lower; a wave looks at
// 64 kLook segments.  `hits`: room for 64 kLook a wave.
template <typename T, int kLook>
__device__ inline void GatherPart(const RowUnits<T>& r, const float* largest, int part, const RowState& at,
                                  uint64_t* found, uint16_t* hits_of, uint32_t* n_found) {
    constexpr int E = RowUnits<T>::E, kGroups = kWave / kSegment, kRounds = 32 / E;
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int32_t units = r.Units(), segments = (units + kSegment - 1) / kSegment;
    uint16_t* hit_segment = hits_of + wave * kLook * kWave;
    const int32_t s0 = (part * kChooseWaves + wave) * kLook * kWave + lane;
    float m[kLook];
#pragma unroll
    for (int l = 0; l < kLook; ++l) m[l] = s0 + l * kWave < segments ? largest[s0 + l * kWave] : -INFINITY;
    if (threadIdx.x == 0) *n_found = 0;
    __syncthreads();
    const float al = at.al, ah = at.ah, bl = at.bl, bh = at.bh, low = fminf(al, bl);
    int n = 0;
#pragma unroll
    for (int l = 0; l < kLook; ++l) {
        const bool hit = m[l] >= low;
        const uint64_t mask = __ballot(hit);
        if (hit) hit_segment[n + __popcll(mask & ((uint64_t{1} << lane) - 1))] = static_cast<uint16_t>(s0 + l * kWave);
        n += __popcll(mask);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int g = 0; g < n; g += kGroups * kRounds) {
        u32x4 raw[kRounds];
        int32_t unit[kRounds];
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            const int j = g + i * kGroups + lane / kSegment;
            unit[i] = j < n ? hit_segment[j] * kSegment + lane % kSegment : units;
            raw[i] = r.Load(unit[i], unit[i] < units);
        }
        // which lanes' elements are in a span, then places for all of the wave's by one addition
        uint64_t in[kRounds * E];
        uint32_t all = 0;
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float x = r.Get(raw[i], e);
                in[i * E + e] = __ballot((x >= al && x <= ah) || (x >= bl && x <= bh));
                all += __popcll(in[i * E + e]);
            }
        }
        if (all == 0) continue;
        uint32_t to = 0;
        if (lane == 0) to = atomicAdd(n_found, all);
        to = __builtin_amdgcn_readfirstlane(to);
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint64_t mask = in[i * E + e];
                if (mask == 0) continue;
                const uint32_t at = to + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
                if (__builtin_amdgcn_inverse_ballot_w64(mask) && at < kList) found[at] = Key(r.Get(raw[i], e), r.Index(unit[i], e));
                to += __popcll(mask);
            }
        }
    }
    __syncthreads();
}

// What a workgroup found, behind what others have put there: one addition to the row's count.
__device__ inline void AddToList(RowState* state, const uint64_t* found, uint32_t total, uint32_t* base) {
    uint64_t* list = reinterpret_cast<uint64_t*>(state + 1) + kBins;
    if (total == 0) return;
    if (threadIdx.x == 0) *base = atomicAdd(&state->n, total);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < total && *base + i < kList; i += kChooseThreads) list[*base + i] = found[i];
}

// The passes after the first.  kCuts: which logits to gather; kFinish: the choice from what was
// gathered; kOneLaunch: these and the gathering between them, by as many workgroups as gather,
// each of which finds the cuts for itself; the last to have gathered goes on; kSmall: the choice
// from a row that the list holds whole, without any of the others.
enum Pass { kCuts, kFinish, kOneLaunch, kSmall };

template <typename T, Pass kPass_, int kT = kChooseThreads>
__global__ __launch_bounds__(kT) void SampleChoose(const SampleArgs p, int gather_parts) {
    constexpr int kW = kT / kWave, kEach = kBins / kT;
    __shared__ Choice s;
    const int tid = static_cast<int>(threadIdx.x);
    const int64_t row = kPass_ == kOneLaunch ? blockIdx.x / gather_parts : blockIdx.x;
    const int gather_part = kPass_ == kOneLaunch ? static_cast<int>(blockIdx.x % gather_parts) : 0;
    const How h = HowOf(p, row);
    const RowUnits<T> units(p, row);
    RowState* state = reinterpret_cast<RowState*>(p.state + row * kStateBytes);
    uint64_t* state_bin = reinterpret_cast<uint64_t*>(state + 1);
    uint64_t* state_list = state_bin + kBins;
    uint32_t flags = 0;
    int32_t top = INT32_MIN;
    uint64_t best = kNoKey;
    float largest = -INFINITY;
    bool all_held = kPass_ == kSmall && p.vocab <= kFewAll;  // in the list, and few
    uint64_t row_reach = 0;
    if constexpr (kPass_ == kFinish) {
        const RowState at = *state;
#pragma unroll
        for (int i = 0; i < kEach; ++i) s.bin[tid + i * kT] = state_bin[tid + i * kT];
        if (at.live == kChosen) return;
        top = at.top;
        largest = at.largest;
        all_held = at.live == kAll && at.n <= kFewAll;
        row_reach = at.reach;
    } else if constexpr (kPass_ == kCuts || kPass_ == kOneLaunch) {
        // lane i of each wave: part i
        const char* parts = p.part + row * p.parts * kPartBytes;
        static_assert(kMaxParts <= kWave, "a lane a part");
        const int lane = tid % kWave;
        if (!h.bad) {
            Part part{INT32_MIN, 0, ~uint64_t{0}, -INFINITY, {}};
            if (lane < p.parts) part = *reinterpret_cast<const Part*>(parts + lane * kPartBytes);
            flags = (__ballot(part.flags & kSome) != 0 ? kSome : 0) | (__ballot(part.flags & kNan) != 0 ? kNan : 0);
            const bool infinite = __ballot(part.largest == INFINITY) != 0;  // then other parts count for nothing
            if (!(part.flags & kSome) || (infinite && part.largest < INFINITY)) part.top = INT32_MIN;
            top = part.top;
            best = part.best;
            largest = part.largest;
#pragma unroll
            for (int off = kWave / 2; off > 0; off /= 2) {
                const int32_t t = __shfl_xor(top, off, kWave);
                top = t > top ? t : top;
                const uint64_t o = __shfl_xor(static_cast<ull>(best), off, kWave);
                best = o < best ? o : best;
                largest = fmaxf(largest, __shfl_xor(largest, off, kWave));
            }
            if (h.t != 0.0f && flags == kSome) {
                // the first bin in each part: as far below the part's largest as s.few says
                if (tid < p.parts) s.few[tid] = static_cast<uint32_t>(part.top == INT32_MIN || part.top - top < -kBins ? -kBins : part.top - top);
                __syncthreads();
                uint64_t sum[kEach] = {};
#pragma unroll 8
                for (int i = 0; i < p.parts; ++i) {
                    const uint64_t* bins = reinterpret_cast<const uint64_t*>(parts + i * kPartBytes + sizeof(Part));
                    const int32_t from = static_cast<int32_t>(s.few[i]) + tid;
#pragma unroll
                    for (int e = 0; e < kEach; ++e) {
                        const int32_t at = from + e * kT;
                        const uint64_t m = bins[at >= 0 ? at : 0];
                        sum[e] += at >= 0 ? m : 0;
                    }
                }
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    s.bin[tid + e * kT] = sum[e];
                    if (kPass_ == kCuts) state_bin[tid + e * kT] = sum[e];
                }
            }
        }
    } else {
        bool nan = false;
#pragma unroll 4
        for (int i = tid; i < p.vocab; i += kT) {
            const float x = T::Get(units.x[i]);
            const uint64_t key = x > -INFINITY ? Key(x, i) : kNoKey;
            nan |= x != x;
            largest = fmaxf(largest, x);
            s.list[i] = key;
            best = key < best ? key : best;
        }
        for (int i = tid; i < kBins; i += kT) s.bin[i] = 0;
        if (tid == 0) s.word[0] = kNoKey;
        largest = BlockMax<kW>(largest, reinterpret_cast<float*>(s.scan_u));
        flags = (largest > -INFINITY ? kSome : 0) | (__syncthreads_or(nan) ? kNan : 0);
        if (h.t == 0.0f) {
            atomicMin(reinterpret_cast<ull*>(&s.word[0]), static_cast<ull>(best));
            __syncthreads();
            best = s.word[0];
        } else if (!h.bad) {
            double f;
            top = BinOf(h, largest, &f);
        }
    }
    if constexpr (kPass_ != kFinish) {
        const bool none = h.bad || flags != kSome;
        if (kPass_ == kCuts && tid == 0) state->live = none || h.t == 0.0f ? kChosen : kLive;
        if (none || h.t == 0.0f) {
            if (tid == 0 && gather_part == 0) {
                p.tokens[row] = none ? -1 : static_cast<int32_t>(best);
                if (p.prob != nullptr) p.prob[row] = none ? 0.0f : 1.0f;
                if (none) RaiseFlag(p.err, 1);
            }
            return;
        }
    }
    Chooser<T, kT> ch{p, h, s, units, p.largest + row * p.segments, top, LeastOf(largest), kLastKey};
    ch.MakeEdges();
    if constexpr (kPass_ == kSmall) {
        for (int i = tid; i < p.vocab; i += kT) {
            uint64_t key = s.list[i];
            if (Logit(static_cast<uint32_t>(key >> 32)) < ch.least) s.list[i] = key = kNoKey;
            s.code[i] = ch.CodeOf(key);
            double place;
            const int b = ch.BinOfKey(key, &place);
            if (s.code[i] != ~0u) ch.AddTo(b, h.k != 0 ? 1 : Weight(place));
        }
    }
    __syncthreads();
    // Where all that can be kept is in the list and few, an element a thread: in order by comparison
    // with all others, and every cut is a count.
    auto in_order = [&](int n) {
        uint64_t key = kNoKey, w = 0;
        if (tid < n) {
            key = kPass_ == kSmall ? s.list[tid] : state_list[tid];
            double f;
            const int b = ch.BinOfKey(key, &f);
            if (key <= kLastKey && b >= 0 && b < kBins) w = ch.Scaled(Weight(f), b);
            if (w == 0) key = kNoKey;
        }
        __syncthreads();
        s.bin[tid] = key;
        s.list[kFewAll + tid] = kNoKey;
        s.sum[tid] = 0;
        __syncthreads();
        int rank = 0;
        if (key != kNoKey) {
#pragma unroll 8
            for (int i = 0; i < n; ++i) rank += s.bin[i] < key ? 1 : 0;
            s.list[kFewAll + rank] = key;
            s.sum[rank] = w;
        }
        __syncthreads();
        w = s.sum[tid];
        uint64_t all;
        const uint64_t upto = ScanBlock<kW>(w, s.scan_u, &all);
        s.sum[tid] = upto;
        int kept = __syncthreads_count(w != 0);
        const uint64_t first = s.sum[0];
        if (h.k != 0 && h.k < kept) kept = h.k;
        if (h.p < 1.0f) {
            const uint64_t sum = row_reach != 0 ? row_reach : Reach(h.p, s.sum[kept - 1]);
            const int before = __syncthreads_count(tid < kept && upto < sum);
            if (before + 1 < kept) kept = before + 1;
        }
        if (h.m > 0.0f) {
            const int enough = __syncthreads_count(w != 0 && static_cast<double>(w) >= static_cast<double>(h.m) * static_cast<double>(first));
            if (enough < kept) kept = enough > 1 ? enough : 1;
        }
        const uint64_t whole = s.sum[kept - 1], bound = Share(h.u, whole);
        const int at = __syncthreads_count(tid < kept && upto <= bound);
        if (tid == (at < kept ? at : kept - 1)) {
            p.tokens[row] = static_cast<int32_t>(s.list[kFewAll + tid]);
            if (p.prob != nullptr) p.prob[row] = static_cast<float>(static_cast<double>(w) / static_cast<double>(whole));
        }
    };
    if (kPass_ != kCuts && all_held) {
        in_order(kPass_ == kSmall ? p.vocab : static_cast<int>(state->n));
        return;
    }
    // Three places are looked for in turn, each where its cut is asked for: the top-k's, the
    // top-p's (with the sum that min-p leaves) and the token's.  The row is gathered once for
    // the first two as a rule, or once for the last two.
    enum { kTopK, kTopP, kToken };
    int last = kBins - 1;       // no element of a later bin can be chosen
    int n = kPass_ == kSmall ? p.vocab : -1;  // elements of the list, where it has all that is needed
    const float u = h.u;
    uint64_t kept = 0, reach = 0;
    double least = 0.0;
    bool by_p = h.p < 1.0f, by_m = h.m > 0.0f;
    Span m{0, 0};
    int p_bin = 0;
    bool first = true, whole_list = false;
#pragma unroll 1
    for (int what = h.k != 0 ? kTopK : kTopP; what <= kToken; ++what) {
        Span a, b;      // bins to gather, if there is no list
        bool look = true, cuts = false;
        int bin;
        uint64_t bound;
        if (what == kTopK) {
            // (where no more than k have a bin, those beyond weigh nothing)
            uint64_t before = 0, held;
            const uint64_t k = static_cast<uint64_t>(h.k);
            last = bin = ch.Narrow(kCount, k, &before, &held);
            held += before;
            cuts = held >= k;
            if (!cuts) last = kBins - 1;
            bound = k - before;
            a = b = {held <= kList ? 0 : last, last};
            look = cuts;
        } else if (what == kTopP) {
            ch.SumBins();
            kept = s.sum[last];
            uint64_t low = kept;  // what is kept will weigh low .. kept
            if (by_p) {
                reach = Reach(h.p, kept);
                p_bin = ch.FirstBins(last, true, reach, reach).lo;
            }
            if (by_m) {
                least = static_cast<double>(h.m) * ch.WeightOf(largest);  // its equals are kept
                const double where = -static_cast<double>(kPerUnit) * log(least / kOne);
                m.hi = where >= kBins ? kBins - 1 : static_cast<int>(where + 0.51);
                m.lo = m.hi > 1 ? m.hi - 2 : 0;
                // whichever cut lies in earlier bins is the one
                if (m.lo > last || (by_p && m.lo > p_bin)) by_m = false;
                else if (by_p && m.hi < p_bin) by_p = false;
                if (m.hi > last) m.hi = last;
            }
            a = {0, -1};
            if (by_p) {
                a = {p_bin, p_bin};
                last = p_bin;
                kept = s.sum[p_bin];
                low = ch.Below(p_bin);
            }
            if (by_m) {
                a = {by_p && p_bin < m.lo ? p_bin : m.lo, by_p && p_bin > m.hi ? p_bin : m.hi};
                if (m.hi < last) last = m.hi;
                if (s.sum[m.hi] < kept) kept = s.sum[m.hi];
                if (ch.Below(m.lo) < low) low = ch.Below(m.lo);
            }
            b = ch.FirstBins(last, false, Share(u, low), Share(u, kept));
            if (a.lo > a.hi) a = b;
            bin = p_bin;
            bound = by_p ? ch.InBin(reach, p_bin, true) : 0;
            look = by_p;
        } else {
            const uint64_t x = Share(u, kept);
            bin = ch.FirstBins(last, false, x, x).lo;
            bound = ch.InBin(x, bin, false);
            a = b = {bin, bin};
        }
        bool whole = true;  // the list serves the places looked for later too
        if ((kPass_ == kCuts || kPass_ == kOneLaunch) && first) {
            bool is_all = a.lo == 0;
            if (what == kTopP) {  // whether all up to the last bin are few
                uint64_t mass = 0, all;
                for (int i = tid; i <= last; i += kT) mass += s.bin[i];
                ScanBlock<kW>(mass, s.scan_u, &all);
                is_all = static_cast<double>(all) * (1 / (0.984 * kOne)) < 0.9 * kFewAll;
                if (is_all) a = b = {0, last};
            }
            const RowState at{top, largest, ch.Lowest(a.hi), ch.Highest(a.lo), ch.Lowest(b.hi), ch.Highest(b.lo), is_all ? kAll : kLive, 0,
                              what == kTopP ? reach : 0, 0, 0};
            if constexpr (kPass_ == kCuts) {
                if (tid == 0) *state = at;
                return;
            }
            GatherPart<T, 1>(units, ch.largest, gather_part, at, s.list, s.some, &s.n_list);
            AddToList(state, s.list, s.n_list, &s.n_few);
            // every wave's part of the list has arrived; one thread's release and acquire then are the
            // workgroup's (by all of them they cost more than the launches that this saves: 64 bf16 rows
            // 90 us for 59)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (tid == 0) {
                s.n_few = __hip_atomic_fetch_add(&state->done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) + 1;
                s.n_list = __hip_atomic_load(&state->n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (s.n_few != static_cast<uint32_t>(gather_parts)) return;
            n = static_cast<int>(s.n_list);
            if (is_all) {
                row_reach = at.reach;
                if (n <= kFewAll) {
                    in_order(n);
                    return;
                }
            }
            whole_list = is_all;
        }
        if ((kPass_ == kFinish || kPass_ == kOneLaunch) && first) {  // what was gathered for this
            first = false;
            if constexpr (kPass_ == kFinish) {
                n = static_cast<int>(state->n);
                whole_list = state->live == kAll;
            }
#pragma unroll 4
            for (int i = tid; i < (n < kList ? n : kList); i += kT) ch.PutInList(i, state_list[i]);
            __syncthreads();
            if (n > kList) n = -1;
            whole = !(what == kTopK && a.lo != 0);
            if (what == kTopP && whole_list) whole = true;
        }
        if (n < 0 && look) {
            n = ch.Gather(bin);
            if (n > kList) n = -1;
            whole = false;
        }
        if (what == kTopP && by_m) {
            uint64_t sum[3] = {0, 0, 0};
            const double e[3] = {ch.Edge(m.lo), ch.Edge(m.lo < m.hi ? m.lo + 1 : m.lo), ch.Edge(m.hi)};
            auto add = [&](int at, double place, uint64_t, uint32_t) {
                const uint64_t w = Weight(place);
#pragma unroll
                for (int i = 0; i < 3; ++i) sum[i] += at - m.lo == i && static_cast<double>(w) * e[i] >= least ? w : 0;
            };
            if (kPass_ == kSmall || (n >= 0 && whole)) ch.InList(n, m, add);
            else ch.Visit(m, [&](int at, double place, uint64_t key) { add(at, place, key, 0); });
            kept = ch.Below(m.lo);
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                uint64_t all;
                ScanBlock<kW>(sum[i], s.scan_u, &all);
                if (m.lo + i <= m.hi) kept += ch.Scaled(all, m.lo + i);
            }
        }
        if (look) {
            constexpr Bound kBounds[3] = {kCount, kReach, kPass};
            const Bound meets = kBounds[what];
            const Place at = kPass_ == kSmall || n >= 0 ? ch.Select(n, bin, meets, bound) : ch.Search(bin, meets, bound);
            if (what == kTopK) {
                ch.limit = at.key;
            } else if (what == kTopP) {
                const uint64_t upto = ch.Below(bin) + ch.Scaled(at.before + at.own, bin);
                if (!by_m || upto < kept) kept = upto;
            } else if (tid == 0) {
                p.tokens[row] = static_cast<int32_t>(at.key);
                if (p.prob != nullptr) p.prob[row] = static_cast<float>(static_cast<double>(at.own) * ch.Edge(bin) / static_cast<double>(kept));
            }
        }
        if (what == kTopK) {  // the masses of what is left
            ch.ClearBins();
            __syncthreads();
            auto add = [&](int at, double place, uint64_t, uint32_t) { ch.AddTo(at, Weight(place)); };
            if (kPass_ == kSmall || (n >= 0 && whole)) ch.InList(n, {0, last}, add);
            else ch.Visit({0, last}, [&](int at, double place, uint64_t key) { add(at, place, key, 0); });
        }
        if (!whole) n = -1;
    }
}

// Between kCuts and kFinish: what a row's workgroup finds goes to the row's list.
template <typename T, int kLook>
__global__ __launch_bounds__(kChooseThreads) void SampleGather(const SampleArgs p, int parts) {
    __shared__ uint64_t found[kList];
    __shared__ uint16_t hits[kChooseWaves * kLook * kWave];
    __shared__ uint32_t n_found, base;
    const int64_t row = blockIdx.x / parts;
    const int part = static_cast<int>(blockIdx.x % parts);
    RowState* state = reinterpret_cast<RowState*>(p.state + row * kStateBytes);
    const RowState at = *state;
    if (at.live == kChosen) return;
    GatherPart<T, kLook>(RowUnits<T>(p, row), p.largest + row * p.segments, part, at, found, hits, &n_found);
    AddToList(state, found, n_found, &base);
}

// Workgroups of the first pass a row: as many as fill the device at 2 a compute unit,
// with kAhead blocks of 64 loads at least for each wave.
int Parts(int64_t n_rows, int64_t vocab, int bytes) {
    const int64_t blocks = (vocab * bytes + 1023) / 1024;
    int64_t parts = (static_cast<int64_t>(ComputeUnits()) * 2 + n_rows - 1) / n_rows;
    const int64_t most = (blocks + kAhead * kWaves - 1) / (kAhead * kWaves);
    if (parts > most) parts = most;
    if (parts > kMaxParts) parts = kMaxParts;
    return static_cast<int>(parts < 1 ? 1 : parts);
}
int64_t Segments(int64_t vocab, int bytes) {  // one more where the row is not aligned
    return (vocab * bytes + 127) / 128 + 1;
}
// Workgroups of the gather a row.
int GatherParts(int64_t vocab, int bytes, int look) {
    const int each = kChooseThreads * look;
    return static_cast<int>((Segments(vocab, bytes) + each - 1) / each);
}

// Rows that one round of launches takes, which is what the workspace is for.
constexpr int64_t kRowsAtOnce = 1024;

int64_t RowBytes(int parts, int64_t vocab, int bytes) {
    return kStateBytes + parts * kPartBytes + (4 * Segments(vocab, bytes) + 15) / 16 * 16;
}

template <typename T>
mlk_status Launch(SampleArgs p, int64_t n_rows, char* workspace, hipStream_t s) {
    constexpr int kBytes = sizeof(typename T::Bits);
    const dim3 block(kChooseThreads);
    const int64_t most = p.vocab <= kList ? n_rows : kRowsAtOnce;
    for (int64_t from = 0; from < n_rows; from += most) {
        const int64_t rows = n_rows - from < most ? n_rows - from : most;
        const dim3 grid(static_cast<unsigned>(rows));
        if (p.vocab <= kList) {
            hipLaunchKernelGGL((SampleChoose<T, kSmall>), grid, block, 0, s, p, 1);
        } else {
            p.parts = Parts(rows, p.vocab, kBytes);
            p.segments = static_cast<int32_t>((Segments(p.vocab, kBytes) + 3) / 4 * 4);
            p.state = workspace;
            p.part = p.state + rows * kStateBytes;
            p.largest = reinterpret_cast<float*>(p.part + rows * p.parts * kPartBytes);
            hipLaunchKernelGGL(SampleBins<T>, dim3(static_cast<unsigned>(rows * p.parts)), dim3(kThreads), 0, s, p);
            const int looks = GatherParts(p.vocab, kBytes, 1);
            // as long as each compute unit has one workgroup of it; at that edge it can be the slower (fp32 rows of 128256: 1 row 32.3 us by
            // the three launches, 27.9 by one, 8 rows 37.2 and 36.6, 16 rows 37.6 and 37.7; of 32000: 64
            // rows 31.6 and 28.8; bf16 rows of 128256, half the bytes: 16 rows 49.0 and 46.7, 32 rows 49.5
            // and 51.1)
            if (rows * looks <= ComputeUnits()) {
                hipLaunchKernelGGL((SampleChoose<T, kOneLaunch>), dim3(static_cast<unsigned>(rows * looks)), block, 0, s, p, looks);
            } else {
                hipLaunchKernelGGL((SampleChoose<T, kCuts>), grid, block, 0, s, p, 1);
                // the fewest looks a workgroup that leave no more than 5 of them to a compute unit: rows with
                // much to gather go over more of them, but the start of one with nothing to gather costs as
                // well (the whole call, rows of 128256 with one look, two and four: 128 in fp32 of mixed settings
                // 59.2, 57.2 and 64.7 us, of top-k 43.6, 38.0 and 36.3; 256 in bf16 of mixed settings 80.1,
                // 84.2 and 98.0, of top-k 48.5, 42.8 and 41.9)
                const int most_groups = 5 * ComputeUnits();
                const int look = rows * looks <= most_groups ? 1 : rows * GatherParts(p.vocab, kBytes, 2) <= most_groups ? 2 : 4;
                const int parts = GatherParts(p.vocab, kBytes, look);
                const dim3 gather(static_cast<unsigned>(rows * parts));
                if (look == 1) hipLaunchKernelGGL((SampleGather<T, 1>), gather, block, 0, s, p, parts);
                else if (look == 2) hipLaunchKernelGGL((SampleGather<T, 2>), gather, block, 0, s, p, parts);
                else hipLaunchKernelGGL((SampleGather<T, 4>), gather, block, 0, s, p, parts);
                // twice the threads where a compute unit has one row at most (rows of 128256, mixed
                // settings, the whole call: 64 in fp32 50.7 us with 256, 46.0 with 512, 256 of them 84.2 and
                // 81.0; 64 in bf16 58.4 and 54.0; 512 rows, with twice the threads in the other passes
                // too, 127 and 137)
                if (rows <= ComputeUnits()) hipLaunchKernelGGL((SampleChoose<T, kFinish, kWideThreads>), grid, dim3(kWideThreads), 0, s, p, 1);
                else hipLaunchKernelGGL((SampleChoose<T, kFinish>), grid, block, 0, s, p, 1);
            }
        }
        const mlk_status st = CheckLaunch("SampleChoose");
        if (st != MLK_OK) return st;
        p.x = static_cast<const typename T::Bits*>(p.x) + rows * p.row;
        p.u += rows;
        p.tokens += rows;
        if (p.prob != nullptr) p.prob += rows;
        if (p.how.temperature != nullptr) p.how.temperature += rows;
        if (p.how.top_k != nullptr) p.how.top_k += rows;
        if (p.how.top_p != nullptr) p.how.top_p += rows;
        if (p.how.min_p != nullptr) p.how.min_p += rows;
    }
    return MLK_OK;
}

}  // namespace
}  // namespace mlk

using namespace mlk;

extern "C" {

int64_t mlk_sample_workspace_bytes(int32_t type, int64_t n_rows, int64_t vocab) {
    if ((type != MLK_F32 && type != MLK_F16 && type != MLK_BF16) || n_rows <= 0 ||
        n_rows > kMaxRows || vocab <= 0 || vocab > kMaxVocab) {
        return 0;
    }
    if (vocab <= kList) return 16;
    const int bytes = TypeBytes(type);
    const int64_t rows = n_rows < kRowsAtOnce ? n_rows : kRowsAtOnce;
    int64_t most = rows * RowBytes(Parts(rows, vocab, bytes), vocab, bytes);
    const int64_t left = n_rows % kRowsAtOnce;  // a last round of few rows has more parts each
    if (n_rows > kRowsAtOnce && left != 0) {
        const int64_t last = left * RowBytes(Parts(left, vocab, bytes), vocab, bytes);
        if (last > most) most = last;
    }
    return most;
}

mlk_status mlk_sample(int32_t type, const void* logits, int64_t row_stride, int64_t n_rows,
                      int64_t vocab, const mlk_sampling* how, const float* uniform,
                      int32_t* tokens, float* prob, void* workspace, size_t workspace_bytes,
                      int32_t* err, void* stream) {
    const char* fn = "mlk_sample";
    if (type != MLK_F32 && type != MLK_F16 && type != MLK_BF16) {
        return Fail(MLK_ERR_INVALID, "%s: unknown element type", fn);
    }
    if (n_rows < 0 || n_rows > kMaxRows || vocab < 1 || vocab > kMaxVocab) {
        return Fail(MLK_ERR_INVALID, "%s: n_rows must be in 0..2^20 and vocab in 1..2^20", fn);
    }
    if (row_stride < vocab || row_stride > INT64_MAX / 8 / kMaxRows) {
        return Fail(MLK_ERR_INVALID, "%s: row_stride must be at least vocab", fn);
    }
    if (n_rows == 0) return MLK_OK;
    const int bytes = TypeBytes(type);
    if (logits == nullptr || !Aligned(logits, bytes)) {
        return Fail(MLK_ERR_INVALID, "%s: logits must be a %d-byte aligned device array", fn, bytes);
    }
    if (uniform == nullptr || tokens == nullptr || !Aligned(uniform, 4) || !Aligned(tokens, 4) ||
        !Aligned(prob, 4)) {
        return Fail(MLK_ERR_INVALID, "%s: uniform and tokens must be 4-byte aligned device arrays, "
                                     "as prob where given", fn);
    }
    SampleArgs p{};
    if (how != nullptr) p.how = *how;
    const void* ins[6] = {logits, uniform, p.how.temperature, p.how.top_k, p.how.top_p, p.how.min_p};
    for (int i = 0; i < 6; ++i) {
        if (!Aligned(ins[i], i == 0 ? 1 : 4)) {
            return Fail(MLK_ERR_INVALID, "%s: the settings must be 4-byte aligned", fn);
        }
        if (ins[i] != nullptr && (ins[i] == tokens || ins[i] == prob)) {
            return Fail(MLK_ERR_INVALID, "%s: tokens and prob may not alias an input", fn);
        }
    }
    if (static_cast<void*>(tokens) == static_cast<void*>(prob)) {
        return Fail(MLK_ERR_INVALID, "%s: tokens and prob may not alias", fn);
    }
    const int64_t need = mlk_sample_workspace_bytes(type, n_rows, vocab);
    if (workspace == nullptr || !Aligned(workspace, 16) || workspace_bytes < static_cast<size_t>(need)) {
        return Fail(MLK_ERR_INVALID, "%s: workspace must be a 16-byte aligned device buffer of %lld "
                                     "bytes", fn, static_cast<long long>(need));
    }
    p.x = logits;
    p.row = row_stride;
    p.vocab = static_cast<int32_t>(vocab);
    p.u = uniform;
    p.tokens = tokens;
    p.prob = prob;
    p.err = err;
    char* ws = static_cast<char*>(workspace);
    const hipStream_t s = AsStream(stream);
    if (type == MLK_F32) return Launch<F32>(p, n_rows, ws, s);
    if (type == MLK_F16) return Launch<F16>(p, n_rows, ws, s);
    return Launch<BF16>(p, n_rows, ws, s);
}

}  // extern "C"
