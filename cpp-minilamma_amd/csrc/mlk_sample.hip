// mlk_sample.hip -- the next token of each row of logits: temperature, top-k,
// top-p and min-p, from given uniform numbers.
//
// In descending order of the logits (the lower index first where they are equal),
// with w_i = exp((x_i - x_1) / T) and C_n = w_1 + .. + w_n, the tokens kept are the
// first n = max(1, min(n_k, n_p, n_m)), and the one chosen is the first with C_i >
// u C_n.  Each cut, and the choice itself, is the place in that order where a count
// or a sum crosses a bound.  A row is not sorted for it: bins of 1/16 of a
// temperature (b = rint(16 x / T), whatever the row's maximum is) say in which bin
// each bound is crossed, and only that bin's elements, or the few above the last
// cut, are put in order.
//
// Bins (one read of the logits, many workgroups a row): every wave has a histogram of
// its own in shared memory, a ring of the 512 bins up to the largest it has met (32
// temperatures; what drops out weighs below 2^-46 of the row's largest), so nothing
// waits for the maximum.  A weight is kept relative to its bin's middle, exp(f / 16)
// with |f| <= 1/2: a polynomial of degree 6 in float64 (Taylor's, within 2^-47), as a
// whole number of 2^-42.  Sums of whole numbers depend on no order: the row's bins
// are the same for every division of the work.  Rows with a top-k count instead, and
// evaluate no weights.  The largest of every 128 bytes is noted for the second pass.
//
// Choice (one workgroup a row): the parts' bins are added, a scan over the 512 finds
// the bins where the bounds are crossed, and the elements of those bins are gathered
// (128 bytes are read again only if their largest lies in the bins looked for),
// sorted in shared memory, and their sums scanned.  Bins of too many elements for that (nearly
// equal logits, high temperatures) are narrowed by the digits of the order's key
// (logit bits, then index), pass by pass over the row.
#include "mlk_paged.h"

#include <cmath>
#include <type_traits>

namespace mlk {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / kWave;
constexpr int kBins = 512;      // of a histogram, a power of two
constexpr int kSort = 2048;     // elements gathered and sorted at once
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
};
constexpr uint32_t kSome = 1, kNan = 2;
constexpr int64_t kPartBytes = sizeof(Part) + kBins * 8;

struct SampleArgs {
    const void* x;
    int64_t row;  // elements
    int32_t vocab, parts, segments;
    mlk_sampling how;
    const float* u;
    int32_t* tokens;
    float* prob;
    char* part;      // [rows][parts] of kPartBytes
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
    if (h.k <= 0 || h.k >= a.vocab) h.k = 0;
    const float t = fmaxf(h.t, 0x1p-14f);
    h.c = 16.0 / static_cast<double>(t);
    h.limit = fminf(t * 0x1p25f, 0x1.fffffep127f);
    return h;
}

// Bin of a logit (at most 2^29 in size by the limit) and its place f in it.
__device__ inline int32_t BinOf(const How& h, float x, double* f) {
    const double v = fminf(fmaxf(x, -h.limit), h.limit);
    constexpr double kRound = 0x1.8p52;
    const double t = fma(v, h.c, kRound);
    *f = fma(v, h.c, -(t - kRound));
    return static_cast<int32_t>(__double2loint(t));
}

// exp(f / 16) 2^42 as a whole number.
__device__ inline uint64_t Weight(double f) {
    constexpr double z = 1.0 / 16;
    double e = z * z * z * z * z * z / 720 * kOne;
    e = fma(e, f, z * z * z * z * z / 120 * kOne);
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
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int64_t row = blockIdx.x / p.parts;
    const int part = static_cast<int>(blockIdx.x % p.parts);
    const How h = HowOf(p, row);
    if (h.bad) return;  // the second pass sees that too
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

    for (int32_t b = b0 + wave * kAhead; b < b1; b += kWaves * kAhead) {
        u32x4 raw[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int32_t unit = (b + a) * kWave + lane;
            raw[a] = r.Load(unit, b + a < b1 && unit < units);
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
            if (b + a < b1 && lane % kSegment == 0) {
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
            double f;
            const int32_t to = BinOf(h, all, &f);
            if (some) {
                const int32_t fresh = to - top < kBins ? to - top : kBins;
                for (int32_t i = lane; i < fresh; i += kWave) mass[(to - i) & (kBins - 1)] = 0;
            }
            top = to;
            some = true;
        }
        if (!some) continue;
        auto add = [&](auto counts) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
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
    }
    __syncthreads();
    uint32_t flags = 0;
    int32_t all_top = INT32_MIN;
    for (int w = 0; w < kWaves; ++w) {
        flags |= flags_of[w];
        if ((flags_of[w] & kSome) && tops[w] > all_top) all_top = tops[w];
        if (best_of[w] < best) best = best_of[w];
    }
    Part* out = reinterpret_cast<Part*>(p.part + blockIdx.x * kPartBytes);
    if (tid == 0) *out = {all_top, flags, best};
    if (h.t == 0.0f || !(flags & kSome)) return;
    uint64_t* bins = reinterpret_cast<uint64_t*>(out + 1);
    for (int i = tid; i < kBins; i += kThreads) {
        const int32_t at = all_top - i;
        uint64_t sum = 0;
        for (int w = 0; w < kWaves; ++w) {
            if ((flags_of[w] & kSome) && static_cast<uint32_t>(tops[w] - at) < kBins) {
                sum += hist[w][at & (kBins - 1)];
            }
        }
        bins[i] = sum;
    }
}

// ------------------------------------------------------------ second pass

// Inclusive sums over the workgroup's threads, in a fixed order; *total over all.
template <typename V>
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
    uint64_t sorted[kSort];
    double edge[kBins];  // exp(-i / 16): a bin's middle, of the largest bin's
    double sum[kBins];   // of the weights up to and with bin i
    uint64_t bin[kBins];  // masses or counts of the bins; of a search's digits
    uint32_t number[kBins];  // a search's counts
    int32_t segment[kWaves][kWave];  // those a wave is to look through
    int32_t tops[kMaxParts];  // the parts' largest bins, INT32_MIN: none
    uint64_t scan_u[kWaves];
    double scan_d[kWaves];
    uint32_t at, n;  // a place looked for; elements gathered
    uint64_t word[3];
};

template <typename T>
struct Chooser {
    const SampleArgs& p;
    const How& h;
    Choice& s;
    RowUnits<T> r;
    const float* largest;
    int32_t top;
    uint64_t limit;  // keys past it are cut off (a top-k too large to be sorted)

    __device__ int Tid() const { return static_cast<int>(threadIdx.x); }

    // First i < n with ok(i) (n: none), monotone or not; every thread gets it.
    template <typename F>
    __device__ int First(int n, const F& ok) {
        __syncthreads();
        if (Tid() == 0) s.at = static_cast<uint32_t>(n);
        __syncthreads();
        for (int i = Tid(); i < n; i += kThreads) {
            if (ok(i)) {
                atomicMin(&s.at, static_cast<uint32_t>(i));
                break;
            }
        }
        __syncthreads();
        return static_cast<int>(s.at);
    }

    // f(whether it is one, bin below the largest, place in it, logit, index) over the elements of
    // bins lo .. hi: of each 128 bytes whose largest is no lower than those.  Whole waves
    // call f.  A wave looks at 64 segments at a time and has all that it needs of
    // them on their way before it takes the first.
    template <typename F>
    __device__ void Visit(int lo, int hi, const F& f) {
        constexpr int E = RowUnits<T>::E, kRounds = kWave / (kWave / kSegment);
        const int lane = Tid() % kWave, wave = Tid() / kWave;
        const int32_t units = r.Units(), segments = (units + kSegment - 1) / kSegment;
        const bool cut = limit != ~uint64_t{0};
        int32_t* mine = s.segment[wave];
        float next = wave * kWave + lane < segments ? largest[wave * kWave + lane] : -INFINITY;
        for (int32_t s0 = wave * kWave; s0 < segments; s0 += kThreads) {
            const float m = next;
            const int32_t then = s0 + kThreads + lane;
            next = then < segments ? largest[then] : -INFINITY;
            double place;
            const bool hit = m > -INFINITY && top - BinOf(h, m, &place) <= hi;
            const uint64_t mask = __ballot(hit);
            const int n = __popcll(mask);
            if (n == 0) continue;
            if (hit) mine[__popcll(mask & ((uint64_t{1} << lane) - 1))] = s0 + lane;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            u32x4 raw[kRounds];
            int32_t unit[kRounds];
#pragma unroll
            for (int i = 0; i < kRounds; ++i) {
                const int j = i * (kWave / kSegment) + lane / kSegment;
                unit[i] = (j < n ? mine[j] : 0) * kSegment + lane % kSegment;
                raw[i] = r.Load(unit[i], j < n && unit[i] < units);
            }
#pragma unroll
            for (int i = 0; i < kRounds; ++i) {
                if (i * (kWave / kSegment) >= n) break;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float x = r.Get(raw[i], e);
                    const int32_t b = top - BinOf(h, x, &place);
                    const int32_t index = r.Index(unit[i], e);
                    bool in = x > -INFINITY && b >= lo && b <= hi;
                    if (cut) in = in && Key(x, index) <= limit;
                    f(in, b, place, x, index);
                }
            }
        }
    }

    // Which of 512 equal ranges of its bin an element lies in, from the largest down.
    static __device__ int RangeOf(double place) {
        const int i = static_cast<int>((0.5 - place) * kBins);
        return i < 0 ? 0 : i < kBins ? i : kBins - 1;
    }

    // The elements of bins lo .. hi (range >= 0: of that range of them) into s.sorted; how many
    // there are (of more than kSort, not all are there).
    __device__ int Gather(int lo, int hi, int range = -1) {
        __syncthreads();
        if (Tid() == 0) s.n = 0;
        __syncthreads();
        const int lane = Tid() % kWave;
        Visit(lo, hi, [&](bool in, int32_t, double place, float x, int32_t i) {
            if (range >= 0) in = in && RangeOf(place) == range;
            const uint64_t mask = __ballot(in);
            if (mask == 0) return;
            uint32_t at = 0;
            if (lane == 0) at = atomicAdd(&s.n, static_cast<uint32_t>(__popcll(mask)));
            at = __builtin_amdgcn_readfirstlane(at) + __popcll(mask & ((uint64_t{1} << lane) - 1));
            if (in && at < kSort) s.sorted[at] = Key(x, i);
        });
        __syncthreads();
        return static_cast<int>(s.n);
    }

    // Bin `bin` by its ranges: the one where the sum of whole weights first reaches (kReach)
    // or passes `bound`; *before: the sum before it.
    __device__ int RangeWhere(int bin, bool reach, uint64_t bound, uint64_t* before) {
        __syncthreads();
        s.bin[Tid()] = 0;
        __syncthreads();
        Visit(bin, bin, [&](bool in, int32_t, double place, float, int32_t) {
            if (in) atomicAdd(reinterpret_cast<ull*>(&s.bin[RangeOf(place)]), static_cast<ull>(Weight(place)));
        });
        __syncthreads();
        uint64_t all;
        const uint64_t mine = s.bin[Tid()], sum = ScanBlock(mine, s.scan_u, &all);
        if (bound >= all) bound = reach ? all : all - 1;
        __syncthreads();
        if ((reach ? sum >= bound : sum > bound) && (reach ? sum - mine < bound : sum - mine <= bound)) {
            s.at = static_cast<uint32_t>(Tid());
            s.word[0] = sum - mine;
        }
        __syncthreads();
        *before = s.word[0];
        return static_cast<int>(s.at);
    }

    // s.sorted[0 .. n - 1] in order, n <= kSort.
    __device__ void Sort(int n) {
        int size = 2;
        while (size < n) size *= 2;
        for (int i = Tid() + n; i < size; i += kThreads) s.sorted[i] = ~uint64_t{0};
        for (int k = 2; k <= size; k *= 2) {
            for (int j = k / 2; j > 0; j /= 2) {
                __syncthreads();
                for (int i = Tid(); i < size / 2; i += kThreads) {
                    const int a = 2 * i - (i & (j - 1)), b = a + j;
                    const uint64_t x = s.sorted[a], y = s.sorted[b];
                    if ((x > y) == ((a & k) == 0)) {
                        s.sorted[a] = y;
                        s.sorted[b] = x;
                    }
                }
            }
        }
        __syncthreads();
    }

    __device__ double WeightOf(uint64_t key) const {
        double f;
        const int32_t b = top - BinOf(h, Logit(static_cast<uint32_t>(key >> 32)), &f);
        return b < 0 || b >= kBins ? 0.0 : static_cast<double>(Weight(f)) * s.edge[b];
    }

    // Sums up to each of the sorted elements a thread holds: 4 neighbours.
    static constexpr int kEach = kSort / kThreads;
    __device__ void SumSorted(int n, double base, double (&w)[kEach], double (&c)[kEach]) {
        double mine = 0, all;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int at = Tid() * kEach + i;
            w[i] = at < n ? WeightOf(s.sorted[at]) : 0.0;
            mine += w[i];
        }
        double before = base + (ScanBlock(mine, s.scan_d, &all) - mine);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            before += w[i];
            c[i] = before;
        }
    }
    // First of the n sorted elements with ok(sum, weight); n if none.
    template <typename F>
    __device__ int FirstSorted(int n, const double (&w)[kEach], const double (&c)[kEach], const F& ok) {
        __syncthreads();
        if (Tid() == 0) s.at = static_cast<uint32_t>(n);
        __syncthreads();
#pragma unroll
        for (int i = kEach - 1; i >= 0; --i) {
            const int at = Tid() * kEach + i;
            if (at < n && ok(c[i], w[i])) atomicMin(&s.at, static_cast<uint32_t>(at));
        }
        __syncthreads();
        return static_cast<int>(s.at);
    }
    // Sum up to sorted element i.
    __device__ double SumAt(int i, const double (&c)[kEach]) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            if (Tid() * kEach + e == i) s.scan_d[0] = c[e];
        }
        __syncthreads();
        const double v = s.scan_d[0];
        __syncthreads();
        return v;
    }

    // By digits of the keys of one bin's elements, pass by pass over the row: the first with
    // count >= bound (kCount), sum >= bound or sum > bound (whole numbers, of this bin's
    // middle).  Its key; *before and *own: the sum before it and its own weight.
    enum Bound { kCount, kReach, kPass };
    __device__ uint64_t Search(int bin, Bound what, uint64_t bound, uint64_t* before, uint64_t* own) {
        uint64_t high = 0, n0 = 0, m0 = 0;
        constexpr int kDigit = 9, kShifts = 8;  // 64 bits: 1 and 7 times 9
        for (int d = kShifts - 1; d >= 0; --d) {
            const int shift = d * kDigit;
            __syncthreads();
            for (int i = Tid(); i < kBins; i += kThreads) {
                s.bin[i] = 0;
                s.number[i] = 0;
            }
            __syncthreads();
            Visit(bin, bin, [&](bool in, int32_t, double f, float x, int32_t i) {
                const uint64_t key = Key(x, i);
                // (the first digit has one bit, the key's highest)
                if (!in || (d < kShifts - 1 && key >> (shift + kDigit) != high)) return;
                const int at = static_cast<int>(key >> shift) & (kBins - 1);
                atomicAdd(&s.number[at], 1u);
                atomicAdd(reinterpret_cast<ull*>(&s.bin[at]), static_cast<ull>(Weight(f)));
            });
            __syncthreads();
            uint64_t sums = 0, counts = 0, all;
            const uint64_t my_m = s.bin[Tid()], my_n = s.number[Tid()];
            sums = m0 + ScanBlock(my_m, s.scan_u, &all);
            counts = n0 + ScanBlock(my_n, s.scan_u, &all);
            const bool ok = my_n != 0 && (what == kCount ? counts >= bound : what == kReach ? sums >= bound : sums > bound);
            __syncthreads();
            if (Tid() == 0) s.at = kBins;
            __syncthreads();
            if (ok) atomicMin(&s.at, static_cast<uint32_t>(Tid()));
            __syncthreads();
            if (s.at == kBins) {  // none: the last element
                if (Tid() == 0) s.at = 0;
                __syncthreads();
                if (my_n != 0) atomicMax(&s.at, static_cast<uint32_t>(Tid()));
                __syncthreads();
            }
            const uint32_t at = s.at;
            if (static_cast<uint32_t>(Tid()) == at) {
                s.word[0] = sums - my_m;
                s.word[1] = counts - my_n;
                s.word[2] = my_m;
            }
            __syncthreads();
            high = (high << kDigit) | at;
            m0 = s.word[0];
            n0 = s.word[1];
            *own = s.word[2];
        }
        *before = m0;
        __syncthreads();
        return high;
    }

    // Sums over the bins from their masses.
    __device__ void SumBins() {
        double all;
        const double mine = static_cast<double>(s.bin[Tid()]) * s.edge[Tid()];
        const double c = ScanBlock(mine, s.scan_d, &all);
        s.sum[Tid()] = c;
        __syncthreads();
    }
    __device__ double Below(int bin) const { return bin > 0 ? s.sum[bin - 1] : 0.0; }

    // The element of bins up to `last` where the sum passes `bound`.
    struct Found {
        uint64_t key;
        double own;
    };
    __device__ Found Pass(double bound, int last) {
        int bin = First(last + 1, [&](int i) { return s.sum[i] > bound; });
        // (rounding: not above the last; and one that has elements)
        if (bin > last) bin = last;
        if (Below(bin) == s.sum[bin]) bin = First(last + 1, [&](int i) { return s.sum[i] == s.sum[last]; });
        const double base = Below(bin);
        const double in = (bound - base) / s.edge[bin];  // in whole weights of the bin
        const uint64_t whole = in > 0.0 ? static_cast<uint64_t>(in) : 0;
        double from = base;
        int n = Gather(bin, bin);
        if (n > kSort) n = GatherRange(bin, false, whole, &from);
        if (n <= kSort) {
            Sort(n);
            double w[kEach], c[kEach];
            SumSorted(n, from, w, c);
            int at = FirstSorted(n, w, c, [&](double sum, double) { return sum > bound; });
            at = at < n ? at : n - 1;
            return {s.sorted[at], WeightOf(s.sorted[at])};
        }
        uint64_t before, own;
        const uint64_t key = Search(bin, kPass, whole, &before, &own);
        return {key, static_cast<double>(own) * s.edge[bin]};
    }

    // The least sum up to an element of bin `bin` that reaches `bound`.
    __device__ double Reach(double bound, int bin) {
        const double base = Below(bin);
        const double in = ceil((bound - base) / s.edge[bin]);
        const uint64_t whole = in > 1.0 ? static_cast<uint64_t>(in) : 1;
        double from = base;
        int n = Gather(bin, bin);
        if (n > kSort) n = GatherRange(bin, true, whole, &from);
        if (n <= kSort) {
            Sort(n);
            double w[kEach], c[kEach];
            SumSorted(n, from, w, c);
            const int at = FirstSorted(n, w, c, [&](double sum, double) { return sum >= bound; });
            return SumAt(at < n ? at : n - 1, c);
        }
        uint64_t before, own;
        Search(bin, kReach, whole, &before, &own);
        return base + static_cast<double>(before + own) * s.edge[bin];
    }

    // The range of a bin in which a bound lies, gathered; *from: the sum before it.
    __device__ int GatherRange(int bin, bool reach, uint64_t whole, double* from) {
        uint64_t before;
        const int range = RangeWhere(bin, reach, whole, &before);
        *from += static_cast<double>(before) * s.edge[bin];
        return Gather(bin, bin, range);
    }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void SampleChoose(const SampleArgs p) {
    __shared__ Choice s;
    const int tid = static_cast<int>(threadIdx.x);
    const int64_t row = blockIdx.x;
    const How h = HowOf(p, row);
    const char* parts = p.part + row * p.parts * kPartBytes;
    uint32_t flags = 0;
    int32_t top = INT32_MIN;
    uint64_t best = ~uint64_t{0};
    if (!h.bad) {
        for (int i = 0; i < p.parts; ++i) {
            const Part part = *reinterpret_cast<const Part*>(parts + i * kPartBytes);
            flags |= part.flags;
            if ((part.flags & kSome) && part.top > top) top = part.top;
            if (part.best < best) best = part.best;
            if (tid == 0) s.tops[i] = part.flags & kSome ? part.top : INT32_MIN;
        }
    }
    __syncthreads();
    if (h.bad || !(flags & kSome) || (flags & kNan)) {
        if (tid == 0) {
            p.tokens[row] = -1;
            if (p.prob != nullptr) p.prob[row] = 0.0f;
            RaiseFlag(p.err, 1);
        }
        return;
    }
    if (h.t == 0.0f) {
        if (tid == 0) {
            p.tokens[row] = static_cast<int32_t>(best);
            if (p.prob != nullptr) p.prob[row] = 1.0f;
        }
        return;
    }
    Chooser<T> ch{p, h, s, RowUnits<T>(p, row), p.largest + row * p.segments, top, ~uint64_t{0}};
    static_assert(kBins == kThreads, "a thread a bin");
    uint64_t mine = 0;
#pragma unroll 8
    for (int i = 0; i < p.parts; ++i) {
        const int32_t at = s.tops[i] == INT32_MIN ? -1 : s.tops[i] - (top - tid);  // this thread's bin in the part
        if (at >= 0) mine += reinterpret_cast<const uint64_t*>(parts + i * kPartBytes + sizeof(Part))[at];
    }
    s.edge[tid] = exp(tid * (-1.0 / 16));
    s.bin[tid] = mine;
    __syncthreads();
    int k = h.k, last = kBins - 1;
    bool in_list = false;  // all that can be chosen is to be sorted
    if (k != 0) {
        uint64_t all;
        const uint64_t upto = ScanBlock(mine, s.scan_u, &all);
        s.bin[tid] = upto;
        __syncthreads();
        if (all <= static_cast<uint64_t>(k)) k = 0;  // the others weigh nothing
        else last = ch.First(kBins, [&](int i) { return s.bin[i] >= static_cast<uint64_t>(k); });
        const uint64_t n = s.bin[last], before = last > 0 ? s.bin[last - 1] : 0;
        in_list = n <= kSort;
        __syncthreads();
        if (!in_list) {
            if (k != 0) {
                uint64_t sum, own;
                ch.limit = ch.Search(last, Chooser<T>::kCount, k - before, &sum, &own);
            }
            // the masses of what is left
            s.bin[tid] = 0;
            __syncthreads();
            ch.Visit(0, last, [&](bool in, int32_t b, double f, float, int32_t) {
                if (in) atomicAdd(reinterpret_cast<ull*>(&s.bin[b]), static_cast<ull>(Weight(f)));
            });
            __syncthreads();
        }
    }
    double least = 0.0;  // a weight's, by min_p
    if (h.m > 0.0f) {
        // the largest weight: that of the row's first, at the largest bin's place
        float m = -INFINITY;
        const int segments = (ch.r.Units() + kSegment - 1) / kSegment;
        for (int i = tid; i < segments; i += kThreads) m = fmaxf(m, ch.largest[i]);
        __syncthreads();
        m = BlockMax<kWaves>(m, reinterpret_cast<float*>(s.scan_u));
        const double w = ch.WeightOf(Key(m, 0));
        least = fmin(static_cast<double>(h.m), 1.0) * w;  // the first at least, and its equals
    }
    double bound;
    if (!in_list) {
        ch.SumBins();
        double kept = s.sum[last];
        if (h.p < 1.0f) {
            const double reach = static_cast<double>(h.p) * kept;
            const int bin = ch.First(last, [&](int i) { return s.sum[i] >= reach; });
            kept = ch.Reach(reach, bin);
            last = bin;
        }
        if (h.m > 0.0f) {
            // the bins that least lies in or beside
            const double where = -16.0 * log(least / kOne);
            int hi = where >= kBins ? kBins - 1 : static_cast<int>(where + 0.51);
            const int lo = hi > 1 ? hi - 2 : 0;
            if (lo <= last) {
                hi = hi < last ? hi : last;
                uint64_t sum[3] = {0, 0, 0};
                ch.Visit(lo, hi, [&](bool in, int32_t b, double f, float, int32_t) {
                    if (!in) return;
                    const uint64_t w = Weight(f);
                    if (static_cast<double>(w) * s.edge[b] < least) return;
#pragma unroll
                    for (int i = 0; i < 3; ++i) sum[i] += b - lo == i ? w : 0;
                });
                double upto = ch.Below(lo);
                for (int i = 0; i < 3; ++i) {
                    uint64_t all;
                    ScanBlock(sum[i], s.scan_u, &all);
                    if (lo + i <= hi) upto += static_cast<double>(all) * s.edge[lo + i];
                }
                if (upto < kept) kept = upto;
                if (hi < last) last = hi;
                __syncthreads();
            }
        }
        bound = static_cast<double>(h.u) * kept;
        const auto found = ch.Pass(bound, last);
        if (tid == 0) {
            p.tokens[row] = static_cast<int32_t>(found.key);
            if (p.prob != nullptr) p.prob[row] = static_cast<float>(found.own / kept);
        }
        return;
    }
    const int n = ch.Gather(0, last);
    ch.Sort(n);
    double w[Chooser<T>::kEach], c[Chooser<T>::kEach];
    ch.SumSorted(n, 0.0, w, c);
    int kept = k != 0 && k < n ? k : n;
    if (h.p < 1.0f) {
        const double reach = static_cast<double>(h.p) * ch.SumAt(kept - 1, c);
        const int at = ch.FirstSorted(kept, w, c, [&](double sum, double) { return sum >= reach; });
        kept = at < kept ? at + 1 : kept;
    }
    if (h.m > 0.0f) {
        const int at = ch.FirstSorted(kept, w, c, [&](double, double weight) { return weight < least; });
        kept = at < 1 ? 1 : at;
    }
    const double whole = ch.SumAt(kept - 1, c);
    bound = static_cast<double>(h.u) * whole;
    int at = ch.FirstSorted(kept, w, c, [&](double sum, double) { return sum > bound; });
    at = at < kept ? at : kept - 1;
    if (tid == 0) {
        p.tokens[row] = static_cast<int32_t>(s.sorted[at]);
        if (p.prob != nullptr) p.prob[row] = static_cast<float>(ch.WeightOf(s.sorted[at]) / whole);
    }
}

// Workgroups of the first pass a row: as many as fill the device at 3 a compute unit,
// with 2 blocks of 64 loads at least for each wave.
int Parts(int64_t n_rows, int64_t vocab, int bytes) {
    const int64_t blocks = (vocab * bytes + 1023) / 1024;
    int64_t parts = (static_cast<int64_t>(ComputeUnits()) * 3 + n_rows - 1) / n_rows;
    const int64_t most = blocks / (2 * kWaves);  // 2 blocks a wave
    if (parts > most) parts = most;
    if (parts > kMaxParts) parts = kMaxParts;
    return static_cast<int>(parts < 1 ? 1 : parts);
}
int64_t Segments(int64_t vocab, int bytes) {  // one more where the row is not aligned
    return (vocab * bytes + 127) / 128 + 1;
}

template <typename T>
void Launch(const SampleArgs& p, int64_t n_rows, hipStream_t s) {
    hipLaunchKernelGGL(SampleBins<T>, dim3(static_cast<unsigned>(n_rows * p.parts)), dim3(kThreads), 0, s, p);
    hipLaunchKernelGGL(SampleChoose<T>, dim3(static_cast<unsigned>(n_rows)), dim3(kThreads), 0, s, p);
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
    const int bytes = TypeBytes(type);
    return n_rows * (Parts(n_rows, vocab, bytes) * kPartBytes + 4 * Segments(vocab, bytes)) + 16;
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
    p.parts = Parts(n_rows, vocab, bytes);
    p.segments = static_cast<int32_t>(Segments(vocab, bytes));
    p.part = static_cast<char*>(workspace);
    p.largest = reinterpret_cast<float*>(p.part + n_rows * p.parts * kPartBytes);
    const hipStream_t s = AsStream(stream);
    if (type == MLK_F32) Launch<F32>(p, n_rows, s);
    else if (type == MLK_F16) Launch<F16>(p, n_rows, s);
    else Launch<BF16>(p, n_rows, s);
    return CheckLaunch("SampleChoose");
}

}  // extern "C"
