// mlk_ragged_tile.hip -- ragged attention of many rows per sequence: whole
// prompts and chunks of them, bound by the matrix cores.
//
// A workgroup takes 256 rows (128 with a head_dim over 128) of one sequence and
// KV head -- (token, query head of the group) pairs, so a group's heads share K
// and V -- and walks the positions its last row attends to, or a chunk of them,
// KT = 64 at a time (32 where the tile or the pieces of q would not fit).  Each
// of its 8 (4) waves owns 32 rows; the tile's K and V rows are shared through LDS:
//   S^T = K Q^T  (v_mfma 32x32x16, 32 positions x 32 rows): K rows as they lie,
//     8 elements a lane; q stays in registers.
//   softmax: a lane holds 16 of each 32 positions of ONE row, so maximum and sum
//     are within the lane but for one exchange of the wave's halves, and the
//     rescale of the results is a plain product.
//   O^T = V^T P^T: S^T's layout is P^T's operand layout, with the positions of
//     a lane's half in the order 16 m + 8 (j / 4) + 4 (l / 32) + j % 4; V^T comes
//     from V's rows by the transposing LDS read (4 positions of 16 dims).
// The next tile's loads are issued before a tile's products and land in
// registers; they are written to LDS after them (16-bit caches: two buffers and
// one barrier a tile; fp32: split into pieces on the way, one buffer).
// LDS rows are unpadded, their 16-byte chunks permuted by the row so that both
// K's reads (16 rows of one chunk) and V's (4 rows of 64 bytes) meet each bank
// once (counted: no conflicts).
//
// 9001 packed bf16 tokens of 70B heads: 567 GFLOP in 643 us, 0.88 PFLOP/s where
// an 8192^3 bf16 product reaches 1.35.  2500 packed fp32 tokens of 8B heads: 6
// products for each of 11.9 GFLOP, 119 us, 0.6 PFLOP/s.  256 rows share a tile's
// loads: with 128 these took 674 and 144 us.  Counted on the packed bf16 call, the
// matrix units are busy 37 % of the cycles and vector instructions issue in 43 %:
// no one resource is full, the two kinds of phase overlap partly.
// Instances: head_dim 64, 128 and 256; another runs on the next one, padded, at that
// one's cost (4096 packed bf16 tokens of 8 heads: 80 in 90 us, 128 in 83).
#include "mlk_ragged.h"

namespace mlk {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* LdsS16x4;

// Row r's chunk permutation (an xor), HD / 8 chunks a row.
template <int HD>
__device__ inline int Swizzle(int r) {
    return HD == 64 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
}

constexpr float kLarge = 4096.0f;  // of a score times the factor

template <typename A, typename C, int HD>
struct TileShape {
    static constexpr int kThreads = TileRows(HD) / 32 * kWave;
    static constexpr int NK = std::is_same<C, F32>::value ? 3 : 1;
    static constexpr int KT = HD != 64 && (NK == 3 || HD == 256 || Pieces<A, C>::NQ == 3) ? 32 : 64;
    static constexpr int NBUF = NK == 3 ? 1 : 2;
    static constexpr int kPlane = KT * HD;             // elements
    static constexpr int NCH = KT * HD / 8 / kThreads;  // chunks a thread stages
    static constexpr int NW = NK == 3 ? 8 : 4;         // dwords a chunk has in memory
};

template <typename A, typename C, int HD, Lie kLie>
__global__ __launch_bounds__((TileShape<A, C, HD>::kThreads), HD <= 128 ? 2 : 1) void AttnTile(const RaggedParams p, int64_t n_slots) {
    typedef Pieces<A, C> P;
    typedef typename P::M M;
    typedef TileShape<A, C, HD> T;
    typedef typename C::Bits CB;
    typedef typename A::Bits AB;
    constexpr int kThreads = T::kThreads, kRows = TileRows(HD);
    constexpr int NQ = P::NQ, NK = T::NK, KT = T::KT, NKB = KT / 32, NCH = T::NCH;
    constexpr int ND = HD / 32, NS = HD / 16;
    constexpr int kTerms = NQ > NK ? NQ : NK;  // products of pieces i, j: i + j < kTerms
    __shared__ __align__(16) uint16_t sk[T::NBUF][NK * T::kPlane];
    __shared__ __align__(16) uint16_t sv[T::NBUF][NK * T::kPlane];

    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int l32 = lane % 32, half = lane / 32;
    const int hd = kLie == kFull ? HD : p.rows.head_dim;
    if (blockIdx.x == 0 && p.taken == 0) CheckSeqs(p.batch, p.err);

    const int kvh = static_cast<int>(blockIdx.x % p.n_kv_heads);
    const int64_t rest = blockIdx.x / p.n_kv_heads;
    const int chunk = static_cast<int>(rest % p.n_chunks);
    // the longest prefixes first
    const int64_t slot = n_slots - 1 - p.taken - rest / p.n_chunks;
    const int group = p.group;
    auto first_slot = [group](int32_t start, int s) {
        return static_cast<int64_t>(start) * group / kRows + s;
    };
    const int s = LastSeq(p.batch, slot, first_slot);
    Seq q;
    if (!LoadSeq(p.batch, s, &q)) return;
    const int64_t m0 = (slot - first_slot(q.t0, s)) * kRows;
    const int64_t rows = static_cast<int64_t>(q.n) * group;
    if (m0 < 0 || m0 >= rows || rows <= p.few_rows) return;
    const int64_t m_last = (m0 + kRows < rows ? m0 + kRows : rows) - 1;
    const int32_t first = q.len - q.n;  // position of the sequence's first new token
    const int32_t lo = first + static_cast<int32_t>(m0 / group);
    const int32_t hi = first + static_cast<int32_t>(m_last / group);
    const int32_t j_begin = chunk * p.chunk;
    if (j_begin > hi) return;
    const int32_t j_end = hi + 1 - j_begin < p.chunk ? hi + 1 : j_begin + p.chunk;

    const int32_t* table =
        p.batch.table == nullptr ? nullptr : p.batch.table + s * p.batch.table_stride;
    const CB* kb = static_cast<const CB*>(p.rows.k) + static_cast<int64_t>(kvh) * hd;
    const CB* vb = static_cast<const CB*>(p.rows.v) + static_cast<int64_t>(kvh) * hd;

    // this lane's row
    const int64_t m = m0 + 32 * wave + l32;
    const bool real = m < rows;
    const int32_t tok = real ? static_cast<int32_t>(m / group) : 0;
    const int h = kvh * group + (real ? static_cast<int>(m % group) : 0);
    const int32_t pos = real ? first + tok : -1;
    // positions that all rows of the wave attend to: up to wave_lo; that any does: below
    // wave_hi
    const int64_t w0 = m0 + 32 * wave;
    const int32_t wave_lo = w0 <= m_last ? first + static_cast<int32_t>(w0 / group) : -1;
    const int64_t w1 = w0 + 31 < m_last ? w0 + 31 : m_last;
    const int32_t wave_hi = w0 <= m_last ? first + static_cast<int32_t>(w1 / group) + 1 : 0;

    float factor = p.factor;
    u32x4 qf[NS][NQ];
    {
        const AB* qr = static_cast<const AB*>(p.q) + static_cast<int64_t>(q.t0 + tok) * p.q_row +
                       static_cast<int64_t>(h) * hd;
        uint32_t raw[NS][sizeof(AB) == 4 ? 8 : 4];
#pragma unroll
        for (int c = 0; c < NS; ++c) {
            LoadRun<A, 8, kLie, false, true>(qr, 16 * c + 8 * half, hd, raw[c]);
        }
        if constexpr (NQ == 1) {
#pragma unroll
            for (int c = 0; c < NS; ++c) qf[c][0] = u32x4{raw[c][0], raw[c][1], raw[c][2], raw[c][3]};
        } else {
            float up = 1.0f;
            if constexpr (P::kScaleQ) {
                float amax = 0.0f;
#pragma unroll
                for (int c = 0; c < NS; ++c) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(__uint_as_float(raw[c][e])));
                }
                const int e = RowExponent(Max32(amax));
                up = ldexpf(1.0f, e);
                factor = RowFactor(p.factor, e);
            }
#pragma unroll
            for (int c = 0; c < NS; ++c) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(raw[c][e]) * up;
                Split8<M, NQ>(x, qf[c]);
            }
        }
    }

    // staging: chunk tid + kThreads * i of the tile; a wave's 64 chunks are kPer
    // neighbouring rows
    constexpr int kChunks = HD / 8, kPer = kWave / kChunks;
    uint32_t gk[NCH][T::NW], gv[NCH][T::NW];
    bool bad = false, special = false;
    const int my_r = lane / kChunks, my_c = lane % kChunks;
    auto first_row = [&](int i) { return kPer * wave + kThreads / kChunks * i; };
    // whole tiles whose kPer rows share a page (or are packed): uniform bases; their
    // pages are looked up a tile ahead
    const bool even = table == nullptr || (1 << p.rows.page_shift) >= kPer;
    int32_t page[NCH] = {};
    auto find = [&](int32_t j0) {
        if (table == nullptr || !even || j0 + KT > j_end) return;
#pragma unroll
        for (int i = 0; i < NCH; ++i) page[i] = ReadIndex(table + ((j0 + first_row(i)) >> p.rows.page_shift));
    };
    auto load = [&](int32_t j0, const CB* base, int64_t row, uint32_t (&g)[NCH][T::NW]) {
        if (even && j0 + KT <= j_end) {
            const uint32_t mine = static_cast<uint32_t>(my_r) * static_cast<uint32_t>(row);
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int32_t j = j0 + first_row(i);
                int64_t at = (static_cast<int64_t>(q.t0) + j) * row;
                if (table != nullptr) {
                    const bool in = page[i] >= 0 && page[i] < p.rows.n_pages;
                    bad |= !in;
                    at = PagedRow(p.rows, in ? page[i] : 0, j);
                }
                LoadRun<C, 8, kLie, false>(base + at + mine, 8 * my_c, hd, g[i]);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int r = first_row(i) + my_r;
            const int32_t j = j0 + r < j_end ? j0 + r : j_end - 1;
            const int64_t at = table != nullptr
                                   ? PagedRow(p.rows, PageOf(p.rows, table, j, &bad), j)
                                   : (static_cast<int64_t>(q.t0) + j) * row;
            LoadRun<C, 8, kLie, false>(base + at, 8 * my_c, hd, g[i]);
        }
    };
    auto put = [&](uint16_t* dst, const uint32_t (&g)[NCH][T::NW]) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int r = first_row(i) + my_r;
            const int at = r * HD + ((my_c ^ Swizzle<HD>(r)) * 8);
            if constexpr (NK == 1) {
                *reinterpret_cast<u32x4*>(dst + at) = u32x4{g[i][0], g[i][1], g[i][2], g[i][3]};
            } else {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(g[i][e]);
                u32x4 w[NK];
                Split8<M, NK>(x, w);
#pragma unroll
                for (int n = 0; n < NK; ++n) {
                    *reinterpret_cast<u32x4*>(dst + n * T::kPlane + at) = w[n];
                }
            }
        }
    };
    auto put_v = [&](int32_t j0, uint16_t* dst) {
        if (j0 + KT - 1 > lo || j0 + KT > j_end) {  // some row does not attend to all of it
#pragma unroll
            for (int i = 0; i < NCH; ++i) special |= OnlyFinite<C, T::NW>(gv[i]);
        }
        put(dst, gv);
    };
    f32x16 o[ND];
    float mx = -INFINITY, l = 0.0f;  // of the scores before the factor; this lane's part
#pragma unroll
    for (int d = 0; d < ND; ++d) {
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    }

    find(j_begin);
    load(j_begin, kb, p.rows.k_row, gk);
    load(j_begin, vb, p.rows.v_row, gv);
    find(j_begin + KT);
    put(sk[0], gk);
    put_v(j_begin, sv[0]);
    __syncthreads();
    // the tile in buffer B; the next one's loads are on their way
    auto compute = [&](int32_t j0, const uint16_t* ks, const uint16_t* vs) {
        f32x16 sc[NKB];
#pragma unroll
        for (int b = 0; b < NKB; ++b) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[b][r] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < NS; ++c) {
#pragma unroll
            for (int b = 0; b < NKB; ++b) {
                u32x4 kf[NK];
#pragma unroll
                for (int n = 0; n < NK; ++n) {
                    kf[n] = *reinterpret_cast<const u32x4*>(
                        ks + n * T::kPlane + (32 * b + l32) * HD +
                        (((2 * c + half) ^ Swizzle<HD>(l32)) * 8));
                }
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
#pragma unroll
                    for (int n = 0; n < NK; ++n) {
                        if (i + n < kTerms) sc[b] = M::Mma32(kf[n], qf[c][i], sc[b]);
                    }
                }
            }
        }
        constexpr int NM = NK == 3 ? 6 : NQ, kSteps = NS * NKB, kDeep = 8 / NK;
        __builtin_amdgcn_sched_group_barrier(0x100, NK * kDeep, 0);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, NM, 0);
            if (i + kDeep < kSteps) __builtin_amdgcn_sched_group_barrier(0x100, NK, 0);
        }
        if (j0 + KT - 1 > wave_lo || j0 + KT > j_end) {
            const int32_t last = (pos < j_end ? pos : j_end - 1) - j0 - 4 * half;
#pragma unroll
            for (int b = 0; b < NKB; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    sc[b][r] = 32 * b + 8 * (r / 4) + r % 4 > last ? -INFINITY : sc[b][r];
                }
                asm volatile("" : "+v"(sc[b]));  // a branch: else every tile pays for the mask
            }
        }
        float top = sc[0][0];
#pragma unroll
        for (int b = 0; b < NKB; ++b) {
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, sc[b][r]);
        }
        const float mn = fmaxf(mx, Max32(top));
        const float from = mn == -INFINITY ? 0.0f : mn;
        if (__ballot(mn != mx) != 0) {
            const float alpha = __builtin_amdgcn_exp2f((mx - from) * factor);
            l *= alpha;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= alpha;
            mx = mn;
        }
        // The weights' exponents are (score - maximum) * factor + W.  With the maximum in
        // the addend that is one instruction a score, off by the addend's rounding: up
        // to kLarge at most 2^-11, like the score's own.  Beyond it the difference is taken
        // first: the largest weight is 2^W however large the scores are.
        const float base = from * factor;
        float off = static_cast<float>(P::W) - base;
        if (__ballot(fabsf(base) > kLarge) != 0) {
            off = static_cast<float>(P::W);
#pragma unroll
            for (int b = 0; b < NKB; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) sc[b][r] -= from;
                asm volatile("" : "+v"(sc[b]));  // a branch, as above
            }
        }
        float sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < NKB; ++b) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                sc[b][r] = __builtin_amdgcn_exp2f(fmaf(sc[b][r], factor, off));
                sum[r % 4] += sc[b][r];
            }
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        const int i16 = lane % 16, g2 = (lane / 16) % 2;
#pragma unroll
        for (int t = 0; t < KT / 16; ++t) {
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = sc[t / 2][8 * (t % 2) + e];
            u32x4 wf[NQ];
            Split8<M, NQ>(w, wf);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                u32x4 vf[NK];
#pragma unroll
                for (int n = 0; n < NK; ++n) {
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj) {
                        const int r = 16 * t + 8 * jj + 4 * half + i16 / 4;
                        const int c = 4 * d + 2 * g2 + (i16 % 4) / 2;
                        const uint16_t* at = vs + n * T::kPlane + r * HD +
                                             ((c ^ Swizzle<HD>(r)) * 8) + 4 * (i16 % 2);
                        const u32x2 x = __builtin_bit_cast(
                            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (LdsS16x4)(const_cast<uint16_t*>(at))));
                        vf[n][2 * jj] = x[0];
                        vf[n][2 * jj + 1] = x[1];
                    }
                }
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
#pragma unroll
                    for (int n = 0; n < NK; ++n) {
                        if (i + n < kTerms) o[d] = M::Mma32(vf[n], wf[i], o[d]);
                    }
                }
            }
        }
    };
    auto step = [&](int32_t j0, int buf) {
        const bool more = j0 + KT < j_end;
        if (more) {
            load(j0 + KT, kb, p.rows.k_row, gk);
            load(j0 + KT, vb, p.rows.v_row, gv);
            find(j0 + 2 * KT);
        }
        if (j0 < wave_hi) compute(j0, sk[buf], sv[buf]);
        const int other = T::NBUF == 1 ? 0 : buf ^ 1;
        if constexpr (T::NBUF == 1) __syncthreads();
        if (more) {
            put(sk[other], gk);
            put_v(j0 + KT, sv[other]);
        }
        __syncthreads();
    };
    if constexpr (T::NBUF == 2) {
        for (int32_t j0 = j_begin; j0 < j_end; j0 += 2 * KT) {
            step(j0, 0);
            if (j0 + KT < j_end) step(j0 + KT, 1);
        }
    } else {
        for (int32_t j0 = j_begin; j0 < j_end; j0 += KT) step(j0, 0);
    }
    if (bad && p.err != nullptr) RaiseFlag(p.err, 1);
    special = __syncthreads_or(special);
    l = Sum32(l);
    if (!real || pos < j_begin) return;
    const int32_t last = pos < j_end ? pos : j_end - 1;
    const int32_t masked_from = (lo < j_end ? lo : j_end) - KT;
    const bool split = pos >= p.chunk;
    const int64_t at = split ? TilePartial(p, q.t0 + tok, h) + chunk : 0;
    if (split && half == 0) p.part_ml[at] = make_float2(mx * factor, l);
    const float inv = split ? 1.0f : 1.0f / l;
    AB* out = static_cast<AB*>(p.out) + (static_cast<int64_t>(q.t0 + tok) * p.n_heads + h) * hd;
    float* part = p.part_o + at * hd;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int dim = 32 * d + 8 * r4 + 4 * half;
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = o[d][4 * r4 + e] * inv;
            if (special) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (dim + e < hd) {
                        x[e] += NonFiniteSum<C>(p.rows, table, q.t0, vb,
                                                masked_from > j_begin ? masked_from : j_begin, last,
                                                dim + e);
                    }
                }
            }
            if (split) {
                if constexpr (kLie == kFull) {
                    *reinterpret_cast<f32x4*>(part + dim) = f32x4{x[0], x[1], x[2], x[3]};
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (dim + e < hd) part[dim + e] = x[e];
                    }
                }
            } else if constexpr (kLie == kFull && sizeof(AB) == 4) {
                *reinterpret_cast<f32x4*>(out + dim) = f32x4{x[0], x[1], x[2], x[3]};
            } else if constexpr (kLie == kFull) {
                *reinterpret_cast<u32x2*>(out + dim) =
                    u32x2{static_cast<uint32_t>(A::Put(x[0])) |
                              (static_cast<uint32_t>(A::Put(x[1])) << 16),
                          static_cast<uint32_t>(A::Put(x[2])) |
                              (static_cast<uint32_t>(A::Put(x[3])) << 16)};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (dim + e < hd) out[dim + e] = A::Put(x[e]);
                }
            }
        }
    }
}

template <typename A, typename C, int HD>
mlk_status Launch(const RaggedParams& p, dim3 grid, int64_t n_slots, hipStream_t s) {
    constexpr int kThreads = TileShape<A, C, HD>::kThreads;
    const dim3 block(kThreads);
    switch (LieOf(p, HD)) {
        case kFull: hipLaunchKernelGGL((AttnTile<A, C, HD, kFull>), grid, block, 0, s, p, n_slots); break;
        case kPadded: hipLaunchKernelGGL((AttnTile<A, C, HD, kPadded>), grid, block, 0, s, p, n_slots); break;
        default: hipLaunchKernelGGL((AttnTile<A, C, HD, kScalar>), grid, block, 0, s, p, n_slots); break;
    }
    return CheckLaunch("AttnTile");
}

struct ByDim {
    const RaggedParams& p;
    dim3 grid;
    int64_t n_slots;
    hipStream_t stream;
    template <typename A, typename C>
    mlk_status Run() const {
        if (p.rows.head_dim <= 64) return Launch<A, C, 64>(p, grid, n_slots, stream);
        if (p.rows.head_dim <= 128) return Launch<A, C, 128>(p, grid, n_slots, stream);
        return Launch<A, C, 256>(p, grid, n_slots, stream);
    }
};

// Row tiles of a batch: sequence s owns the slots from start[s] * group / rows
// + s on, at least as many as it has tiles, whatever the lengths.
int64_t TileSlots(int64_t n_seqs, int64_t n_tokens, int32_t group, int rows) {
    return n_tokens * group / rows + n_seqs;
}

}  // namespace

int64_t TileBlocks(const RaggedParams& p) {
    return TileSlots(p.batch.n_seqs, p.batch.n_tokens, p.group, TileRows(p.rows.head_dim)) *
           p.n_chunks * p.n_kv_heads;
}

mlk_status LaunchTile(const RaggedParams& p, int32_t type, int32_t cache_type, hipStream_t stream) {
    const int64_t slots = TileSlots(p.batch.n_seqs, p.batch.n_tokens, p.group,
                                    TileRows(p.rows.head_dim));
    RaggedParams part = p;
    const int64_t per_slot = static_cast<int64_t>(p.n_chunks) * p.n_kv_heads;
    const int64_t most = kMaxBlocks / per_slot;  // row tiles of a launch
    mlk_status st = MLK_OK;
    for (part.taken = 0; part.taken < slots && st == MLK_OK; part.taken += most) {
        const int64_t here = slots - part.taken < most ? slots - part.taken : most;
        const dim3 grid(static_cast<unsigned>(here * per_slot));
        st = ByType(type, cache_type, ByDim{part, grid, slots, stream});
    }
    return st;
}

}  // namespace mlk
