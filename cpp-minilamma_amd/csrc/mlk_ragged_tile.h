// mlk_ragged_tile.h -- ragged attention of many rows per sequence: whole
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
// kScored: with score functions and masks.  A tile's positions run from the first that any of
// its rows sees (chunks from what the window alone leaves, so that the join knows them);
// waves pass over tiles of positions that none of their rows sees.  7001 bf16 tokens of 70B
// heads in documents (120 GFLOP of what the masks leave): 252 to 259 us, 214 without the cap, and 190
// to 232 as the plain kernel's own sequences: a tile of 256 rows (32 tokens) walks 572 positions on
// average, nine tiles of K, beside a start and an end that cost what some 300 positions do; 11 %
// of the scores walked are of positions that the row does not see (8 of the 219 tiles lie across an edge of
// documents).
#pragma once

#include "mlk_ragged.h"

#include <climits>

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

template <typename A, typename C, int HD, Lie kLie, bool kScored>
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
    // the last row tiles first: of whole causal prompts those with the most positions to walk (documents
    // or a window make others the longest)
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
    [[maybe_unused]] const int32_t lo = first + static_cast<int32_t>(m0 / group);
    const int32_t hi = first + static_cast<int32_t>(m_last / group);
    // kScored: chunk 0 begins at `base`; the tile's rows see up to `most`
    const int32_t base0 = kScored ? TileBase(p, q, m0) : 0;
    const int32_t most = kScored ? SeenBy({nullptr, p.scores.prefix, nullptr, 0.0f, 0}, s, 0, hi, q.len).hi : hi;
    const int64_t chunk_at = base0 + static_cast<int64_t>(chunk) * p.chunk;
    if (chunk_at > most) return;
    int32_t j_begin = static_cast<int32_t>(chunk_at);
    const int32_t j_end = most + 1 - j_begin < p.chunk ? most + 1 : j_begin + p.chunk;

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
    int32_t wave_lo = w0 <= m_last ? first + static_cast<int32_t>(w0 / group) : -1;
    const int64_t w1 = w0 + 31 < m_last ? w0 + 31 : m_last;
    int32_t wave_hi = w0 <= m_last ? first + static_cast<int32_t>(w1 / group) + 1 : 0;
    // kScored: what this lane's row sees; from where all rows of the wave see, and any does
    int32_t row_lo = 0, row_hi = pos, wave_from = 0, wave_any = 0;
    // positions that all rows of the tile see: all_lo .. all_hi
    int32_t all_lo = 0, all_hi = lo;
    float slope = 0.0f;
    if constexpr (kScored) {
        const Seen seen = real ? SeenBy(p.scores, s, q.t0 + tok, pos, q.len) : Seen{0, -1};
        row_lo = seen.lo;
        row_hi = seen.hi;
        slope = SlopeOf(p, h);
        const bool sees = seen.lo <= seen.hi;
        int32_t least_lo = sees ? seen.lo : INT32_MAX, most_lo = real ? seen.lo : 0;
        int32_t least_hi = real ? seen.hi : INT32_MAX, most_hi = sees ? seen.hi : -1;
#pragma unroll
        for (int off = 16; off > 0; off /= 2) {
            const int32_t a = __shfl_xor(least_lo, off, kWave), b = __shfl_xor(most_lo, off, kWave);
            const int32_t c = __shfl_xor(least_hi, off, kWave), d = __shfl_xor(most_hi, off, kWave);
            least_lo = a < least_lo ? a : least_lo;
            most_lo = b > most_lo ? b : most_lo;
            least_hi = c < least_hi ? c : least_hi;
            most_hi = d > most_hi ? d : most_hi;
        }
        wave_any = __builtin_amdgcn_readfirstlane(least_lo);
        wave_from = __builtin_amdgcn_readfirstlane(most_lo);
        wave_lo = __builtin_amdgcn_readfirstlane(least_hi);
        wave_hi = __builtin_amdgcn_readfirstlane(most_hi) + 1;
        __shared__ int32_t bounds[3];  // least and most first position, least last one
        if (tid == 0) {
            bounds[0] = INT32_MAX;
            bounds[1] = 0;
            bounds[2] = INT32_MAX;
        }
        __syncthreads();
        if (lane == 0 && w0 <= m_last) {
            atomicMin(&bounds[0], wave_any);
            atomicMax(&bounds[1], wave_from);
            atomicMin(&bounds[2], wave_lo);
        }
        __syncthreads();
        all_lo = bounds[1];
        all_hi = bounds[2];
        if (chunk == 0 && real && !sees && half == 0) {  // a row that sees nothing
            AB* out = static_cast<AB*>(p.out) + (static_cast<int64_t>(q.t0 + tok) * p.n_heads + h) * hd;
            for (int d = 0; d < hd; ++d) out[d] = A::Put(0.0f);
        }
        const int32_t from = bounds[0] / kTileAlign * kTileAlign;
        if (from >= j_end) return;  // none of the rows has a part here
        if (from > j_begin) j_begin = from;
    }

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

    // scores that Score has gone over have no factor left
    const bool as_they_are = !kScored || AsTheyAre(p);
    [[maybe_unused]] const float raw_factor = factor;
    if (!as_they_are) factor = 1.0f;

    // staging: chunk tid + kThreads * i of the tile; a wave's 64 chunks are kPer
    // neighbouring rows
    constexpr int kChunks = HD / 8, kPer = kWave / kChunks;
    uint32_t gk[NCH][T::NW], gv[NCH][T::NW];
    bool bad = false, special = false;
    [[maybe_unused]] Seen met{INT32_MAX, -1};  // kScored: positions of the first and last tile that was
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
        // some row does not attend to all of it
        if (j0 + KT - 1 > all_hi || j0 + KT > j_end || (kScored && j0 < all_lo)) {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const bool hit = OnlyFinite<C, T::NW>(gv[i]);
                special |= hit;
                if (kScored && hit) met = {j0 < met.lo ? j0 : met.lo, j0 + KT - 1};
            }
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
        if (kScored && !as_they_are) {
#pragma unroll
            for (int b = 0; b < NKB; ++b) {
                float x[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = sc[b][r];
                Score<16>(p, raw_factor, slope, pos - j0 - 4 * half, x, [&](int r) { return 32 * b + 8 * (r / 4) + r % 4; });
#pragma unroll
                for (int r = 0; r < 16; ++r) sc[b][r] = x[r];
            }
        }
        if (j0 + KT - 1 > wave_lo || j0 + KT > j_end || (kScored && j0 < wave_from)) {
            const int32_t last = (row_hi < j_end ? row_hi : j_end - 1) - j0 - 4 * half;
            const int32_t from = row_lo - j0 - 4 * half;
#pragma unroll
            for (int b = 0; b < NKB; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at = 32 * b + 8 * (r / 4) + r % 4;
                    sc[b][r] = at > last || (kScored && at < from) ? -INFINITY : sc[b][r];
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
        if (j0 < wave_hi && (!kScored || j0 + KT > wave_any)) compute(j0, sk[buf], sv[buf]);
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
    if (kScored && special) {
        __shared__ int32_t span[2];
        if (tid == 0) {
            span[0] = INT32_MAX;
            span[1] = -1;
        }
        __syncthreads();
        atomicMin(&span[0], met.lo);
        atomicMax(&span[1], met.hi);
        __syncthreads();
        met = {span[0], span[1]};
    }
    l = Sum32(l);
    if (!real) return;
    int32_t last = row_hi < j_end ? row_hi : j_end - 1;
    int32_t masked_from = (lo < j_end ? lo : j_end) - KT;
    bool split = pos >= p.chunk;
    if constexpr (kScored) {
        if (row_lo > row_hi) return;
        const int32_t c0 = TileFirstChunk(p, base0, row_lo), c1 = (row_hi - base0) / p.chunk;
        if (chunk < c0 || chunk > c1) return;
        masked_from = row_lo > met.lo ? row_lo : met.lo;
        last = last < met.hi ? last : met.hi;
        split = c0 != c1;
    } else {
        if (pos < j_begin) return;
    }
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

template <int HD, bool kScored>
struct TileByType {
    const RaggedParams& p;
    dim3 grid;
    int64_t n_slots;
    hipStream_t stream;
    template <typename A, typename C>
    mlk_status Run() const {
        const dim3 block(TileShape<A, C, HD>::kThreads);
        switch (LieOf(p, HD)) {
            case kFull: hipLaunchKernelGGL((AttnTile<A, C, HD, kFull, kScored>), grid, block, 0, stream, p, n_slots); break;
            case kPadded: hipLaunchKernelGGL((AttnTile<A, C, HD, kPadded, kScored>), grid, block, 0, stream, p, n_slots); break;
            default: hipLaunchKernelGGL((AttnTile<A, C, HD, kScalar, kScored>), grid, block, 0, stream, p, n_slots); break;
        }
        return CheckLaunch("AttnTile");
    }
};

}  // namespace

template <int HD, bool kScored>
mlk_status LaunchTileAt(const RaggedParams& p, dim3 grid, int64_t n_slots, int32_t type,
                        int32_t cache_type, hipStream_t stream) {
    return ByType(type, cache_type, TileByType<HD, kScored>{p, grid, n_slots, stream});
}

}  // namespace mlk
