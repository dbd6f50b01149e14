// mlk_ragged_few.hip -- ragged attention of few rows per sequence: decode steps
// and short chunks, bound by the bytes of K and V.
//
// A workgroup takes a range of units of 32 positions, whatever sequences and
// heads they belong to (DivideFew): as many workgroups as the device holds, each
// with the same share, whether the lengths are alike or not.  Its rows are the
// (new token, query head of the group) pairs, at most 16 * NB, so each K and V row
// is read once for all of them.  The 8 waves (4 with two blocks of rows or a
// head_dim over 128) take neighbouring heads of the same positions, which are
// neighbours in memory, or where that leaves workers idle several waves take a
// head's positions 32 at a time (16 for fp32), with softmax statistics of their
// own that are joined at the end.  A row that several workers hold parts of is
// joined by a second kernel.
//
// Nothing is staged: both products take their operands from registers as the
// loads leave them.
//   S^T = K Q^T (16 positions x 16 rows a matrix instruction): a lane's
//     operand is 8 neighbouring elements of one K row, a 16-byte load.
//   O^T = V^T P^T: S^T's result layout (lane l: row l % 16, positions
//     4 (l / 16) + r) is P^T's operand layout with the positions in the order
//     16 (j / 4) + 4 (l / 16) + j % 4, j = 0 .. 7.  V^T's operand holds the same
//     8 positions of one dim; which dim belongs to which of the HD / 16
//     instructions is free, so lane l takes dims VE (l % 16) .. + VE - 1 of each
//     of its 8 positions, one load each, and instruction e their e-th: one byte
//     permute per operand dword.  The results then are runs of VE dims.
//   fp32 caches multiply in fp32 (v_mfma_f32_16x16x4_f32): 16 rows need 64
//     TFLOP/s at 8 TB/s, below its rate, and no pieces are formed.
// A tile's loads are issued when the one before has been used, so each wave
// keeps one tile (16 KB at head_dim 128) in flight through its arithmetic; they
// are non-temporal, no other workgroup reads those rows.  Pages are looked up a
// tile ahead by scalar loads, which do not queue behind the rows.
//
// 64 sequences of 8B heads, bf16, 1.10 GB of K and V: 190 us with the join, 5.8
// TB/s; of the time before, waves on neighbouring heads instead of one head 7 us,
// non-temporal loads 12, scalar look-ups 5.  4 sequences of 70B heads, fp32 over
// fp16, 0.79 GB: 146 us, 5.4 TB/s.  A kernel that only reads reached 5.0 to 7.5 TB/s,
// by its access pattern.  A single fp32 sequence (67 MB, 26 us) is far from its
// bytes: length, page, row and join each wait for the one before.
// Instances: head_dim 64, 128 and 256; another runs on the next one, padded.
#include "mlk_ragged.h"

namespace mlk {
namespace {

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

__device__ inline uint32_t LowHalves(uint32_t a, uint32_t b) {
    return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ inline uint32_t HighHalves(uint32_t a, uint32_t b) {
    return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// Per half: the larger of x and min(y, least).
__device__ inline uint32_t AtLeast(uint32_t x, uint32_t y, uint16_t least) {
    const u16x2 a = __builtin_bit_cast(u16x2, x), b = __builtin_bit_cast(u16x2, y);
    const u16x2 c = {least, least};
    return __builtin_bit_cast(uint32_t,
                              __builtin_elementwise_max(a, __builtin_elementwise_min(b, c)));
}

// K and V operands of one tile in registers, and their loads.
template <typename C, int HD, Lie kLie>
struct FewTile {
    static constexpr bool kF32 = std::is_same<C, F32>::value;
    static constexpr int KT = kF32 ? 16 : 32;        // positions
    static constexpr int NBK = KT / 16;              // blocks of 16 positions
    static constexpr int NKW = HD * (kF32 ? 4 : 2) / 16;  // dwords a lane has of a K row (4 lanes a row)
    static constexpr int NVW = HD * (kF32 ? 4 : 2) / 64;  // and of a V row (16 lanes a row)
    static constexpr int VE = kF32 ? 4 : (HD >= 128 ? 8 : 4);  // dims a lane's run has
    static constexpr int NVR = HD / 16 / VE;         // runs
    static constexpr int NKEY = kF32 ? 4 : 8;        // positions a lane's V operand has
    typedef typename C::Bits B;
    uint32_t k[NBK][NKW];
    uint32_t v[NKEY][NVW];

    // K row at `row`, this lane's dims: 16-bit 32 c + 8 g .. + 7, fp32 16 c + 4 g .. + 3
    __device__ void LoadK(int b, const B* row, int g, int hd) {
        constexpr int N = kF32 ? 4 : 8, S = 4 * N;
#pragma unroll
        for (int c = 0; c < HD / S; ++c) LoadRun<C, N, kLie, true>(row, S * c + N * g, hd, &k[b][4 * c]);
    }
    // V row at `row`, dims 16 VE n + VE (l % 16) .. + VE - 1
    __device__ void LoadV(int j, const B* row, int i16, int hd) {
        constexpr int W = VE * sizeof(B) / 4;
#pragma unroll
        for (int n = 0; n < NVR; ++n) {
            LoadRun<C, VE, kLie, true>(row, 16 * VE * n + VE * i16, hd, &v[j][W * n]);
        }
    }
};

// What addresses a tile needs: the sequence's table or first row.
struct FewRows {
    const RowsAt* at;
    const int32_t* table;  // nullptr: packed
    int64_t t0;
    int32_t end;  // positions the workgroup may read: 0 .. end - 1
};

// Element offsets of position j's K and V rows, lane by lane, clamped to the last.
__device__ inline void RowOffsets(const FewRows& r, int32_t j, int64_t* ko, int64_t* vo, bool* bad) {
    j = j < r.end ? j : r.end - 1;
    if (r.table != nullptr) {
        *ko = *vo = PagedRow(*r.at, PageOf(*r.at, r.table, j, bad), j);
    } else {
        *ko = (r.t0 + j) * r.at->k_row;
        *vo = (r.t0 + j) * r.at->v_row;
    }
}

template <typename A, typename C, int HD, int NB, int kWaves, Lie kLie>
__global__ __launch_bounds__(kWaves * kWave) void AttnFew(const RaggedParams p) {
    constexpr int kThreads = kWaves * kWave;
    typedef Pieces<A, C> P;
    typedef typename P::M M;
    typedef FewTile<C, HD, kLie> Tile;
    typedef typename C::Bits CB;
    typedef typename A::Bits AB;
    constexpr bool kF32 = Tile::kF32;
    constexpr int KT = Tile::KT, NBK = Tile::NBK, NI = HD / 16;
    constexpr int NQ = kF32 ? 1 : P::NQ, NW = P::NW;
    constexpr float kW = kF32 ? 0.0f : static_cast<float>(P::W);
    constexpr int kOLd = HD + 4;  // row stride of a wave's results in shared memory
    __shared__ float so[kWaves][16 * NB][kOLd];
    __shared__ float sm[kWaves][16 * NB], sl[kWaves][16 * NB];

    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int i16 = lane % 16, g4 = lane / 16;
    const int hd = kLie == kFull ? HD : p.rows.head_dim;
    if (blockIdx.x == 0 && p.taken == 0) CheckSeqs(p.batch, p.err);
    FewWork work;
    int64_t unit, end;  // this worker's units
    if (p.workers == 0) {
        work.heads = 1;
        work.s = static_cast<int>(p.taken + blockIdx.x / p.n_kv_heads);
        work.units = FewUnits(p, work.s);
        work.before = 0;
        unit = static_cast<int64_t>(blockIdx.x % p.n_kv_heads) * work.units;
        end = unit + work.units;
    } else {
        if (!FindFewWork(p, blockIdx.x, &work)) return;
        unit = blockIdx.x * work.share;
        end = unit + work.share;
    }
    const int heads = __builtin_amdgcn_readfirstlane(work.heads);  // of a block
    const int blocks = p.n_kv_heads / heads;
    const int along = kWaves / heads;   // waves of a head, taking tiles in turn
    const int my_head = wave % heads, my_turn = wave / heads;
    for (bool first = true; unit < end; first = false) {
        while (work.units == 0 || unit >= (work.before + work.units) * blocks) {
            work.before += work.units;
            if (++work.s >= p.batch.n_seqs) return;
            work.units = FewUnits(p, work.s);
        }
        const int s = __builtin_amdgcn_readfirstlane(work.s);
        const int32_t units = __builtin_amdgcn_readfirstlane(work.units);
        const int64_t in_seq = unit - work.before * blocks;
        const int head0 = __builtin_amdgcn_readfirstlane(static_cast<int>(in_seq / units)) * heads;
        const int kvh = head0 + my_head;
        const int32_t u0 = __builtin_amdgcn_readfirstlane(static_cast<int>(in_seq % units));
        const int32_t u1 = __builtin_amdgcn_readfirstlane(
            end - unit < units - u0 ? u0 + static_cast<int32_t>(end - unit) : units);
        unit += u1 - u0;
        Seq loaded;
        if (!LoadSeq(p.batch, s, &loaded)) return;
        const Seq q = loaded;
        const int rows = q.n * p.group;
        const int32_t j_begin = u0 * kFewKeys;
        if (j_begin >= q.len) continue;
        const int32_t j_end = q.len - j_begin > (u1 - u0) * kFewKeys ? u1 * kFewKeys : q.len;
        const bool split = u0 != 0 || j_end < q.len;

        const FewRows fr{&p.rows,
                         p.batch.table == nullptr ? nullptr : p.batch.table + s * p.batch.table_stride,
                         q.t0, j_end};
        const CB* kb = static_cast<const CB*>(p.rows.k) + static_cast<int64_t>(kvh) * hd;
        const CB* vb = static_cast<const CB*>(p.rows.v) + static_cast<int64_t>(kvh) * hd;

        // the rows' positions and q as it lies in memory; converted when the first
        // tile's loads are on their way
        constexpr int NQR = kF32 ? HD / 16 : HD / 32;  // runs of q a lane holds
        constexpr int NQW = kF32 ? 4 : (sizeof(AB) == 4 ? 8 : 4);
        int32_t pos[NB];
        uint32_t raw[NB][NQR][NQW];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int m = 16 * nb + i16;
            const bool real = m < rows;
            const int i = real ? m / p.group : 0;
            pos[nb] = real ? q.len - q.n + i : -1;
            const AB* qr = static_cast<const AB*>(p.q) + static_cast<int64_t>(q.t0 + i) * p.q_row +
                           static_cast<int64_t>(kvh * p.group + (real ? m % p.group : 0)) * hd;
#pragma unroll
            for (int c = 0; c < NQR; ++c) {
                if constexpr (kF32) {
                    LoadRun<F32, 4, kLie, false, true>(qr, 16 * c + 4 * g4, hd, raw[nb][c]);
                } else {
                    LoadRun<A, 8, kLie, false, true>(qr, 32 * c + 8 * g4, hd, raw[nb][c]);
                }
            }
        }

        Tile tile;
        bool bad = false;
        // 16-position blocks whose rows lie evenly apart: whole pages' parts, or packed
        const bool even = fr.table == nullptr || p.rows.page_shift >= 4;
        // else, pages of 4 positions or more: a lane's K row and its 4 V rows of a block
        // have a page each
        const bool lanes = !even && p.rows.page_shift >= 2;
        // element offsets of the blocks' first rows; the pages of the tile after the
        // next are looked up a tile ahead, so that no load waits for its page
        // (scalars: as arrays they stayed in scratch memory, decode of 64 rows 189 -> 233 us)
        int32_t page0 = 0, page1 = 0, page_k0 = 0, page_k1 = 0, page_v0 = 0, page_v1 = 0;
        const int shift = p.rows.page_shift;
        auto find = [&](int32_t j) __attribute__((always_inline)) {
            if (fr.table == nullptr) return;
            if (even) {
                if (j < j_end) page0 = ReadIndex(fr.table + (j >> shift));
                if (NBK > 1 && j + 16 < j_end) page1 = ReadIndex(fr.table + ((j + 16) >> shift));
            } else if (lanes && j + KT <= j_end) {
                page_k0 = ReadIndex(fr.table + ((j + i16) >> shift));
                page_v0 = ReadIndex(fr.table + ((j + 4 * g4) >> shift));
                if (NBK > 1) {
                    page_k1 = ReadIndex(fr.table + ((j + 16 + i16) >> shift));
                    page_v1 = ReadIndex(fr.table + ((j + 16 + 4 * g4) >> shift));
                }
            }
        };
        auto lane_row = [&](int32_t pg, int32_t j) __attribute__((always_inline)) -> int64_t {
            const bool in = pg >= 0 && pg < p.rows.n_pages;
            if (!in) bad = true;
            return PagedRow(p.rows, in ? pg : 0, j);
        };
        auto block_base = [&](int b, int32_t j, int64_t row) __attribute__((always_inline)) -> int64_t {
            if (fr.table == nullptr) return (fr.t0 + j) * row;  // j + 15 < end
            return lane_row(b == 0 ? page0 : page1, j);
        };
        auto load_k = [&](int32_t j0) __attribute__((always_inline)) {
            if (even && j0 + KT <= j_end) {
#pragma unroll
                for (int b = 0; b < NBK; ++b) {
                    const CB* base = kb + block_base(b, j0 + 16 * b, p.rows.k_row);
                    tile.LoadK(b, base + i16 * static_cast<uint32_t>(p.rows.k_row), g4, hd);
                }
                return;
            }
            if (lanes && j0 + KT <= j_end) {
#pragma unroll
                for (int b = 0; b < NBK; ++b) {
                    tile.LoadK(b, kb + lane_row(b == 0 ? page_k0 : page_k1, j0 + 16 * b + i16), g4, hd);
                }
                return;
            }
#pragma unroll
            for (int b = 0; b < NBK; ++b) {
                int64_t ko, vo;
                RowOffsets(fr, j0 + 16 * b + i16, &ko, &vo, &bad);
                tile.LoadK(b, kb + ko, g4, hd);
            }
        };
        auto load_v = [&](int32_t j0) __attribute__((always_inline)) {
            if (even && j0 + KT <= j_end) {
#pragma unroll
                for (int b = 0; b < NBK; ++b) {
                    const CB* base = vb + block_base(b, j0 + 16 * b, p.rows.v_row);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        tile.LoadV(4 * b + r, base + r * p.rows.v_row +
                                   (4 * g4) * static_cast<uint32_t>(p.rows.v_row), i16, hd);
                    }
                }
                return;
            }
            if (lanes && j0 + KT <= j_end) {
#pragma unroll
                for (int b = 0; b < NBK; ++b) {
                    const CB* base = vb + lane_row(b == 0 ? page_v0 : page_v1, j0 + 16 * b + 4 * g4);
#pragma unroll
                    for (int r = 0; r < 4; ++r) tile.LoadV(4 * b + r, base + r * p.rows.v_row, i16, hd);
                }
                return;
            }
#pragma unroll
            for (int j = 0; j < Tile::NKEY; ++j) {
                int64_t ko, vo;
                RowOffsets(fr, j0 + 16 * (j / 4) + 4 * g4 + j % 4, &ko, &vo, &bad);
                tile.LoadV(j, vb + vo, i16, hd);
            }
        };

        const int32_t step = along * KT;
        int32_t j0 = j_begin + my_turn * KT;
        if (j0 < j_end) {
            find(j0);
            load_k(j0);
            load_v(j0);
            find(j0 + step);
        }

        float factor[NB];
        u32x4 qp[NB][NQR][NQ];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            factor[nb] = p.factor;
            float up = 1.0f;
            if constexpr (!kF32 && P::kScaleQ) {
                float amax = 0.0f;
#pragma unroll
                for (int c = 0; c < NQR; ++c) {
#pragma unroll
                    for (int e = 0; e < NQW; ++e) amax = fmaxf(amax, fabsf(__uint_as_float(raw[nb][c][e])));
                }
                const int e = RowExponent(Max32(Max16(amax)));
                up = ldexpf(1.0f, e);
                factor[nb] = RowFactor(p.factor, e);
            }
#pragma unroll
            for (int c = 0; c < NQR; ++c) {
                if constexpr (NQ == 1) {
                    qp[nb][c][0] = u32x4{raw[nb][c][0], raw[nb][c][1], raw[nb][c][2], raw[nb][c][3]};
                } else {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(raw[nb][c][e]) * up;
                    Split8<M, NQ>(x, qp[nb][c]);
                }
            }
        }

        f32x4 o[NB][NI];
        float m[NB], l[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m[nb] = -INFINITY;  // of the scores before the factor
            l[nb] = 0.0f;       // this lane's part of the sum
#pragma unroll
            for (int e = 0; e < NI; ++e) o[nb][e] = f32x4{0, 0, 0, 0};
        }
        const int32_t first_pos = q.len - q.n;  // the lowest position of a row
        bool special = false;                   // met a non-finite V in a masked tile

        for (; j0 < j_end; j0 += step) {
            const int32_t jn = j0 + step;
            f32x4 sc[NB][NBK];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                for (int b = 0; b < NBK; ++b) {
                    f32x4 a = {0, 0, 0, 0};
                    if constexpr (kF32) {
#pragma unroll
                        for (int c = 0; c < HD / 16; ++c) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                a = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    __uint_as_float(tile.k[b][4 * c + e]),
                                    __uint_as_float(qp[nb][c][0][e]), a, 0, 0, 0);
                            }
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < HD / 32; ++c) {
                            const u32x4 kk = {tile.k[b][4 * c], tile.k[b][4 * c + 1],
                                              tile.k[b][4 * c + 2], tile.k[b][4 * c + 3]};
#pragma unroll
                            for (int n = 0; n < NQ; ++n) a = M::Mma16(kk, qp[nb][c][n], a);
                        }
                    }
                    sc[nb][b] = a;
                }
            }
            if (jn < j_end) load_k(jn);

            const bool masked = j0 + KT - 1 > first_pos || j0 + KT > j_end;
            float w[NB][4 * NBK];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float top = -INFINITY;
#pragma unroll
                for (int b = 0; b < NBK; ++b) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float x = sc[nb][b][r];
                        const int32_t j = j0 + 16 * b + 4 * g4 + r;
                        if (masked && (j > pos[nb] || j >= j_end)) x = -INFINITY;
                        w[nb][4 * b + r] = x;
                        top = fmaxf(top, x);
                    }
                }
                top = Max32(Max16(top));
                const float mn = fmaxf(m[nb], top);
                const float base = mn == -INFINITY ? 0.0f : mn;
                if (__ballot(mn != m[nb]) != 0) {
                    const float alpha = __builtin_amdgcn_exp2f((m[nb] - base) * factor[nb]);
                    l[nb] *= alpha;
#pragma unroll
                    for (int e = 0; e < NI; ++e) o[nb][e] *= alpha;
                    m[nb] = mn;
                }
                // the difference first: the largest weight is 2^kW however large the scores are
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 4 * NBK; ++i) {
                    w[nb][i] = __builtin_amdgcn_exp2f(fmaf(w[nb][i] - base, factor[nb], kW));
                    sum += w[nb][i];
                }
                l[nb] += sum;
            }

            if (masked) {
#pragma unroll
                for (int j = 0; j < Tile::NKEY; ++j) {
                    special |= OnlyFinite<C, Tile::NVW>(tile.v[j]);
                }
            }
            if constexpr (kF32) {
#pragma unroll
                for (int e = 0; e < NI; ++e) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            o[nb][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __uint_as_float(tile.v[r][e]), w[nb][r], o[nb][e], 0, 0, 0);
                        }
                    }
                }
            } else {
                u32x4 wp[NB][NW];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    Split8<M, NW>(w[nb], wp[nb]);
                    if constexpr (sizeof(AB) == 2) {
                        // no second piece 0 beside a first that is not: an infinity in V
                        // stays one (0 * inf is NaN)
                        constexpr uint16_t kLeast = C::kType == MLK_F16 ? 0x0001 : 0x0080;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            wp[nb][1][i] = AtLeast(wp[nb][1][i], wp[nb][0][i], kLeast);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < NI; ++e) {
                    u32x4 a;  // the e-th dim of each of the lane's positions
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t x = tile.v[2 * i][e / 2], y = tile.v[2 * i + 1][e / 2];
                        a[i] = e % 2 ? HighHalves(x, y) : LowHalves(x, y);
                    }
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                        for (int n = 0; n < NW; ++n) o[nb][e] = M::Mma16(a, wp[nb][n], o[nb][e]);
                    }
                }
            }
            if (jn < j_end) {
                load_v(jn);
                find(jn + step);
            }
        }
        if (bad && p.err != nullptr) RaiseFlag(p.err, 1);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) m[nb] *= factor[nb];  // as the joins take it

        const int32_t masked_from0 = (first_pos < j_end ? first_pos : j_end) - KT;
        const int32_t masked_from = masked_from0 > j_begin ? masked_from0 : j_begin;
        const int place = first ? 0 : 1;
        if (along == 1) {
            // the wave has its head's positions to itself
            const bool any_special = __ballot(special) != 0;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float lt = Sum32(Sum16(l[nb]));
                const int row = 16 * nb + i16;
                if (row >= rows) continue;
                const int i = row / p.group, h = kvh * p.group + row % p.group;
                const int64_t at = FewPartial(p, blockIdx.x, place, my_head, row);
                AB* out = static_cast<AB*>(p.out) + (static_cast<int64_t>(q.t0 + i) * p.n_heads + h) * hd;
                float* part = p.part_o + at * hd;
                if (split && g4 == 0) p.part_ml[at] = make_float2(m[nb], lt);
                const float inv = split ? 1.0f : 1.0f / lt;
                const int32_t last = pos[nb] < j_end ? pos[nb] : j_end - 1;
#pragma unroll
                for (int n = 0; n < Tile::NVR; ++n) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int d0 = 16 * Tile::VE * n + Tile::VE * (4 * g4 + r);
                        float x[Tile::VE];
#pragma unroll
                        for (int e = 0; e < Tile::VE; ++e) x[e] = o[nb][Tile::VE * n + e][r] * inv;
                        if (any_special) {
                            for (int e = 0; e < Tile::VE; ++e) {
                                if (d0 + e < hd) {
                                    x[e] += NonFiniteSum<C>(p.rows, fr.table, fr.t0, vb, masked_from,
                                                            last, d0 + e);
                                }
                            }
                        }
#pragma unroll
                        for (int e = 0; e < Tile::VE; ++e) {
                            if (kLie == kFull || d0 + e < hd) {
                                if (split) part[d0 + e] = x[e];
                                else out[d0 + e] = A::Put(x[e]);
                            }
                        }
                    }
                }
            }
        } else {
            // join the waves of a head: all relative to the largest maximum
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float lt = Sum32(Sum16(l[nb]));
                if (g4 == 0) {
                    sm[wave][16 * nb + i16] = m[nb];
                    sl[wave][16 * nb + i16] = lt;
                }
            }
            __syncthreads();
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const int row = 16 * nb + i16;
                float top = -INFINITY;
                for (int w = my_head; w < kWaves; w += heads) top = fmaxf(top, sm[w][row]);
                const float f = __builtin_amdgcn_exp2f(m[nb] - (top == -INFINITY ? 0.0f : top));
#pragma unroll
                for (int e = 0; e < NI; ++e) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int d = 16 * Tile::VE * (e / Tile::VE) + Tile::VE * (4 * g4 + r) + e % Tile::VE;
                        so[wave][row][d] = o[nb][e][r] * f;
                    }
                }
            }
            special = __syncthreads_or(special);
            for (int u = tid; u < heads * rows * HD; u += kThreads) {
                const int d = u % HD, row = u / HD % rows, hb = u / HD / rows;
                if (kLie != kFull && d >= hd) continue;
                float top = -INFINITY, lt = 0.0f, sum = 0.0f;
                for (int w = hb; w < kWaves; w += heads) top = fmaxf(top, sm[w][row]);
                const float base = top == -INFINITY ? 0.0f : top;
                for (int w = hb; w < kWaves; w += heads) {
                    lt += sl[w][row] * __builtin_amdgcn_exp2f(sm[w][row] - base);
                    sum += so[w][row][d];
                }
                const int i = row / p.group, h = (head0 + hb) * p.group + row % p.group;
                if (special) {
                    const int32_t last = first_pos + i < j_end ? first_pos + i : j_end - 1;
                    sum += NonFiniteSum<C>(p.rows, fr.table, fr.t0,
                                           static_cast<const CB*>(p.rows.v) +
                                               static_cast<int64_t>(head0 + hb) * hd,
                                           masked_from, last, d);
                }
                if (split) {
                    const int64_t at = FewPartial(p, blockIdx.x, place, hb, row);
                    p.part_o[at * hd + d] = sum;
                    if (d == 0) p.part_ml[at] = make_float2(top, lt);
                } else {
                    AB* out = static_cast<AB*>(p.out) +
                              (static_cast<int64_t>(q.t0 + i) * p.n_heads + h) * hd;
                    out[d] = A::Put(sum / lt);
                }
            }
            __syncthreads();  // the next pair writes over what was read here
        }
    }
}

template <typename A, typename C, int HD, int NB, int kWaves>
void Start(const RaggedParams& p, dim3 grid, hipStream_t s) {
    const dim3 block(kWaves * kWave);
    switch (LieOf(p, HD)) {
        case kFull: hipLaunchKernelGGL((AttnFew<A, C, HD, NB, kWaves, kFull>), grid, block, 0, s, p); break;
        case kPadded: hipLaunchKernelGGL((AttnFew<A, C, HD, NB, kWaves, kPadded>), grid, block, 0, s, p); break;
        default: hipLaunchKernelGGL((AttnFew<A, C, HD, NB, kWaves, kScalar>), grid, block, 0, s, p); break;
    }
}

template <typename A, typename C, int HD>
mlk_status Launch(const RaggedParams& p, dim3 grid, hipStream_t s) {
    if constexpr (HD <= 128) {
        if (p.few_rows <= 16) Start<A, C, HD, 1, 8>(p, grid, s);
        else Start<A, C, HD, 2, 4>(p, grid, s);
    } else {
        Start<A, C, HD, 1, 4>(p, grid, s);
    }
    return CheckLaunch("AttnFew");
}

struct ByDim {
    const RaggedParams& p;
    dim3 grid;
    hipStream_t stream;
    template <typename A, typename C>
    mlk_status Run() const {
        if (p.rows.head_dim <= 64) return Launch<A, C, 64>(p, grid, stream);
        if (p.rows.head_dim <= 128) return Launch<A, C, 128>(p, grid, stream);
        return Launch<A, C, 256>(p, grid, stream);
    }
};

}  // namespace

mlk_status LaunchFew(const RaggedParams& p, int32_t type, int32_t cache_type, hipStream_t stream) {
    if (p.workers != 0) {
        return ByType(type, cache_type, ByDim{p, dim3(static_cast<unsigned>(p.workers)), stream});
    }
    RaggedParams part = p;
    const int64_t most = kMaxBlocks / p.n_kv_heads;  // sequences of a launch
    mlk_status st = MLK_OK;
    for (part.taken = 0; part.taken < p.batch.n_seqs && st == MLK_OK; part.taken += most) {
        const int64_t left = p.batch.n_seqs - part.taken;
        const dim3 grid(static_cast<unsigned>((left < most ? left : most) * p.n_kv_heads));
        st = ByType(type, cache_type, ByDim{part, grid, stream});
    }
    return st;
}

}  // namespace mlk
