// mlk_ragged.hip -- attention of many sequences' tokens, over pages of a cache
// or over rows of a packed buffer: which kernels a call runs, how it splits
// positions, and the join of split rows.
//
// Token row t at position p of its sequence, head h on KV head h / (H / KV):
//   s_j = scale (q . k_j), j <= p;  w = softmax(s);  out = sum_j w_j v_j.
// Sequences of few rows (new tokens x query heads of a group, at most FewMost)
// are bound by the bytes of K and V (mlk_ragged_few.h); the others by the
// matrix cores (mlk_ragged_tile.h).  A batch of both kinds runs both kernels,
// each leaving the other's sequences alone.
#include "mlk_ragged.h"

namespace mlk {
namespace {

constexpr int kThreads = 256;

// out = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c over a row's n parts.  A
// group of L lanes (4 dims each) takes every `per_row`-th part of a row, the
// groups' sums are added in order.  What costs is latency, not bytes: the first
// kAhead parts of each group are on their way before the maxima are looked at
// (one 8B decode row over 32 parts: 21 us with one wave walking them all, 6 us).
constexpr int kAhead = 4;

// Row of `n` parts: the first at partial `base`, the second at `next`, and from
// there one every `step`.
struct JoinRow {
    int64_t base, next, step;
    int32_t t, h, n;
    bool blind;  // sees nothing: zeros
};

template <typename A, int L>
__device__ inline void Join(const RaggedParams& p, const JoinRow& row, int part_of, int per_row,
                            f32x4 (*sums)[L]) {
    const int lane = static_cast<int>(threadIdx.x) % L, g = static_cast<int>(threadIdx.x) / L;
    const int hd = p.rows.head_dim, n = row.n;
    const bool wide = hd % 4 == 0;
    auto part = [&](int c) { return c == 0 ? row.base : row.next + (c - 1) * row.step; };
    auto dims = [&](int c) {
        f32x4 x = {0, 0, 0, 0};
        const float* at = p.part_o + part(c) * hd + 4 * lane;
        if (wide) {
            if (4 * lane < hd) x = *reinterpret_cast<const f32x4*>(at);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (4 * lane + e < hd) x[e] = at[e];
            }
        }
        return x;
    };
    f32x4 ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int c = part_of + per_row * i;
        if (c < n) ahead[i] = dims(c);
    }
    float m = -INFINITY;
    for (int c = lane; c < n; c += L) m = fmaxf(m, p.part_ml[part(c)].x);
#pragma unroll
    for (int off = L / 2; off > 0; off /= 2) m = fmaxf(m, __shfl_xor(m, off, kWave));
    if (m == -INFINITY) m = 0.0f;
    float l = 0.0f;
    for (int c = lane; c < n; c += L) {
        const float2 ml = p.part_ml[part(c)];
        l = fmaf(ml.y, __builtin_amdgcn_exp2f(ml.x - m), l);
    }
#pragma unroll
    for (int off = L / 2; off > 0; off /= 2) l += __shfl_xor(l, off, kWave);
    f32x4 o = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int c = part_of + per_row * i;
        if (c < n) o += ahead[i] * __builtin_amdgcn_exp2f(p.part_ml[part(c)].x - m);
    }
#pragma unroll 4
    for (int c = part_of + per_row * kAhead; c < n; c += per_row) {
        o += dims(c) * __builtin_amdgcn_exp2f(p.part_ml[part(c)].x - m);
    }
    if (per_row > 1) {
        sums[g][lane] = o;
        __syncthreads();
    }
    if (part_of != 0 || n == 0) return;
    for (int i = 1; i < per_row; ++i) o += sums[g + i][lane];
    typename A::Bits* out = static_cast<typename A::Bits*>(p.out) +
                            (static_cast<int64_t>(row.t) * p.n_heads + row.h) * hd;
    const float inv = row.blind ? 0.0f : 1.0f / l;
    if (p.vec) {  // out is 16-byte aligned, head_dim a multiple of 8
        if (4 * lane < hd) {
            typedef typename A::Bits Out4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<Out4*>(out + 4 * lane) =
                Out4{A::Put(o[0] * inv), A::Put(o[1] * inv), A::Put(o[2] * inv), A::Put(o[3] * inv)};
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (4 * lane + e < hd) out[4 * lane + e] = A::Put(o[e] * inv);
    }
}

// Few-row kernel's rows, a place's after the other's: block = place * per_place
// + place of its rows.  A place is a sequence, all heads; or, in batches of more
// sequences than workers, a worker, standing for the one (sequence, block of heads)
// that it is the second to hold a part of: others have no parts to join, and looking
// for each sequence's share is work for all the sequences before it.  (The whole call,
// 8B heads, bf16, by sequence and by worker: 16384 sequences of lengths to 1024 21.5
// and 6.7 ms, 1024 of them 0.50 and 0.46; 64 of lengths to 8192 191 and 195 us, one
// of 8191 in fp32 27 and 38.)
template <typename A, int L, bool kByWorker, bool kScored>
__device__ inline void JoinFewRows(const RaggedParams& p, uint32_t block, int per_row, int per_place,
                                   f32x4 (*sums)[L]) {
    constexpr int NG = kThreads / L;
    const int g = static_cast<int>(threadIdx.x) / L;
    const int rows_here = NG / per_row;
    const int place = static_cast<int>(block / per_place);
    const int64_t first = static_cast<int64_t>(block % per_place) * rows_here;
    const int64_t in_place = first + g / per_row;
    FewWork work;
    int64_t head0 = 0, heads = p.n_kv_heads;
    if constexpr (kByWorker) {
        if (!FindFewWork<kScored>(p, place, &work)) return;
        const int64_t blocks = p.n_kv_heads / work.heads, unit = place * work.share;
        const int64_t block = (unit - work.before * blocks) / work.units;
        const int64_t u0 = work.before * blocks + block * work.units;
        if (u0 / work.share != place - 1) return;
        head0 = block * work.heads;
        heads = work.heads;
    } else {
        work.s = place;
        work.units = FewUnits<kScored>(p, place);
        if (work.units == 0) return;
    }
    Seq q;
    if (!LoadSeq(p.batch, work.s, &q)) return;
    const int64_t rows = static_cast<int64_t>(q.n) * p.group;
    if (first >= rows * heads) return;  // none of the workgroup's rows is one
    if constexpr (!kByWorker) {
        work.before = 0;
        DivideFew(p, p.batch.n_seqs == 1 ? work.units : CountFewUnits<kScored>(p, work.s, &work.before), &work);
    }
    const int m = static_cast<int>(in_place % rows);
    JoinRow row{};
    if (in_place < rows * heads) {
        const int64_t kvh = head0 + in_place / rows;
        const int64_t u0 = work.before * (p.n_kv_heads / work.heads) + kvh / work.heads * work.units;
        const int32_t held = FewHeld(q, FewFirst<kScored>(p, q));
        const int64_t w0 = u0 / work.share, w1 = (u0 + held - 1) / work.share;
        const int head = static_cast<int>(kvh % work.heads);
        if (w1 > w0) {
            row.t = q.t0 + m / p.group;
            row.h = static_cast<int>(kvh) * p.group + m % p.group;
            row.n = static_cast<int>(w1 - w0) + 1;
            row.base = FewPartial(p, w0, u0 == w0 * work.share ? 0 : 1, head, m);
            row.next = FewPartial(p, w0 + 1, 0, head, m);
            row.step = 2 * kFewHeads * p.few_rows;
            if constexpr (kScored) {
                const Seen seen = SeenBy(p.scores, work.s, row.t, q.len - q.n + m / p.group, q.len);
                row.blind = seen.lo > seen.hi;
            }
        }
    }
    Join<A, L>(p, row, g % per_row, per_row, sums);
}

// Tile kernel's rows: block = token * per_token + place of its heads.
template <typename A, int L, bool kScored>
__device__ inline void JoinTileRows(const RaggedParams& p, uint32_t block, int per_row, int per_token,
                                    f32x4 (*sums)[L]) {
    constexpr int NG = kThreads / L;
    const int g = static_cast<int>(threadIdx.x) / L;
    const int32_t t = static_cast<int32_t>(block / per_token);
    const int32_t h = static_cast<int32_t>(block % per_token) * (NG / per_row) + g / per_row;
    const int s = LastSeq(p.batch, t, [](int32_t a, int) { return a; });
    Seq q;
    if (!LoadSeq(p.batch, s, &q) || t < q.t0 || t >= q.t0 + q.n) return;
    const int32_t pos = q.len - q.n + (t - q.t0);
    if (static_cast<int64_t>(q.n) * p.group <= p.few_rows || (!kScored && pos < p.chunk)) return;
    JoinRow row{0, 0, 1, t, h, 0, false};
    if (h < p.n_heads) {
        row.base = TilePartial(p, t, h);
        row.n = pos / p.chunk + 1;
        if constexpr (kScored) {
            // the row's tile, and which of its chunks have a part of the row
            const int64_t m = static_cast<int64_t>(t - q.t0) * p.group + h % p.group;
            const int rows = TileRows(p.rows.head_dim);
            const int32_t base = TileBase(p, q, m / rows * rows);
            const Seen seen = SeenBy(p.scores, s, t, pos, q.len);
            const int32_t c0 = TileFirstChunk(p, base, seen.lo);
            row.base += c0;
            row.n = seen.lo > seen.hi ? 0 : (seen.hi - base) / p.chunk - c0 + 1;
            if (row.n <= 1) row.n = 0;  // written by the tile
        }
        row.next = row.base + 1;
    }
    Join<A, L>(p, row, g % per_row, per_row, sums);
}

// A row's parts go over so many groups that each has them on their way at once, up to
// the workgroup's (a row over more groups only waits for them at the barrier).
inline int PerRow(int groups, int64_t parts) {
    int per_row = 1;
    while (per_row < groups && per_row * kAhead < parts) per_row *= 2;
    return per_row;
}

inline int JoinGroups(const RaggedParams& p) { return p.rows.head_dim <= 128 ? 8 : 4; }
inline int JoinFewPerRow(const RaggedParams& p) {
    // parts of a row where the sequences are alike and few_heads heads go together
    const int64_t pairs = static_cast<int64_t>(p.batch.n_seqs) * p.n_kv_heads / p.few_heads;
    return PerRow(JoinGroups(p), (p.workers + pairs - 1) / pairs + 1);
}
inline bool JoinByWorker(const RaggedParams& p) { return p.batch.n_seqs > p.workers; }
inline int64_t JoinFewPerPlace(const RaggedParams& p) {
    const int64_t heads = JoinByWorker(p) ? p.few_heads : p.n_kv_heads;
    return (heads * p.few_rows * JoinFewPerRow(p) + JoinGroups(p) - 1) / JoinGroups(p);
}
inline int64_t JoinFewBlocks(const RaggedParams& p) {
    return JoinFewPerPlace(p) * (JoinByWorker(p) ? p.workers : p.batch.n_seqs);
}
inline int64_t JoinTilePerToken(const RaggedParams& p) {
    const int heads = JoinGroups(p) / PerRow(JoinGroups(p), p.n_chunks);
    return (p.n_heads + heads - 1) / heads;
}
inline int64_t JoinTileBlocks(const RaggedParams& p) {
    return JoinTilePerToken(p) * p.batch.n_tokens;
}

template <typename A, int L, bool kByWorker, bool kScored>
__global__ __launch_bounds__(kThreads) void JoinFew(const RaggedParams p, int per_row, int per_place) {
    __shared__ f32x4 sums[kThreads / L][L];
    JoinFewRows<A, L, kByWorker, kScored>(p, blockIdx.x, per_row, per_place, sums);
}
template <typename A, int L, bool kScored>
__global__ __launch_bounds__(kThreads) void JoinTile(const RaggedParams p, int per_row, int per_token) {
    __shared__ f32x4 sums[kThreads / L][L];
    JoinTileRows<A, L, kScored>(p, blockIdx.x, per_row, per_token, sums);
}

// Both, where a mixed batch leaves both: the few-row kernel's rows by the first few_blocks
// workgroups, the tile kernel's by the others.  Neither waits for the other, and each is a chain
// of loads (calls with one launch for each and with one for both: 32 sequences of 8B heads, one
// of 1023 new tokens, 170.1 and 163.6 us; 20 with a window of 1000, 900 new tokens, 116.6 and 110.8).
struct JoinParams {
    RaggedParams few, tile;
    uint32_t few_blocks;
    int few_per_row, few_per_place, tile_per_row, tile_per_token;
};
template <typename A, int L, bool kByWorker, bool kScored>
__global__ __launch_bounds__(kThreads) void JoinBoth(const JoinParams p) {
    __shared__ f32x4 sums[kThreads / L][L];
    if (blockIdx.x < p.few_blocks) {
        JoinFewRows<A, L, kByWorker, kScored>(p.few, blockIdx.x, p.few_per_row, p.few_per_place, sums);
    } else {
        JoinTileRows<A, L, kScored>(p.tile, blockIdx.x - p.few_blocks, p.tile_per_row, p.tile_per_token, sums);
    }
}

// `few`, `tile`: null where those rows have no parts.
template <typename A, int L, bool kScored>
void StartJoin(const RaggedParams* few, const RaggedParams* tile, hipStream_t s) {
    JoinParams p{};
    int64_t blocks = 0;
    if (few != nullptr) {
        p.few = *few;
        p.few_per_row = JoinFewPerRow(*few);
        p.few_per_place = static_cast<int>(JoinFewPerPlace(*few));
        blocks = JoinFewBlocks(*few);
        p.few_blocks = static_cast<uint32_t>(blocks);
    }
    if (tile != nullptr) {
        p.tile = *tile;
        p.tile_per_row = PerRow(JoinGroups(*tile), tile->n_chunks);
        p.tile_per_token = static_cast<int>(JoinTilePerToken(*tile));
        blocks += JoinTileBlocks(*tile);
    }
    const dim3 grid(static_cast<unsigned>(blocks)), block(kThreads);
    const bool by_worker = few != nullptr && JoinByWorker(*few);
    if (few == nullptr) {
        hipLaunchKernelGGL((JoinTile<A, L, kScored>), grid, block, 0, s, p.tile, p.tile_per_row, p.tile_per_token);
    } else if (tile == nullptr) {
        if (by_worker) hipLaunchKernelGGL((JoinFew<A, L, true, kScored>), grid, block, 0, s, p.few, p.few_per_row, p.few_per_place);
        else hipLaunchKernelGGL((JoinFew<A, L, false, kScored>), grid, block, 0, s, p.few, p.few_per_row, p.few_per_place);
    } else {
        if (by_worker) hipLaunchKernelGGL((JoinBoth<A, L, true, kScored>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((JoinBoth<A, L, false, kScored>), grid, block, 0, s, p);
    }
}
template <bool kScored>
mlk_status LaunchJoin(const RaggedParams* few, const RaggedParams* tile, int32_t type, hipStream_t s) {
    const bool narrow = JoinGroups(few != nullptr ? *few : *tile) == 8;
    if (type == MLK_F32) (narrow ? StartJoin<F32, 32, kScored> : StartJoin<F32, 64, kScored>)(few, tile, s);
    else if (type == MLK_F16) (narrow ? StartJoin<F16, 32, kScored> : StartJoin<F16, 64, kScored>)(few, tile, s);
    else (narrow ? StartJoin<BF16, 32, kScored> : StartJoin<BF16, 64, kScored>)(few, tile, s);
    return CheckLaunch("Join");
}

// ------------------------------------------------------------ the kernels' launches

template <int HD, bool kScored>
struct FewAt {
    static mlk_status Run(const RaggedParams& p, dim3 grid, int32_t type, int32_t cache_type, hipStream_t s) {
        return LaunchFewAt<HD, kScored>(p, grid, type, cache_type, s);
    }
};
template <int HD, bool kScored>
struct TileAt {
    static mlk_status Run(const RaggedParams& p, dim3 grid, int64_t slots, int32_t type, int32_t cache_type, hipStream_t s) {
        return LaunchTileAt<HD, kScored>(p, grid, slots, type, cache_type, s);
    }
};

template <bool kScored>
mlk_status LaunchFew(const RaggedParams& p, int32_t type, int32_t cache_type, hipStream_t stream) {
    if (p.workers != 0) {
        return ByDim<FewAt, kScored>(p.rows.head_dim, p, dim3(static_cast<unsigned>(p.workers)), type,
                            cache_type, stream);
    }
    RaggedParams part = p;
    const int64_t most = kMaxBlocks / p.n_kv_heads;  // sequences of a launch
    mlk_status st = MLK_OK;
    for (part.taken = 0; part.taken < p.batch.n_seqs && st == MLK_OK; part.taken += most) {
        const int64_t left = p.batch.n_seqs - part.taken;
        const dim3 grid(static_cast<unsigned>((left < most ? left : most) * p.n_kv_heads));
        st = ByDim<FewAt, kScored>(p.rows.head_dim, part, grid, type, cache_type, stream);
    }
    return st;
}

// Row tiles of a batch: sequence s owns the slots from start[s] * group / rows
// + s on, at least as many as it has tiles, whatever the lengths.
int64_t TileSlots(int64_t n_seqs, int64_t n_tokens, int32_t group, int rows) {
    return n_tokens * group / rows + n_seqs;
}
int64_t TileBlocks(const RaggedParams& p) {
    return TileSlots(p.batch.n_seqs, p.batch.n_tokens, p.group, TileRows(p.rows.head_dim)) *
           p.n_chunks * p.n_kv_heads;
}

template <bool kScored>
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
        st = ByDim<TileAt, kScored>(p.rows.head_dim, part, grid, slots, type, cache_type, stream);
    }
    return st;
}

// ------------------------------------------------------------ the plan

int64_t Larger(int64_t a, int64_t b) { return a > b ? a : b; }
int64_t RoundUp(int64_t a, int64_t to) { return (a + to - 1) / to * to; }

struct Plan {
    int64_t few_rows = 0, few_workers = 0, few_partials = 0;
    bool tile = false;
    int64_t chunk = 0, n_chunks = 1, tile_partials = 0;
};

int64_t PartBytes(int64_t partials, int32_t hd) {
    return RoundUp(RoundUp(partials * 4 * hd, 16) + partials * 8, 256);
}
int64_t PlanBytes(const Plan& plan, int32_t hd) {
    return PartBytes(plan.few_partials, hd) + PartBytes(plan.tile_partials, hd);
}

constexpr int64_t kFewUnsplit = 512;   // longest sequences that are not split
constexpr int64_t kTileLeast = 256;    // positions of a tile row's least chunk
constexpr int64_t kTileMost = 64;      // most chunks of a tile row
constexpr int64_t kTileFixed = 300;    // what a tile's start and end cost, in positions
constexpr int64_t kTileJoin = 300;     // what the join costs

// Positions that the rows of `tokens` neighbouring tokens see at most, of max_len, from a
// multiple of `align` on.
int64_t SpanOf(const Scores& scores, int64_t max_len, int64_t tokens, int64_t align) {
    if (scores.window == 0 || scores.prefix != nullptr) return max_len;
    const int64_t span = scores.window + tokens + align;
    return span < max_len ? span : max_len;
}

Plan MakePlan(int64_t n_seqs, int64_t n_tokens, int64_t max_new, int64_t longest, int32_t n_heads,
              int32_t n_kv_heads, int32_t head_dim, bool packed, const Scores& scores,
              bool scored) {
    Plan plan;
    const int64_t group = n_heads / n_kv_heads, cus = ComputeUnits();
    int64_t max_len = SpanOf(scores, longest, max_new, kFewKeys);
    const int64_t most = FewMost(head_dim), max_rows = max_new * group;
    plan.tile = max_rows > most;
    // a mixed batch of short sequences is left to the tile kernel alone
    if (!plan.tile || (!packed && n_seqs > 1 && group <= 16 && max_len > kFewUnsplit &&
                       n_tokens < n_seqs * max_new)) {
        // beside the tile kernel one block of rows, decode steps', is enough
        const int64_t limit = plan.tile ? 16 : most;
        plan.few_rows = max_rows < limit ? max_rows : limit;
        if (max_len > kFewUnsplit) {
            const int64_t units = n_seqs * n_kv_heads * ((max_len + kFewKeys - 1) / kFewKeys + kFewRun);
            // 8 waves per compute unit: two such workgroups' loads get in each other's
            // way (64 bf16 decode rows of the 8B heads: 189 us, with twice as many 213)
            plan.few_workers = cus * 8 / FewWaves(head_dim, static_cast<int32_t>(plan.few_rows));
            const int64_t most_workers = (units + kFewRun - 1) / kFewRun;
            if (plan.few_workers > most_workers) plan.few_workers = most_workers;
            plan.few_partials = 2 * plan.few_workers * kFewHeads * plan.few_rows;
        }
    }
    if (plan.tile) {
        // Positions split into n chunks where that shortens the call: a compute unit has
        // one tile at a time, so rounds(n) * (chunk + kTileFixed), and the join if any
        // (1023 bf16 tokens after 3000 beside 31 decode rows: n = 1 252 us, 2 171, 3 210;
        // 3 x 448 fp16 tokens after 2800: n = 2 206, 3 172; 2500 packed fp32 tokens in 9
        // prompts: n = 1 120, 2 160; all of the 8B heads).
        // The tiles are estimated: in a mixed batch all sequences but one bring one token,
        // in others each but one has half a tile more than its rows fill.
        max_len = SpanOf(scores, longest, TileRows(head_dim) / group + 1, kTileAlign);
        const bool mixed = plan.few_rows > 0;
        const int64_t rows = (n_tokens - (mixed ? n_seqs - 1 : 0)) * group;
        const int64_t each = TileRows(head_dim);
        const int64_t tiles =
            ((rows + each - 1) / each + (mixed ? 0 : (n_seqs - 1) / 2)) * n_kv_heads;
        RaggedParams grid{};  // what a launch's size follows from
        grid.batch.n_seqs = static_cast<int32_t>(n_seqs);
        grid.batch.n_tokens = static_cast<int32_t>(n_tokens);
        grid.rows.head_dim = head_dim;
        grid.n_heads = n_heads;
        grid.n_kv_heads = n_kv_heads;
        grid.group = static_cast<int32_t>(group);
        int64_t best = INT64_MAX;
        for (int64_t n = 1; n <= kTileMost && (n == 1 || (n - 1) * kTileLeast < max_len); ++n) {
            grid.n_chunks = static_cast<int32_t>(n);
            if (n > 1 && (TileBlocks(grid) > kMaxBlocks || JoinTileBlocks(grid) > kMaxBlocks)) break;
            // (a window's span is short: rounded to whole tiles, its chunks stay alike; 900 fp32
            // tokens over fp16, a window of 1000, the whole call: two chunks of 576 123 us, of 768
            // and 329 137)
            int64_t chunk = RoundUp((max_len + n - 1) / n, scored ? kTileAlign : kTileLeast);
            if (chunk < kTileLeast) chunk = kTileLeast;
            const int64_t cost = ((tiles < 1 ? 1 : tiles) * n + cus - 1) / cus * (chunk + kTileFixed) +
                                 (n > 1 ? kTileJoin : 0);
            if (cost < best) {
                best = cost;
                plan.chunk = chunk;
            }
        }
        plan.n_chunks = (max_len + plan.chunk - 1) / plan.chunk;
        if (plan.n_chunks > 1) plan.tile_partials = n_tokens * n_heads * plan.n_chunks;
    }
    return plan;
}

bool Multiple8(int64_t a) { return a % 8 == 0; }

}  // namespace

int64_t AttendWorkspace(int64_t n_seqs, int64_t n_tokens, int64_t max_new, int64_t max_len,
                        int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, bool packed,
                        const Scores& scores, bool scored) {
    if (n_seqs <= 0 || n_tokens <= 0 || max_new <= 0 || max_len <= 0 || n_heads <= 0 ||
        n_kv_heads <= 0 || n_heads % n_kv_heads != 0 || n_heads > 65536 || head_dim <= 0 ||
        head_dim > 256 || n_seqs > kMaxSeqs || n_tokens > kMaxTokens || max_len > (1 << 30)) {
        return 0;
    }
    if (packed && max_len > n_tokens) max_len = n_tokens;
    if (max_new > max_len) max_new = max_len;
    if (max_new > n_tokens) max_new = n_tokens;
    return PlanBytes(
        MakePlan(n_seqs, n_tokens, max_new, max_len, n_heads, n_kv_heads, head_dim, packed, scores,
                 scored),
        head_dim);
}

template <bool kScored>
mlk_status AttendAs(const AttendArgs& a) {
    const int32_t hd = a.rows.head_dim;
    const Ragged& b = a.batch;
    Plan plan = MakePlan(b.n_seqs, b.n_tokens, b.max_new, b.max_len, a.n_heads, a.n_kv_heads, hd,
                         b.table == nullptr, a.scores, kScored);
    if (static_cast<int64_t>(a.workspace_bytes) < PlanBytes(plan, hd)) {  // no split
        plan.few_workers = plan.few_partials = plan.tile_partials = 0;
        plan.chunk = b.max_len;
        plan.n_chunks = 1;
    }
    RaggedParams p{};
    p.batch = b;
    p.rows = a.rows;
    p.q = a.q;
    p.q_row = a.q_row;
    p.out = a.out;
    p.n_heads = a.n_heads;
    p.n_kv_heads = a.n_kv_heads;
    p.group = a.n_heads / a.n_kv_heads;
    const bool capped = a.scores.softcap > 0.0f;
    p.factor = capped ? a.scale / a.scores.softcap : a.scale * kLog2e;
    p.scores = a.scores;
    p.cap = a.scores.softcap * kLog2e;
    p.vec = hd % 8 == 0 && Multiple8(a.q_row) && Multiple8(a.rows.k_row) &&
            Multiple8(a.rows.v_row) && Multiple8(a.rows.page_stride) && Aligned(a.q, 16) &&
            Aligned(a.rows.k, 16) && Aligned(a.rows.v, 16) && Aligned(a.out, 16);
    p.few_rows = static_cast<int32_t>(plan.few_rows);
    p.err = a.err;
    char* ws = static_cast<char*>(a.workspace);
    auto place = [&](int64_t partials, RaggedParams* to) {
        to->part_o = reinterpret_cast<float*>(ws);
        to->part_ml = reinterpret_cast<float2*>(ws + RoundUp(partials * 4 * hd, 16));
        ws += PartBytes(partials, hd);
    };
    RaggedParams few = p, tile = p;
    int64_t blocks = 0;
    if (plan.few_rows > 0) {
        few.workers = static_cast<int32_t>(plan.few_workers);
        few.few_heads = FewWaves(hd, few.few_rows);
        while (a.n_kv_heads % few.few_heads != 0) few.few_heads /= 2;
        if (few.workers > 0 && JoinFewBlocks(few) > kMaxBlocks) few.workers = 0;  // thousands of heads: no split
        if (few.workers > 0) place(plan.few_partials, &few);
        blocks = static_cast<int64_t>(b.n_seqs) * a.n_kv_heads;
    }
    if (plan.tile) {
        tile.chunk = static_cast<int32_t>(plan.chunk);
        tile.n_chunks = static_cast<int32_t>(plan.n_chunks);
        if (tile.n_chunks > 1) place(plan.tile_partials, &tile);
        blocks = Larger(blocks, TileBlocks(tile) / tile.n_chunks);
    }
    // (depends neither on the lengths nor on the workspace)
    if (blocks > kMaxCallBlocks) {
        return Fail(MLK_ERR_INVALID, "attention: %lld workgroups exceed a call's 2^35",
                    static_cast<long long>(blocks));
    }
    mlk_status st = MLK_OK;
    if (plan.few_rows > 0) st = LaunchFew<kScored>(few, a.type, a.cache_type, a.stream);
    if (plan.tile && st == MLK_OK) st = LaunchTile<kScored>(tile, a.type, a.cache_type, a.stream);
    if (st != MLK_OK) return st;
    const bool join_few = plan.few_rows > 0 && few.workers > 0, join_tile = plan.tile && tile.n_chunks > 1;
    if (!join_few && !join_tile) return MLK_OK;
    return LaunchJoin<kScored>(join_few ? &few : nullptr, join_tile ? &tile : nullptr, a.type, a.stream);
}

mlk_status Attend(const AttendArgs& a) { return AttendAs<false>(a); }
mlk_status AttendScored(const AttendArgs& a) { return AttendAs<true>(a); }

}  // namespace mlk
