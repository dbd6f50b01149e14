// mlk_ragged.hip -- attention of many sequences' tokens, over pages of a cache
// or over rows of a packed buffer: which kernels a call runs, how it splits
// positions, and the join of split rows.
//
// Token row t at position p of its sequence, head h on KV head h / (H / KV):
//   s_j = scale (q . k_j), j <= p;  w = softmax(s);  out = sum_j w_j v_j.
// Sequences of few rows (new tokens x query heads of a group, at most FewMost)
// are bound by the bytes of K and V (mlk_ragged_few.hip); the others by the
// matrix cores (mlk_ragged_tile.hip).  A batch of both kinds runs both kernels,
// each leaving the other's sequences alone.
#include "mlk_ragged.h"

namespace mlk {
namespace {

constexpr int kThreads = 256;

// out = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c over a row's chunks, a wave
// per row, chunks in order.
template <typename A, bool kFew>
__global__ __launch_bounds__(kThreads) void AttnJoin(const RaggedParams p) {
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * (kThreads / kWave) +
                       __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int hd = p.rows.head_dim;
    Seq q;
    int64_t base;
    int32_t t, h, n;
    if constexpr (kFew) {
        const int row = static_cast<int>(id % p.few_rows);
        const int64_t rest = id / p.few_rows;
        const int kvh = static_cast<int>(rest % p.n_kv_heads);
        const int64_t s = rest / p.n_kv_heads;
        if (s >= p.batch.n_seqs || !LoadSeq(p.batch, static_cast<int>(s), &q)) return;
        const int64_t rows = static_cast<int64_t>(q.n) * p.group;
        if (rows > p.few_rows || row >= rows || q.len <= p.chunk) return;
        t = q.t0 + row / p.group;
        h = kvh * p.group + row % p.group;
        n = (q.len + p.chunk - 1) / p.chunk;
        base = FewPartial(p, static_cast<int>(s), kvh, row);
    } else {
        if (id >= static_cast<int64_t>(p.batch.n_tokens) * p.n_heads) return;
        t = static_cast<int32_t>(id / p.n_heads);
        h = static_cast<int32_t>(id % p.n_heads);
        const int s = LastSeq(p.batch, t, [](int32_t a, int) { return a; });
        if (!LoadSeq(p.batch, s, &q) || t < q.t0 || t >= q.t0 + q.n) return;
        const int32_t pos = q.len - q.n + (t - q.t0);
        if (static_cast<int64_t>(q.n) * p.group <= p.few_rows || pos < p.chunk) return;
        n = pos / p.chunk + 1;
        base = TilePartial(p, t, h);
    }
    float m = -INFINITY;
    for (int c = lane; c < n; c += kWave) m = fmaxf(m, p.part_ml[base + c].x);
    m = WaveMax(m);
    if (m == -INFINITY) m = 0.0f;
    float l = 0.0f, o[4] = {0, 0, 0, 0};
    const float* part = p.part_o + base * hd;
#pragma unroll 4
    for (int c = 0; c < n; ++c) {
        const float2 ml = p.part_ml[base + c];
        const float f = __builtin_amdgcn_exp2f(ml.x - m);
        l = fmaf(ml.y, f, l);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + kWave * i;
            if (d < hd) o[i] = fmaf(part[static_cast<int64_t>(c) * hd + d], f, o[i]);
        }
    }
    typename A::Bits* out =
        static_cast<typename A::Bits*>(p.out) + (static_cast<int64_t>(t) * p.n_heads + h) * hd;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + kWave * i;
        if (d < hd) out[d] = A::Put(o[i] / l);
    }
}

template <bool kFew>
mlk_status LaunchJoin(const RaggedParams& p, int32_t type, int64_t waves, hipStream_t s) {
    const int64_t blocks = (waves + kThreads / kWave - 1) / (kThreads / kWave);
    if (blocks > 0x7FFFFFFF) return Fail(MLK_ERR_INVALID, "attention: too many rows to join");
    const dim3 grid(static_cast<unsigned>(blocks));
    if (type == MLK_F32) hipLaunchKernelGGL((AttnJoin<F32, kFew>), grid, dim3(kThreads), 0, s, p);
    else if (type == MLK_F16) hipLaunchKernelGGL((AttnJoin<F16, kFew>), grid, dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL((AttnJoin<BF16, kFew>), grid, dim3(kThreads), 0, s, p);
    return CheckLaunch("AttnJoin");
}

struct Part {
    bool run = false;
    int64_t chunk = 0, n_chunks = 1, partials = 0;  // partials: rows times chunks
    int64_t Bytes(int32_t hd) const {
        return n_chunks > 1 ? (partials * (4 * hd + 8) + 255) / 256 * 256 : 0;
    }
};
struct Plan {
    int32_t few_rows = 0;
    Part few, tile;
};

// Chunks of at least `least` positions (and a multiple of it), as many as bring
// `base` workgroups to about `want`.
Part Split(int64_t base, int64_t want, int64_t least, int64_t max_len) {
    Part part;
    part.run = true;
    int64_t n = base > 0 ? (want + base - 1) / base : 1;
    const int64_t most = (max_len + least - 1) / least;
    if (n > most) n = most;
    if (n < 1) n = 1;
    part.chunk = ((max_len + n - 1) / n + least - 1) / least * least;
    part.n_chunks = (max_len + part.chunk - 1) / part.chunk;
    return part;
}

Plan MakePlan(int64_t n_seqs, int64_t n_tokens, int64_t max_new, int64_t max_len, int32_t n_heads,
              int32_t n_kv_heads, int32_t head_dim, bool packed) {
    Plan plan;
    const int64_t group = n_heads / n_kv_heads, cus = ComputeUnits();
    const int64_t most = FewMost(head_dim), max_rows = max_new * group;
    plan.tile.run = max_rows > most;
    // a mixed batch of short sequences is left to the tile kernel alone
    plan.few.run = !plan.tile.run || (!packed && n_seqs > 1 && group <= most && max_len >= 512 &&
                                      n_tokens < n_seqs * max_new);
    if (plan.few.run) {
        plan.few_rows = static_cast<int32_t>(max_rows < most ? max_rows : most);
        plan.few = Split(n_seqs * n_kv_heads, 3 * cus, 256, max_len);
        plan.few.partials = n_seqs * n_kv_heads * plan.few_rows * plan.few.n_chunks;
    }
    if (plan.tile.run) {
        plan.tile = Split((n_tokens * group / 128 + n_seqs) * n_kv_heads, 2 * cus, 512, max_len);
        plan.tile.partials = n_tokens * n_heads * plan.tile.n_chunks;
    }
    return plan;
}

bool Multiple8(int64_t a) { return a % 8 == 0; }

}  // namespace

int64_t AttendWorkspace(int64_t n_seqs, int64_t n_tokens, int64_t max_new, int64_t max_len,
                        int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, bool packed) {
    if (n_seqs <= 0 || n_tokens <= 0 || max_new <= 0 || max_len <= 0 || n_heads <= 0 ||
        n_kv_heads <= 0 || n_heads % n_kv_heads != 0 || n_heads > 65536 || head_dim <= 0 ||
        head_dim > 256 || n_seqs > (1 << 24) || n_tokens > (1 << 28) || max_len > (1 << 30)) {
        return 0;
    }
    if (max_new > max_len) max_new = max_len;
    if (max_new > n_tokens) max_new = n_tokens;
    const Plan plan =
        MakePlan(n_seqs, n_tokens, max_new, max_len, n_heads, n_kv_heads, head_dim, packed);
    return plan.few.Bytes(head_dim) + plan.tile.Bytes(head_dim);
}

mlk_status Attend(const AttendArgs& a) {
    const int32_t hd = a.rows.head_dim;
    const Ragged& b = a.batch;
    Plan plan = MakePlan(b.n_seqs, b.n_tokens, b.max_new, b.max_len, a.n_heads, a.n_kv_heads, hd,
                         b.table == nullptr);
    if (static_cast<int64_t>(a.workspace_bytes) < plan.few.Bytes(hd) + plan.tile.Bytes(hd)) {
        for (Part* part : {&plan.few, &plan.tile}) {  // no split
            part->chunk = b.max_len;
            part->n_chunks = 1;
        }
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
    p.factor = a.scale * kLog2e;
    p.vec = hd % 8 == 0 && Multiple8(a.q_row) && Multiple8(a.rows.k_row) &&
            Multiple8(a.rows.v_row) && Multiple8(a.rows.page_stride) && Aligned(a.q, 16) &&
            Aligned(a.rows.k, 16) && Aligned(a.rows.v, 16) && Aligned(a.out, 16);
    p.few_rows = plan.few_rows;
    p.err = a.err;
    char* ws = static_cast<char*>(a.workspace);
    auto place = [&](const Part& part) {
        p.chunk = static_cast<int32_t>(part.chunk);
        p.n_chunks = static_cast<int32_t>(part.n_chunks);
        p.part_o = nullptr;
        p.part_ml = nullptr;
        if (part.n_chunks > 1) {
            p.part_o = reinterpret_cast<float*>(ws);
            p.part_ml = reinterpret_cast<float2*>(ws + part.partials * 4 * hd);
            ws += part.Bytes(hd);
        }
    };
    if (plan.few.run) {
        place(plan.few);
        mlk_status st = LaunchFew(p, a.type, a.cache_type, a.stream);
        if (st != MLK_OK) return st;
        if (p.n_chunks > 1) {
            st = LaunchJoin<true>(p, a.type, static_cast<int64_t>(b.n_seqs) * a.n_kv_heads * p.few_rows,
                                  a.stream);
            if (st != MLK_OK) return st;
        }
    }
    if (plan.tile.run) {
        place(plan.tile);
        mlk_status st = LaunchTile(p, a.type, a.cache_type, a.stream);
        if (st != MLK_OK) return st;
        if (p.n_chunks > 1) {
            st = LaunchJoin<false>(p, a.type, static_cast<int64_t>(b.n_tokens) * a.n_heads, a.stream);
            if (st != MLK_OK) return st;
        }
    }
    return MLK_OK;
}

}  // namespace mlk
