// mlk_scored.hip -- attention of many sequences' tokens with score functions and
// masks, one workgroup a (token row, head): the scores of 256 positions at a time,
// then their weights times V, dim by dim, with the running maximum and sum of the
// softmax.
#include "mlk_paged.h"

#include <cmath>

namespace mlk {
namespace {

constexpr int kThreads = 256;

template <typename A, typename C>
__global__ __launch_bounds__(kThreads) void AttnScored(const AttendArgs p) {
    __shared__ float sq[256], sw[kThreads], scratch[2][kThreads / kWave];
    __shared__ int64_t srow[kThreads];
    const int tid = static_cast<int>(threadIdx.x), hd = p.rows.head_dim;
    if (blockIdx.x == 0) CheckSeqs(p.batch, p.err);
    const int32_t t = static_cast<int32_t>(blockIdx.x / p.n_heads);
    const int h = static_cast<int>(blockIdx.x % p.n_heads), kvh = h / (p.n_heads / p.n_kv_heads);
    const int s = LastSeq(p.batch, t, [](int32_t a, int) { return a; });
    Seq q;
    if (!LoadSeq(p.batch, s, &q) || t < q.t0 || t >= q.t0 + q.n) return;
    const int32_t pos = q.len - q.n + (t - q.t0);
    const Seen seen = SeenBy(p.scores, s, t, pos, q.len);
    const int32_t* table = p.batch.table == nullptr ? nullptr : p.batch.table + s * p.batch.table_stride;
    const typename A::Bits* qr = static_cast<const typename A::Bits*>(p.q) + t * p.q_row + h * hd;
    const typename C::Bits* k = static_cast<const typename C::Bits*>(p.rows.k) + kvh * hd;
    const typename C::Bits* v = static_cast<const typename C::Bits*>(p.rows.v) + kvh * hd;
    if (tid < hd) sq[tid] = A::Get(qr[tid]);
    const float slope = p.scores.slopes != nullptr ? p.scores.slopes[h] : 0.0f, cap = p.scores.softcap;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    bool bad = false;
    __syncthreads();
    for (int32_t j0 = seen.lo; j0 <= seen.hi; j0 += kThreads) {
        const int32_t j = j0 + tid;
        float x = -INFINITY;
        if (j <= seen.hi) {
            int64_t ko = (static_cast<int64_t>(q.t0) + j) * p.rows.k_row, vo = (static_cast<int64_t>(q.t0) + j) * p.rows.v_row;
            if (table != nullptr) ko = vo = PagedRow(p.rows, PageOf(p.rows, table, j, &bad), j);
            srow[tid] = vo;
            float dot = 0.0f;
            for (int d = 0; d < hd; ++d) dot = fmaf(sq[d], C::Get(k[ko + d]), dot);
            x = dot * p.scale;
            if (cap > 0.0f) x = cap * tanhf(x / cap);
            if (p.scores.slopes != nullptr) x -= slope * fabsf(static_cast<float>(pos - j));
        }
        const float top = fmaxf(m, BlockMax<kThreads / kWave>(x, scratch[0]));
        const float base = top == -INFINITY ? 0.0f : top;
        const float w = expf(x - base);
        sw[tid] = w;
        const float f = expf(m - base);
        l = l * f + w;  // this thread's part
        o *= f;
        m = top;
        __syncthreads();
        const int n = seen.hi - j0 + 1 < kThreads ? seen.hi - j0 + 1 : kThreads;
        if (tid < hd) {
            for (int i = 0; i < n; ++i) o = fmaf(sw[i], C::Get(v[srow[i] + tid]), o);
        }
        __syncthreads();
    }
    if (bad) RaiseFlag(p.err, 1);
    double all = WaveSum(static_cast<double>(l));
    if (tid % kWave == 0) scratch[1][tid / kWave] = static_cast<float>(all);
    __syncthreads();
    float sum = 0.0f;
    for (int i = 0; i < kThreads / kWave; ++i) sum += scratch[1][i];
    if (tid < hd) {
        static_cast<typename A::Bits*>(p.out)[(static_cast<int64_t>(t) * p.n_heads + h) * hd + tid] =
            A::Put(seen.lo > seen.hi ? 0.0f : o / sum);
    }
}

}  // namespace

mlk_status AttendScored(const AttendArgs& a) {
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.batch.n_tokens) * a.n_heads)), block(kThreads);
    const hipStream_t s = a.stream;
    if (a.type == MLK_F16) hipLaunchKernelGGL((AttnScored<F16, F16>), grid, block, 0, s, a);
    else if (a.type == MLK_BF16) hipLaunchKernelGGL((AttnScored<BF16, BF16>), grid, block, 0, s, a);
    else if (a.cache_type == MLK_F16) hipLaunchKernelGGL((AttnScored<F32, F16>), grid, block, 0, s, a);
    else if (a.cache_type == MLK_BF16) hipLaunchKernelGGL((AttnScored<F32, BF16>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((AttnScored<F32, F32>), grid, block, 0, s, a);
    return CheckLaunch("AttnScored");
}

}  // namespace mlk
