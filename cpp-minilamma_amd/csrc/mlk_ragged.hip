// mlk_ragged.hip -- attention of many sequences' tokens, over pages of a cache
// or over rows of a packed buffer.
//
// Token row t at position p of its sequence, head h on KV head h / (H / KV):
//   s_j = scale (q . k_j), j <= p;  w = softmax(s);  out = sum_j w_j v_j.
//
// One wave per token and head: 64 positions at a time, a score per lane (q in
// shared memory), the running maximum and sum of the softmax, then the
// weighted rows with a lane per dim.
#include "mlk_paged.h"

#include <climits>
#include <cmath>

namespace mlk {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;

template <typename A, typename C>
__global__ __launch_bounds__(kThreads) void RaggedRows(AttendArgs p) {
    __shared__ float qs[kThreads / kWave][kMaxDim];
    const int wave = static_cast<int>(threadIdx.x) / kWave;
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    if (blockIdx.x == 0) CheckSeqs(p.batch, p.err);
    const int64_t id = static_cast<int64_t>(blockIdx.x) * (kThreads / kWave) + wave;
    const int32_t t = static_cast<int32_t>(id / p.n_heads);
    const int h = static_cast<int>(id % p.n_heads);
    if (t >= p.batch.n_tokens) return;
    const int s = LastSeq(p.batch, t, [](int32_t a, int) { return a; });
    Seq q;
    if (!LoadSeq(p.batch, s, &q) || t < q.t0 || t >= q.t0 + q.n) return;
    const int hd = p.rows.head_dim;
    const int32_t pos = q.len - q.n + (t - q.t0);
    const int kvh = h / (p.n_heads / p.n_kv_heads);
    typedef typename A::Bits AB;
    typedef typename C::Bits CB;
    const AB* qr = static_cast<const AB*>(p.q) + t * p.q_row + static_cast<int64_t>(h) * hd;
    for (int d = lane; d < hd; d += kWave) qs[wave][d] = A::Get(qr[d]);
    __builtin_amdgcn_wave_barrier();
    const int32_t* table = p.batch.table == nullptr
                               ? nullptr : p.batch.table + s * p.batch.table_stride;
    float m = -INFINITY, l = 0.0f, acc[kMaxDim / kWave] = {};
    for (int32_t j0 = 0; j0 <= pos; j0 += kWave) {
        const int32_t j = j0 + lane <= pos ? j0 + lane : pos;
        int64_t ko, vo;
        if (table != nullptr) {
            bool bad = false;
            ko = vo = PagedRow(p.rows, PageOf(p.rows, table, j, &bad), j);
            if (bad) RaiseFlag(p.err, 1);
        } else {
            ko = static_cast<int64_t>(q.t0 + j) * p.rows.k_row;
            vo = static_cast<int64_t>(q.t0 + j) * p.rows.v_row;
        }
        const CB* kr = static_cast<const CB*>(p.rows.k) + ko + static_cast<int64_t>(kvh) * hd;
        float sc = 0.0f;
        for (int d = 0; d < hd; ++d) sc = fmaf(qs[wave][d], C::Get(kr[d]), sc);
        sc = j0 + lane <= pos ? sc * p.scale : -INFINITY;
        const float mn = fmaxf(m, WaveMax(sc));
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float alpha = expf(m - base);
        const float w = j0 + lane <= pos ? expf(sc - base) : 0.0f;
        m = mn;
        float sum = w;
        for (int off = kWave / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
        l = l * alpha + sum;
#pragma unroll
        for (int i = 0; i < kMaxDim / kWave; ++i) acc[i] *= alpha;
        const int n = pos - j0 + 1 < kWave ? pos - j0 + 1 : kWave;
        for (int i = 0; i < n; ++i) {
            const float wi = __shfl(w, i, kWave);
            const int64_t o = __shfl(vo, i, kWave);
            const CB* vr = static_cast<const CB*>(p.rows.v) + o + static_cast<int64_t>(kvh) * hd;
#pragma unroll
            for (int e = 0; e < kMaxDim / kWave; ++e) {
                if (e * kWave + lane < hd) acc[e] = fmaf(wi, C::Get(vr[e * kWave + lane]), acc[e]);
            }
        }
    }
    AB* o = static_cast<AB*>(p.out) + (static_cast<int64_t>(t) * p.n_heads + h) * hd;
#pragma unroll
    for (int e = 0; e < kMaxDim / kWave; ++e) {
        if (e * kWave + lane < hd) o[e * kWave + lane] = A::Put(acc[e] / l);
    }
}

template <typename A, typename C>
mlk_status Launch(const AttendArgs& a) {
    const int64_t waves = static_cast<int64_t>(a.batch.n_tokens) * a.n_heads;
    const int64_t blocks = (waves + kThreads / kWave - 1) / (kThreads / kWave);
    if (blocks > INT32_MAX) {
        return Fail(MLK_ERR_INVALID, "attention: n_tokens * n_heads exceeds 2^31 waves");
    }
    hipLaunchKernelGGL((RaggedRows<A, C>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                       a.stream, a);
    return CheckLaunch("RaggedRows");
}

}  // namespace

int64_t AttendWorkspace(int64_t, int64_t, int64_t, int64_t, int32_t, int32_t, int32_t) {
    return 0;
}

mlk_status Attend(const AttendArgs& a) {
    if (a.type == MLK_F16) return Launch<F16, F16>(a);
    if (a.type == MLK_BF16) return Launch<BF16, BF16>(a);
    if (a.cache_type == MLK_F16) return Launch<F32, F16>(a);
    if (a.cache_type == MLK_BF16) return Launch<F32, BF16>(a);
    return Launch<F32, F32>(a);
}

}  // namespace mlk
