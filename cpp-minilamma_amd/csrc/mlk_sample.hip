// mlk_sample.hip -- the next token of each row of logits: temperature, top-k,
// top-p and min-p, from given uniform numbers.
//
// In descending order of the logits (the lower index first where they are equal),
// with w_i = exp((x_i - x_1) / T) and C_n = w_1 + .. + w_n, the tokens kept are the
// first n = max(1, min(n_k, n_p, n_m)), and the one chosen is the first with C_i >
// u C_n.  Nothing is sorted: each cut is a search for the place in that order where a
// count or a sum crosses a bound, by histograms of the order's digits (an element's
// place is its logit's bits, descending, then its index), each pass over the row
// narrowing the place by one digit.  Sums are of whole numbers, w_i 2^42 rounded: they
// do not depend on the order in which they are added.
#include "mlk_paged.h"

#include <cmath>

namespace mlk {
namespace {

constexpr int kThreads = 1024, kBins = 2048;
constexpr int64_t kMaxVocab = 1 << 20, kMaxRows = 1 << 20;
constexpr int kIndexBits = 20;
constexpr double kOne = 0x1p42;  // a weight of 1

struct SampleArgs {
    const void* x;
    int64_t row;  // elements
    int32_t vocab;
    mlk_sampling how;
    const float* u;
    int32_t* tokens;
    float* prob;
    int32_t* err;
};

// Descending order of logits as ascending whole numbers; equal for +0 and -0.
__device__ inline uint32_t Descending(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b >> 31 ? b : ~b & 0x7FFFFFFFu;
}

struct Row {
    const void* x;
    int32_t vocab;
    float top;       // the largest logit
    double inverse;  // 1 / temperature
};

__device__ inline uint64_t Weight(const Row& r, float x) {
    if (x == r.top) return static_cast<uint64_t>(kOne);
    const double w = exp((static_cast<double>(x) - r.top) * r.inverse);
    return static_cast<uint64_t>(rint(w * kOne));
}

enum Bound { kCount, kReach, kPass };  // count >= bound, sum >= bound, sum > bound

// The first place in the order whose count (or sum) meets `bound`, the sum up to
// and with it, and its own weight.
struct Place {
    uint64_t key, sum, own;
};

template <typename T>
__device__ Place Search(const Row& r, Bound what, uint64_t bound, uint32_t* cnt, uint64_t* mass,
                        uint64_t* shared) {
    const int tid = static_cast<int>(threadIdx.x);
    const typename T::Bits* x = static_cast<const typename T::Bits*>(r.x);
    uint64_t high = 0, n0 = 0, m0 = 0, own = 0;
    const int shifts[5] = {41, 30, 20, 10, 0}, bits[5] = {11, 11, 10, 10, 10};
    for (int d = 0; d < 5; ++d) {
        for (int i = tid; i < kBins; i += kThreads) {
            cnt[i] = 0;
            mass[i] = 0;
        }
        __syncthreads();
        for (int i = tid; i < r.vocab; i += kThreads) {
            const float v = T::Get(x[i]);
            if (v == -INFINITY) continue;
            const uint64_t key = (static_cast<uint64_t>(Descending(v)) << kIndexBits) | static_cast<uint32_t>(i);
            if (key >> (shifts[d] + bits[d]) != high) continue;
            const int b = static_cast<int>(key >> shifts[d]) & ((1 << bits[d]) - 1);
            atomicAdd(&cnt[b], 1u);
            atomicAdd(reinterpret_cast<unsigned long long*>(&mass[b]), static_cast<unsigned long long>(Weight(r, v)));
        }
        __syncthreads();
        if (tid == 0) {
            uint64_t n = n0, m = m0;
            int last = -1, at = -1;
            for (int b = 0; b < 1 << bits[d]; ++b) {
                if (cnt[b] == 0) continue;
                last = b;
                const uint64_t n1 = n + cnt[b], m1 = m + mass[b];
                if (what == kCount ? n1 >= bound : what == kReach ? m1 >= bound : m1 > bound) {
                    at = b;
                    break;
                }
                n = n1;
                m = m1;
            }
            if (at < 0) {  // none does: the last element
                at = last;
                n -= cnt[at];
                m -= mass[at];
            }
            shared[0] = at;
            shared[1] = n;
            shared[2] = m;
            shared[3] = mass[at];
        }
        __syncthreads();
        high = (high << bits[d]) | shared[0];
        n0 = shared[1];
        m0 = shared[2];
        own = shared[3];
        __syncthreads();
    }
    return {high, m0 + own, own};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void SampleRow(const SampleArgs p) {
    __shared__ uint32_t cnt[kBins];
    __shared__ uint64_t mass[kBins], shared[4];
    __shared__ float tops[kThreads / kWave];
    const int tid = static_cast<int>(threadIdx.x);
    const int64_t row = blockIdx.x;
    const typename T::Bits* x = static_cast<const typename T::Bits*>(p.x) + row * p.row;
    const float t = p.how.temperature != nullptr ? p.how.temperature[row] : 1.0f;
    const int32_t k = p.how.top_k != nullptr ? p.how.top_k[row] : 0;
    const float top_p = p.how.top_p != nullptr ? p.how.top_p[row] : 1.0f;
    const float min_p = p.how.min_p != nullptr ? p.how.min_p[row] : 0.0f;
    const float u = t == 0.0f ? 0.0f : p.u[row];
    bool bad = !(t >= 0.0f) || !(u >= 0.0f && u < 1.0f) || top_p != top_p || min_p != min_p;
    float top = -INFINITY;
    for (int i = tid; i < p.vocab; i += kThreads) {
        const float v = T::Get(x[i]);
        if (v != v) bad = true;
        top = fmaxf(top, v);
    }
    top = BlockMax<kThreads / kWave>(top, tops);
    bad = __syncthreads_or(bad || top == -INFINITY);
    if (bad) {
        if (tid == 0) {
            p.tokens[row] = -1;
            if (p.prob != nullptr) p.prob[row] = 0.0f;
            RaiseFlag(p.err, 1);
        }
        return;
    }
    const Row r{x, p.vocab, top, 1.0 / fmaxf(t, 0x1p-14f)};
    Place cut = Search<T>(r, kCount, t == 0.0f ? 1 : k > 0 ? k : p.vocab, cnt, mass, shared);
    uint64_t kept = cut.sum;
    if (top_p < 1.0f) {
        const double bound = ceil(static_cast<double>(top_p) * static_cast<double>(kept));
        cut = Search<T>(r, kReach, bound < 1.0 ? 1 : static_cast<uint64_t>(bound), cnt, mass, shared);
        kept = cut.sum < kept ? cut.sum : kept;
    }
    if (min_p > 0.0f) {
        uint64_t sum = 0;
        for (int i = tid; i < p.vocab; i += kThreads) {
            const float v = T::Get(x[i]);
            const uint64_t w = v == -INFINITY ? 0 : Weight(r, v);
            if (static_cast<double>(w) >= static_cast<double>(min_p) * kOne) sum += w;
        }
        if (tid == 0) shared[0] = 0;
        __syncthreads();
        atomicAdd(reinterpret_cast<unsigned long long*>(shared), static_cast<unsigned long long>(sum));
        __syncthreads();
        kept = shared[0] < kept ? shared[0] : kept;
        if (kept == 0) kept = static_cast<uint64_t>(kOne);
        __syncthreads();
    }
    const uint64_t bound = static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(kept));
    const Place at = Search<T>(r, kPass, bound, cnt, mass, shared);
    if (tid == 0) {
        p.tokens[row] = static_cast<int32_t>(at.key & ((1 << kIndexBits) - 1));
        if (p.prob != nullptr) p.prob[row] = static_cast<float>(static_cast<double>(at.own) / static_cast<double>(kept));
    }
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
    return 16;
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
    const dim3 grid(static_cast<unsigned>(n_rows)), block(kThreads);
    const hipStream_t s = AsStream(stream);
    if (type == MLK_F32) hipLaunchKernelGGL(SampleRow<F32>, grid, block, 0, s, p);
    else if (type == MLK_F16) hipLaunchKernelGGL(SampleRow<F16>, grid, block, 0, s, p);
    else hipLaunchKernelGGL(SampleRow<BF16>, grid, block, 0, s, p);
    return CheckLaunch("SampleRow");
}

}  // extern "C"
