// hawk_rows.hip — losses over rows of logits on gfx950: the log-probability of
// a row's target, the clipped policy loss with a KL term, the preference loss
// of pairs of sequences, and their gradients by the logits.
//
// The mathematics.  All of them go through a row's log-sum-exp and its target:
// lse = m + log sum exp(l - m), and the gradient of any loss by a row's logits
// is c (1[v = target] - exp(l - lse)) with one number c a row.  In base 2, with
// k = scale log2(e) rounded once and used for every term of a row, the target's
// l_y k - m - log2(sum) is exact in k (a different scale by 6e-8), so nothing
// is lost between the target's term and the sum's.

#include "hawk_core.h"
#include "hawk_internal.h"
#include "hawk_vec.h"

#include <hip/hip_runtime.h>
#include <cmath>
#include <cstdint>
#include <string>

namespace {

using namespace hawk_vec;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

template <class T>
struct RowArgs {
    const T* logits;
    T* bar_logits;
    const void* target;
    float *logp, *lse;
    float* row_loss;          // each row's weighted loss, or NULL
    const float* bar_logp;    // the gradient's c (before scale), or NULL
    const float *bar_loss, *old_logp, *ref_logp, *advantage, *weight;
    int64_t rows, vocab, row_stride, bar_stride;
    float scale, low, high, kl, even;   // low, high: the ratio's bounds; even: the weight where weight is NULL
    int target64;
};

enum Work { kLogp, kPolicy, kGradient, kPolicyGradient };

// exp2 that flushes results below 2^-126 to 0, and a log2 to 1 ulp: the
// hardware's own.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ int64_t target_of(const void* target, int wide, int64_t n) {
    return wide ? static_cast<const int64_t*>(target)[n] : static_cast<const int32_t*>(target)[n];
}

// A row's loss by its log-probability (times its weight) and the loss's
// derivative by it (times weight and bar_loss).  A weight of 0 gives 0.
template <class T>
__device__ __forceinline__ void policy_row(const RowArgs<T>& a, int64_t n, float logp, float& loss, float& slope) {
    const float w = a.weight ? a.weight[n] : a.even;
    loss = slope = 0.0f;
    if (w == 0.0f) return;
    const float A = a.advantage[n];
    const float r = expf(logp - a.old_logp[n]);
    const float plain = r * A, clipped = fminf(fmaxf(r, a.low), a.high) * A;
    // a NaN ratio stays one: fminf and fmaxf would drop it
    if (!(r == r)) { loss = slope = r; return; }
    loss = plain <= clipped ? -plain : -clipped;
    slope = plain <= clipped ? -plain : 0.0f;
    if (!(A == A)) loss = slope = A;
    if (a.kl != 0.0f) {
        const float d = a.ref_logp[n] - logp;
        loss += a.kl * (expm1f(d) - d);
        slope -= a.kl * expm1f(d);
    }
    loss *= w;
    slope *= a.bar_loss ? w * *a.bar_loss : w;
}

// (m, s) of a run of a row: its largest logit x and the sum of 2^((x - m) k).
// The difference is taken before the product, so a row of the type's lowest
// value is a row of equal logits.  m = -inf with s = 0 for none above -inf.
__device__ __forceinline__ float floor_of(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2, float k) {
    const float top = fmaxf(m, m2), base = floor_of(top);
    s = s * exp2_fast((m - base) * k) + s2 * exp2_fast((m2 - base) * k);
    m = top;
}

template <class T, Work W, bool Grad>
__global__ void __launch_bounds__(kThreads) hawk_row(const RowArgs<T> a) {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const int64_t n = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T* row = a.logits + n * a.row_stride;
    const int64_t y = target_of(a.target, a.target64, n);
    const bool out = y < 0;
    const int64_t whole = a.vocab / V * V;
    T* bar = Grad ? a.bar_logits + n * a.bar_stride : nullptr;
    const float k = a.scale * kLog2e;
    float c = 0.0f, lse = 0.0f;
    if (!out) {
        const float at = y < a.vocab ? static_cast<float>(row[y]) : NAN;
        if constexpr (W == kLogp || W == kPolicy) {
            float m = -INFINITY, s = 0.0f;
            for (int64_t v = static_cast<int64_t>(tid) * V; v < whole; v += kThreads * V) {
                float x[V], top = m;
                load<T, V>(row + v, x);
#pragma unroll
                for (int j = 0; j < V; ++j) top = fmaxf(top, x[j]);
                const float base = floor_of(top);
                s *= exp2_fast((m - base) * k);
                m = top;
#pragma unroll
                for (int j = 0; j < V; ++j) s += exp2_fast((x[j] - base) * k);
            }
            for (int64_t v = whole + tid; v < a.vocab; v += kThreads) {
                const float x = static_cast<float>(row[v]), top = fmaxf(m, x), base = floor_of(top);
                s = s * exp2_fast((m - base) * k) + exp2_fast((x - base) * k);
                m = top;
            }
            __shared__ float lds_m[kWaves], lds_s[kWaves];
            for (int d = 32; d > 0; d >>= 1) {
                const float m2 = __shfl_xor(m, d), s2 = __shfl_xor(s, d);
                join(m, s, m2, s2, k);
            }
            if (lane == 0) { lds_m[wave] = m; lds_s[wave] = s; }
            __syncthreads();
            m = lds_m[0];
            s = lds_s[0];
            for (int w = 1; w < kWaves; ++w) join(m, s, lds_m[w], lds_s[w], k);
            const float base = floor_of(m), logs = log2f(s);
            lse = fused(base, a.scale, logs * kLn2);
            const float logp = ((at - base) * k - logs) * kLn2;
            float loss = 0.0f;
            if constexpr (W == kPolicy) policy_row(a, n, logp, loss, c);
            if (tid == 0) {
                if (a.logp) a.logp[n] = logp;
                if (a.lse) a.lse[n] = lse;
                if (W == kPolicy && a.row_loss) a.row_loss[n] = loss;
            }
        } else {
            lse = a.lse[n];
            if constexpr (W == kGradient) c = a.bar_logp[n];
            else {
                float loss;
                policy_row(a, n, a.logp[n], loss, c);
            }
            if (y >= a.vocab) c = NAN;
        }
    } else if ((W == kLogp || W == kPolicy) && tid == 0) {
        if (a.logp) a.logp[n] = 0.0f;
        if (a.lse) a.lse[n] = 0.0f;
        if (W == kPolicy && a.row_loss) a.row_loss[n] = 0.0f;
    }
    if constexpr (Grad) {
        c *= a.scale;
        if (out || c == 0.0f) {
            const float zero[V] = {};
            for (int64_t v = static_cast<int64_t>(tid) * V; v < whole; v += kThreads * V) store<T, V>(bar + v, zero);
            for (int64_t v = whole + tid; v < a.vocab; v += kThreads) bar[v] = static_cast<T>(0.0f);
            return;
        }
        auto gradient = [&](float x, int64_t v) {
            const float p = exp2_fast(fused(x, a.scale, -lse) * kLog2e);
            return v == y ? c - c * p : -c * p;
        };
        for (int64_t v = static_cast<int64_t>(tid) * V; v < whole; v += kThreads * V) {
            float x[V];
            load<T, V>(row + v, x);
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = gradient(x[j], v + j);
            store<T, V>(bar + v, x);
        }
        for (int64_t v = whole + tid; v < a.vocab; v += kThreads)
            bar[v] = static_cast<T>(gradient(static_cast<float>(row[v]), v));
    }
}

// The sum of `count` numbers in 64 bits: each thread its own stride in order,
// then a fixed tree.
__device__ __forceinline__ double sum_block(const float* x, int64_t count) {
    __shared__ double lds[kWaves];
    double t = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += kThreads) t += static_cast<double>(x[i]);
    for (int d = 32; d > 0; d >>= 1) t += __shfl_xor(t, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = t;
    __syncthreads();
    t = 0.0;
    for (int w = 0; w < kWaves; ++w) t += lds[w];
    return t;
}

__global__ void __launch_bounds__(kThreads) hawk_row_total(const float* x, int64_t count, float* out) {
    const double t = sum_block(x, count);
    if (threadIdx.x == 0) *out = static_cast<float>(t);
}

struct PairArgs {
    const void *offsets, *target;
    const float *logp, *ref_logp, *weight, *bar_loss;
    float *margin, *pair_loss, *bar_logp;
    int64_t rows, pairs;
    float beta, smoothing, even;
    int offsets64, target64;
};

__device__ __forceinline__ int64_t cut_of(const PairArgs& a, int64_t k) {
    const int64_t v = a.offsets64 ? static_cast<const int64_t*>(a.offsets)[k] : static_cast<const int32_t*>(a.offsets)[k];
    return v < 0 ? 0 : v > a.rows ? a.rows : v;
}

// One wave a pair: both sequences' log ratios summed in 64 bits, then the loss.
__global__ void __launch_bounds__(kThreads) hawk_pair_loss(const PairArgs a) {
    const int64_t p = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (p >= a.pairs) return;
    const int64_t c0 = cut_of(a, 2 * p), c1 = cut_of(a, 2 * p + 1), c2 = cut_of(a, 2 * p + 2);
    double t = 0.0;
    for (int64_t n = c0 + lane; n < c2; n += 64) {
        if (target_of(a.target, a.target64, n) < 0) continue;
        const double r = static_cast<double>(a.logp[n]) - (a.ref_logp ? static_cast<double>(a.ref_logp[n]) : 0.0);
        t += n < c1 ? r : -r;
    }
    for (int d = 32; d > 0; d >>= 1) t += __shfl_xor(t, d);
    if (lane != 0) return;
    const float w = a.weight ? a.weight[p] : a.even;
    const double z = static_cast<double>(a.beta) * t;
    // -log sigma(z) and -log sigma(-z) = z - log sigma(z), neither overflowing
    const double soft = log1p(exp(-fabs(z)));
    const double lose = soft + (z < 0.0 ? -z : 0.0), win = soft + (z > 0.0 ? z : 0.0);
    const double loss = (z == z) ? (1.0 - a.smoothing) * lose + a.smoothing * win : z;
    if (a.margin) a.margin[p] = static_cast<float>(t);
    if (a.pair_loss) a.pair_loss[p] = w == 0.0f ? 0.0f : static_cast<float>(w * loss);
}

// The derivative of the loss by each row's log-probability: one wave a pair.
__global__ void __launch_bounds__(kThreads) hawk_pair_slope(const PairArgs a) {
    const int64_t p = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (p >= a.pairs) return;
    const int64_t c0 = cut_of(a, 2 * p), c1 = cut_of(a, 2 * p + 1), c2 = cut_of(a, 2 * p + 2);
    const float w = a.weight ? a.weight[p] : a.even;
    float up, down;
    sigmoid(a.beta * a.margin[p], up, down);
    float slope = a.beta * w * (a.smoothing * up - (1.0f - a.smoothing) * down);
    if (a.bar_loss) slope *= *a.bar_loss;
    if (w == 0.0f) slope = 0.0f;
    for (int64_t n = c0 + lane; n < c2; n += 64) a.bar_logp[n] = n < c1 ? slope : -slope;
    // rows that no sequence holds
    if (p == 0) for (int64_t n = lane; n < c0; n += 64) a.bar_logp[n] = 0.0f;
    if (p == a.pairs - 1) for (int64_t n = c2 + lane; n < a.rows; n += 64) a.bar_logp[n] = 0.0f;
}

int check_job(const hk_row_loss_job* j, const std::string& who) {
    using hawk_internal::set_error;
    if (!j) return set_error(HK_EVALUE, who + ": a job is required");
    if (j->rows < 0 || j->vocab < 0 || j->pairs < 0) return set_error(HK_EVALUE, who + ": sizes must be >= 0");
    if (j->rows > INT32_MAX) return set_error(HK_EVALUE, who + ": more than 2^31 - 1 rows");
    if (j->dtype != HK_F32 && j->dtype != HK_BF16 && j->dtype != HK_F16)
        return set_error(HK_EVALUE, who + ": logits are 32- or 16-bit floating point");
    if (!(j->scale > 0.0f) || !std::isfinite(j->scale)) return set_error(HK_EVALUE, who + ": scale must be positive and finite");
    if (j->rows > 0 && (!j->logits || !j->target)) return set_error(HK_EVALUE, who + ": logits and target are required");
    return HK_OK;
}

template <class T>
RowArgs<T> args_of(const hk_row_loss_job& j) {
    RowArgs<T> a{};
    a.logits = static_cast<const T*>(j.logits);
    a.bar_logits = static_cast<T*>(j.bar_logits);
    a.target = j.target;
    a.logp = j.logp;
    a.lse = j.lse;
    a.bar_logp = j.bar_logp;
    a.bar_loss = j.bar_loss;
    a.old_logp = j.old_logp;
    a.ref_logp = j.ref_logp;
    a.advantage = j.advantage;
    a.weight = j.weight;
    a.rows = j.rows;
    a.vocab = j.vocab;
    a.row_stride = j.row_stride;
    a.bar_stride = j.bar_stride;
    a.scale = j.scale;
    a.low = 1.0f - j.clip_low;
    a.high = 1.0f + j.clip_high;
    a.kl = j.kl;
    a.even = j.rows > 0 ? 1.0f / static_cast<float>(j.rows) : 0.0f;
    a.target64 = j.target64;
    return a;
}

int launched(const char* what) {
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? HK_OK : hawk_internal::set_hip_error(what, err);
}

template <class T, Work W>
int rows_of(const RowArgs<T>& a, hipStream_t s) {
    if (a.rows == 0) return HK_OK;
    const dim3 grid(static_cast<unsigned>(a.rows)), block(kThreads);
    if constexpr (W == kGradient || W == kPolicyGradient) hipLaunchKernelGGL((hawk_row<T, W, true>), grid, block, 0, s, a);
    else if (W == kPolicy && a.bar_logits) hipLaunchKernelGGL((hawk_row<T, W, W == kPolicy>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((hawk_row<T, W, false>), grid, block, 0, s, a);
    return launched("hawk_row launch");
}

// Calls f with the logits' type.
template <class F>
int typed(int dtype, F&& f) {
    switch (dtype) {
        case HK_BF16: return f(bf16{});
        case HK_F16: return f(f16{});
        default: return f(float{});
    }
}

PairArgs pairs_of(const hk_row_loss_job& j) {
    PairArgs p{};
    p.offsets = j.offsets;
    p.target = j.target;
    p.logp = j.logp;
    p.ref_logp = j.ref_logp;
    p.weight = j.weight;
    p.bar_loss = j.bar_loss;
    p.margin = j.margin;
    p.rows = j.rows;
    p.pairs = j.pairs;
    p.beta = j.beta;
    p.smoothing = j.smoothing;
    p.even = j.pairs > 0 ? 1.0f / static_cast<float>(j.pairs) : 0.0f;
    p.offsets64 = j.offsets64;
    p.target64 = j.target64;
    return p;
}

int total(const float* x, int64_t count, float* out, hipStream_t s) {
    hipLaunchKernelGGL(hawk_row_total, dim3(1), dim3(kThreads), 0, s, x, count, out);
    return launched("hawk_row_total launch");
}

}  // namespace

extern "C" {

size_t hk_row_loss_scratch_bytes(const hk_row_loss_job* job) {
    if (!job || job->rows < 0 || job->pairs < 0) return 0;
    return sizeof(float) * static_cast<size_t>(job->rows + job->pairs + 1);
}

int hk_token_logp(const hk_row_loss_job* job, void* scratch, void* stream) {
    (void)scratch;
    const int rc = check_job(job, "hk_token_logp");
    if (rc != HK_OK) return rc;
    return typed(job->dtype, [&](auto t) {
        typedef decltype(t) T;
        return rows_of<T, kLogp>(args_of<T>(*job), static_cast<hipStream_t>(stream));
    });
}

int hk_token_logp_vjp(const hk_row_loss_job* job, void* scratch, void* stream) {
    (void)scratch;
    const int rc = check_job(job, "hk_token_logp_vjp");
    if (rc != HK_OK) return rc;
    if (job->rows > 0 && (!job->lse || !job->bar_logp || !job->bar_logits))
        return hawk_internal::set_error(HK_EVALUE, "hk_token_logp_vjp: lse, bar_logp and bar_logits are required");
    return typed(job->dtype, [&](auto t) {
        typedef decltype(t) T;
        return rows_of<T, kGradient>(args_of<T>(*job), static_cast<hipStream_t>(stream));
    });
}

static int check_policy(const hk_row_loss_job* j, const std::string& who) {
    const int rc = check_job(j, who);
    if (rc != HK_OK) return rc;
    if (j->rows > 0 && (!j->old_logp || !j->advantage || (j->kl != 0.0f && !j->ref_logp)))
        return hawk_internal::set_error(HK_EVALUE, who + ": old_logp and advantage (and ref_logp where kl is not 0) are required");
    return HK_OK;
}

int hk_policy_loss(const hk_row_loss_job* job, void* scratch, void* stream) {
    int rc = check_policy(job, "hk_policy_loss");
    if (rc != HK_OK) return rc;
    if (job->rows > 0 && job->loss && !scratch) return hawk_internal::set_error(HK_EVALUE, "hk_policy_loss: scratch is required");
    hipStream_t s = static_cast<hipStream_t>(stream);
    rc = typed(job->dtype, [&](auto t) {
        typedef decltype(t) T;
        RowArgs<T> a = args_of<T>(*job);
        a.row_loss = job->loss ? static_cast<float*>(scratch) : nullptr;
        return rows_of<T, kPolicy>(a, s);
    });
    if (rc != HK_OK || !job->loss) return rc;
    return total(static_cast<const float*>(scratch), job->rows, job->loss, s);
}

int hk_policy_loss_vjp(const hk_row_loss_job* job, void* scratch, void* stream) {
    (void)scratch;
    const int rc = check_policy(job, "hk_policy_loss_vjp");
    if (rc != HK_OK) return rc;
    if (job->rows > 0 && (!job->lse || !job->logp || !job->bar_logits))
        return hawk_internal::set_error(HK_EVALUE, "hk_policy_loss_vjp: logp, lse and bar_logits are required");
    return typed(job->dtype, [&](auto t) {
        typedef decltype(t) T;
        return rows_of<T, kPolicyGradient>(args_of<T>(*job), static_cast<hipStream_t>(stream));
    });
}

static int check_pairs(const hk_row_loss_job* j, const void* scratch, const std::string& who) {
    using hawk_internal::set_error;
    const int rc = check_job(j, who);
    if (rc != HK_OK) return rc;
    if (j->pairs > 0 && !j->offsets) return set_error(HK_EVALUE, who + ": offsets are required");
    if (j->pairs == 0 && j->rows > 0) return set_error(HK_EVALUE, who + ": rows without a pair");
    if ((j->rows > 0 || j->pairs > 0) && !scratch) return set_error(HK_EVALUE, who + ": scratch is required");
    return HK_OK;
}

int hk_preference_loss(const hk_row_loss_job* job, void* scratch, void* stream) {
    int rc = check_pairs(job, scratch, "hk_preference_loss");
    if (rc != HK_OK) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    float* pair_loss = static_cast<float*>(scratch);
    float* logp = job->logp ? job->logp : pair_loss + job->pairs;
    rc = typed(job->dtype, [&](auto t) {
        typedef decltype(t) T;
        RowArgs<T> a = args_of<T>(*job);
        a.logp = logp;
        return rows_of<T, kLogp>(a, s);
    });
    if (rc != HK_OK) return rc;
    if (job->pairs > 0) {
        PairArgs p = pairs_of(*job);
        p.logp = logp;
        p.pair_loss = pair_loss;
        hipLaunchKernelGGL(hawk_pair_loss, dim3(static_cast<unsigned>((job->pairs + kWaves - 1) / kWaves)),
                           dim3(kThreads), 0, s, p);
        rc = launched("hawk_pair_loss launch");
        if (rc != HK_OK) return rc;
    }
    return job->loss ? total(pair_loss, job->pairs, job->loss, s) : HK_OK;
}

int hk_preference_loss_vjp(const hk_row_loss_job* job, void* scratch, void* stream) {
    int rc = check_pairs(job, scratch, "hk_preference_loss_vjp");
    if (rc != HK_OK) return rc;
    if (job->rows == 0) return HK_OK;
    if (!job->lse || !job->margin || !job->bar_logits)
        return hawk_internal::set_error(HK_EVALUE, "hk_preference_loss_vjp: lse, margin and bar_logits are required");
    hipStream_t s = static_cast<hipStream_t>(stream);
    PairArgs p = pairs_of(*job);
    p.bar_logp = static_cast<float*>(scratch);
    hipLaunchKernelGGL(hawk_pair_slope, dim3(static_cast<unsigned>((job->pairs + kWaves - 1) / kWaves)), dim3(kThreads),
                       0, s, p);
    rc = launched("hawk_pair_slope launch");
    if (rc != HK_OK) return rc;
    return typed(job->dtype, [&](auto t) {
        typedef decltype(t) T;
        RowArgs<T> a = args_of<T>(*job);
        a.bar_logp = p.bar_logp;
        return rows_of<T, kGradient>(a, s);
    });
}

}  // extern "C"
