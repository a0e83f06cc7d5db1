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
#include <type_traits>

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

// A run of a row: its largest logit m and the sum s of 2^((x - m) k).  The
// difference comes before the product, so a row of the type's lowest value is a
// row of equal logits.  m = -inf with s = 0 where no logit is above -inf.
__device__ __forceinline__ float floor_of(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2, float k) {
    const float top = fmaxf(m, m2), base = floor_of(top);
    s = s * exp2_fast((m - base) * k) + s2 * exp2_fast((m2 - base) * k);
    m = top;
}

template <class T> constexpr int kVec = 16 / static_cast<int>(sizeof(T));

// Sixteen bytes of a row as words: what waits in registers stays packed.
typedef uint32_t Words __attribute__((ext_vector_type(4)));
template <class T> using Pack = Raw<T, kVec<T>>;
template <class T>
__device__ __forceinline__ float element(const Words& w, int j) {
    return widen<T, kVec<T>>(__builtin_bit_cast(Pack<T>, w), j);
}

// Vector v of a row, -inf past its end; an out row (nothing of it is read) is -inf throughout.
template <class T, bool Stream>
__device__ __forceinline__ Words row_vector(const T* row, int64_t v, int64_t vocab, bool out) {
    constexpr int V = kVec<T>;
    Words x = __builtin_bit_cast(Words, (splat<T, V>(static_cast<T>(-INFINITY))));
    if (!out) {
        if (v + V <= vocab) {
            x = __builtin_bit_cast(Words, (load_raw<T, V, Stream>(row + v)));
        } else if (v < vocab) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (v + j >= vocab) continue;
                if constexpr (sizeof(T) == 4) {
                    x[j] = __builtin_bit_cast(uint32_t, row[v + j]);
                } else {
                    const uint32_t bits = __builtin_bit_cast(uint16_t, row[v + j]);
                    x[j / 2] = j & 1 ? (x[j / 2] & 0xffffu) | bits << 16 : (x[j / 2] & 0xffff0000u) | bits;
                }
            }
        }
    }
    return x;
}
template <class T, bool Stream>
__device__ __forceinline__ void put_vector(T* row, int64_t v, int64_t vocab, const float (&x)[kVec<T>]) {
    constexpr int V = kVec<T>;
    if (v + V <= vocab) {
        store<T, V, Stream>(row + v, x);
    } else if (v < vocab) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (v + j < vocab) row[v + j] = static_cast<T>(x[j]);
    }
}

// (m, s) of L lanes' runs joined in every lane: a fixed tree within a wave, the
// waves in order.  `turn` alternates, so one barrier a row is enough.
template <int L>
__device__ __forceinline__ void join_lanes(float& m, float& s, float k, int turn) {
#pragma unroll
    for (int d = (L < 64 ? L : 64) / 2; d > 0; d >>= 1) {
        const float m2 = __shfl_xor(m, d), s2 = __shfl_xor(s, d);
        join(m, s, m2, s2, k);
    }
    if constexpr (L > 64) {
        constexpr int W = L / 64;
        __shared__ float lds[2][2][W];
        if ((threadIdx.x & 63) == 0) {
            lds[turn][0][threadIdx.x >> 6] = m;
            lds[turn][1][threadIdx.x >> 6] = s;
        }
        __syncthreads();
        const int w = threadIdx.x & (W - 1);
        m = lds[turn][0][w];
        s = lds[turn][1][w];
#pragma unroll
        for (int d = W / 2; d > 0; d >>= 1) {
            const float m2 = __shfl_xor(m, d), s2 = __shfl_xor(s, d);
            join(m, s, m2, s2, k);
        }
    }
}

// What a row's (m, s) and target give; lane 0 of the row writes it.
template <Work W, class T>
__device__ __forceinline__ void finish_row(const RowArgs<T>& a, int64_t n, bool out, bool writes, float top, float s,
                                           float at, float& logs, float& c) {
    logs = log2f(s);
    float logp = 0.0f, lse = 0.0f, loss = 0.0f;
    c = 0.0f;
    if (!out) {
        const float ln = logs * kLn2;
        lse = fused(top, a.scale, ln);
        logp = fused(at - top, a.scale, -ln);
        if constexpr (W == kPolicy) policy_row(a, n, logp, loss, c);
    }
    if (writes) {
        if (a.logp) a.logp[n] = logp;
        if (a.lse) a.lse[n] = lse;
        if (W == kPolicy && a.row_loss) a.row_loss[n] = loss;
    }
    c *= a.scale;
}

// A number that is one for the L lanes of a row, told to the compiler where they
// are whole waves: rows are then addressed by a scalar and a lane's offset.
template <int L>
__device__ __forceinline__ int one_of(int x) {
    if constexpr (L >= 64) return __builtin_amdgcn_readfirstlane(x);
    else return x;
}

// Rows held whole in the registers of L lanes, NV vectors a lane: one read of the
// logits for the loss and, where bar_logits is given, its gradient.  A workgroup
// goes from row to row, and a vector's register takes the next row's as soon as
// its gradient is stored, so loads run beside the second pass over the row.  The
// row has more than half the vectors (NV > 1), so the first half needs no bounds.
template <class T, int L, int NV, Work W, bool Grad, bool Stream>
__global__ void __launch_bounds__((L > kThreads ? L : kThreads)) hawk_row_held(const RowArgs<T> a) {
    constexpr int V = kVec<T>, R = (L > kThreads ? L : kThreads) / L;
    const int lane = threadIdx.x % L, sub = one_of<L>(threadIdx.x / L), mine = lane * V;
    const int vocab = static_cast<int>(a.vocab);
    const float k = a.scale * kLog2e;
    const int64_t step = static_cast<int64_t>(gridDim.x) * R;
    int64_t n = static_cast<int64_t>(blockIdx.x) * R + sub;
    // -1: nothing of the row is read; vocab: a target past the vocabulary
    auto target = [&](int64_t row) -> int {
        if (row >= a.rows) return -1;
        const int64_t y = target_of(a.target, a.target64, row);
        return one_of<L>(y < 0 ? -1 : y < vocab ? static_cast<int>(y) : vocab);
    };
    // A row that is left out is not read: its lanes go on with what they hold, and
    // nothing of it is used.
    auto fetch = [&](Words& x, const T* row, int i) {
        const int rest = vocab - i * L * V;     // what the row has from the lanes' first vector on
        if (i < NV / 2) {
            x = __builtin_bit_cast(Words, (load_raw<T, V, Stream>(row + i * L * V + static_cast<unsigned>(mine))));
        } else {
            x = __builtin_bit_cast(Words, (splat<T, V>(static_cast<T>(-INFINITY))));
            if (mine + V <= rest) x = __builtin_bit_cast(Words, (load_raw<T, V, Stream>(row + i * L * V + static_cast<unsigned>(mine))));
            else if (mine < rest) x = row_vector<T, Stream>(row + i * L * V, mine, rest, false);
        }
    };
    int y = target(n);
    Words x[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        x[i] = Words{0, 0, 0, 0};
        if (y >= 0) fetch(x[i], a.logits + n * a.row_stride, i);
    }
    int turn = 0;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * R; base < a.rows; base += step, turn ^= 1) {
        const bool real = n < a.rows, out = y < 0;
        float at = out ? 0.0f : y < vocab ? static_cast<float>(a.logits[n * a.row_stride + y]) : NAN;
        const int64_t next = n + step;
        const int next_y = target(next);
        float m = -INFINITY, s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) m = fmaxf(m, element<T>(x[i], j));
        const float own = floor_of(m);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            forget(x[i]);
#pragma unroll
            for (int j = 0; j < V; ++j) s += exp2_fast((element<T>(x[i], j) - own) * k);
            asm volatile("" : "+v"(s));
        }
        // read before any lane may store the gradient over it
        asm volatile("" : "+v"(at));
        join_lanes<L>(m, s, k, turn);
        const float top = floor_of(m);
        float logs, c;
        finish_row<W>(a, n, out, real && lane == 0, top, s, at, logs, c);
        const T* ahead = a.logits + next * a.row_stride;
        if constexpr (Grad) {
            T* bar = a.bar_logits + n * a.bar_stride;
            const bool zero = out || c == 0.0f;
            if (real) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int rest = vocab - i * L * V, hit = y - mine - i * L * V;
                    float g[V];
                    forget(x[i]);
#pragma unroll
                    for (int j = 0; j < V; ++j) g[j] = -c * exp2_fast(fused(element<T>(x[i], j) - top, k, -logs));
                    if (hit >= 0 && hit < V) {
#pragma unroll
                        for (int j = 0; j < V; ++j) g[j] = j == hit ? c + g[j] : g[j];
                    }
                    if (zero) {
#pragma unroll
                        for (int j = 0; j < V; ++j) g[j] = 0.0f;
                    }
                    if (i < NV / 2 || mine + V <= rest) store<T, V, Stream>(bar + i * L * V + static_cast<unsigned>(mine), g);
                    else put_vector<T, Stream>(bar + i * L * V, mine, rest, g);
                    if (next_y >= 0) fetch(x[i], ahead, i);
                    asm volatile("" ::: "memory");     // a vector is stored before the next one is widened
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (next_y >= 0) fetch(x[i], ahead, i);
        }
        n = next;
        y = next_y;
    }
}

// Rows of any length, a workgroup of L lanes each, kAhead vectors a lane at a
// time: the log-sum-exp as a running (m, s), then, for the gradient, the row
// once more.
constexpr int kAhead = 4;
template <class T, int L, Work W, bool Stream>
__global__ void __launch_bounds__(L) hawk_row_long(const RowArgs<T> a) {
    constexpr int V = kVec<T>;
    const int64_t n = blockIdx.x;
    const int lane = threadIdx.x;
    const float k = a.scale * kLog2e;
    const T* row = a.logits + n * a.row_stride;
    const int64_t y = target_of(a.target, a.target64, n);
    const bool out = y < 0;
    float at = out ? 0.0f : y < a.vocab ? static_cast<float>(row[y]) : NAN;
    float m = -INFINITY, s = 0.0f;
    if (!out) {
        for (int64_t v0 = static_cast<int64_t>(lane) * V; v0 < a.vocab; v0 += kAhead * L * V) {
            Words x[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) x[i] = row_vector<T, Stream>(row, v0 + i * L * V, a.vocab, false);
            float top = m;
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) top = fmaxf(top, element<T>(x[i], j));
            const float base = floor_of(top);
            s *= exp2_fast((m - base) * k);
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) s += exp2_fast((element<T>(x[i], j) - base) * k);
            m = top;
        }
    }
    asm volatile("" : "+v"(at));
    join_lanes<L>(m, s, k, 0);
    const float top = floor_of(m);
    float logs, c;
    finish_row<W>(a, n, out, lane == 0, top, s, at, logs, c);
    if (W != kPolicy || !a.bar_logits) return;
    T* bar = a.bar_logits + n * a.bar_stride;
    const bool zero = out || c == 0.0f;
    for (int64_t v = static_cast<int64_t>(lane) * V; v < a.vocab; v += L * V) {
        const Words x = row_vector<T, Stream>(row, v, a.vocab, zero);
        float g[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float p = exp2_fast(fused(element<T>(x, j) - top, k, -logs));
            g[j] = zero ? 0.0f : v + j == y ? c - c * p : -c * p;
        }
        put_vector<T, Stream>(bar, v, a.vocab, g);
    }
}

// The gradient from a saved lse: L lanes a row, kAhead vectors a lane at a time.
template <class T, int L, Work W, bool Stream>
__global__ void __launch_bounds__((L > kThreads ? L : kThreads)) hawk_row_gradient(const RowArgs<T> a) {
    constexpr int V = kVec<T>, R = (L > kThreads ? L : kThreads) / L;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * R + threadIdx.x / L;
    const int lane = threadIdx.x % L;
    if (n >= a.rows) return;
    const int64_t y = target_of(a.target, a.target64, n);
    const T* row = a.logits + n * a.row_stride;
    T* bar = a.bar_logits + n * a.bar_stride;
    float c = 0.0f, lse = 0.0f;
    if (y >= 0) {
        lse = a.lse[n];
        if constexpr (W == kGradient) {
            c = a.bar_logp[n];
        } else {
            float loss;
            policy_row(a, n, a.logp[n], loss, c);
        }
        c = (y < a.vocab ? c : NAN) * a.scale;
    }
    const bool zero = c == 0.0f;
    for (int64_t v0 = static_cast<int64_t>(lane) * V; v0 < a.vocab; v0 += kAhead * L * V) {
        Words x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) x[i] = row_vector<T, Stream>(row, v0 + i * L * V, a.vocab, zero);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t v = v0 + i * L * V;
            float g[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                // l - lse is rounded once, from the saved lse, before it is taken to base 2
                const float p = exp2_fast(fused(element<T>(x[i], j), a.scale, -lse) * kLog2e);
                g[j] = zero ? 0.0f : -c * p;
            }
            if (y >= v && y < v + V) {
#pragma unroll
                for (int j = 0; j < V; ++j) g[j] = v + j == y ? c + g[j] : g[j];
            }
            put_vector<T, Stream>(bar, v, a.vocab, g);
        }
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

// Rows that begin and end with 128-byte lines are passed as a stream.
template <class T>
bool whole_lines(const RowArgs<T>& a) {
    auto whole = [&](const T* p, int64_t stride) {
        return !p || (reinterpret_cast<uintptr_t>(p) % 128 == 0 && (stride * static_cast<int64_t>(sizeof(T))) % 128 == 0);
    };
    return whole(a.logits, a.row_stride) && whole(a.bar_logits, a.bar_stride);
}

constexpr int64_t kUnits = 256;  // compute units

template <class T, int L, int NV, Work W, bool Grad, bool Stream>
void launch_held(const RowArgs<T>& a, hipStream_t s) {
    constexpr int threads = L > kThreads ? L : kThreads, R = threads / L;
    const int64_t blocks = (a.rows + R - 1) / R;
    // as many workgroups as the card holds at once, each taking row after row
    const int64_t most = kUnits * (L > kThreads ? 1 : NV >= 16 ? 4 : 8);
    hipLaunchKernelGGL((hawk_row_held<T, L, NV, W, Grad, Stream>), dim3(static_cast<unsigned>(blocks < most ? blocks : most)),
                       dim3(threads), 0, s, a);
}

template <class T, Work W>
int rows_of(const RowArgs<T>& a, hipStream_t s) {
    if (a.rows == 0) return HK_OK;
    const int64_t vectors = (a.vocab + kVec<T> - 1) / kVec<T>;
    const bool stream = whole_lines(a), few = a.rows < 2 * kUnits;
    if constexpr (W == kGradient || W == kPolicyGradient) {
        auto go = [&](auto lanes) {
            constexpr int L = decltype(lanes)::value, R = (L > kThreads ? L : kThreads) / L;
            const dim3 grid(static_cast<unsigned>((a.rows + R - 1) / R)), block(R * L);
            if (stream) hipLaunchKernelGGL((hawk_row_gradient<T, L, W, true>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((hawk_row_gradient<T, L, W, false>), grid, block, 0, s, a);
        };
        if (vectors <= 32) go(std::integral_constant<int, 16>{});
        else if (vectors <= 256) go(std::integral_constant<int, 64>{});
        else if (few && vectors > 4096) go(std::integral_constant<int, 1024>{});
        else go(std::integral_constant<int, 256>{});
    } else {
        const bool hold = W == kPolicy && a.bar_logits;
        auto held = [&](auto lanes, auto count) {
            constexpr int L = decltype(lanes)::value, NV = decltype(count)::value;
            if constexpr (L >= 256) {         // taken for the gradient alone
                if (stream) launch_held<T, L, NV, W, W == kPolicy, true>(a, s);
                else launch_held<T, L, NV, W, W == kPolicy, false>(a, s);
            } else {
                if (hold) launch_held<T, L, NV, W, W == kPolicy, false>(a, s);
                else launch_held<T, L, NV, W, false, false>(a, s);
            }
        };
        std::integral_constant<int, 16> l16;
        std::integral_constant<int, 64> l64;
        std::integral_constant<int, 256> l256;
        std::integral_constant<int, 1024> l1024;
        std::integral_constant<int, 1> n1;
        std::integral_constant<int, 2> n2;
        std::integral_constant<int, 4> n4;
        std::integral_constant<int, 8> n8;
        std::integral_constant<int, 16> n16;
        if (vectors <= 16) held(l16, n1);
        else if (vectors <= 32) held(l16, n2);
        else if (vectors <= 64) held(l16, n4);
        else if (vectors <= 128) held(l64, n2);
        else if (vectors <= 256) held(l64, n4);
        else if (vectors <= 512) held(l64, n8);
        else if (W == kPolicy && hold && vectors <= 16384) {
            if constexpr (W == kPolicy) {
                if (vectors <= 1024) held(l256, n4);
                else if (vectors <= 2048) held(l256, n8);
                else if (vectors <= 4096 && few) held(l1024, n4);
                else if (vectors <= 4096) held(l256, n16);
                else if (vectors <= 8192) held(l1024, n8);
                else held(l1024, n16);
            }
        } else {
            const dim3 grid(static_cast<unsigned>(a.rows));
            const bool big = few || (W == kPolicy && a.bar_logits);
            if (big && stream) hipLaunchKernelGGL((hawk_row_long<T, 1024, W, true>), grid, dim3(1024), 0, s, a);
            else if (big) hipLaunchKernelGGL((hawk_row_long<T, 1024, W, false>), grid, dim3(1024), 0, s, a);
            else if (stream) hipLaunchKernelGGL((hawk_row_long<T, 256, W, true>), grid, dim3(256), 0, s, a);
            else hipLaunchKernelGGL((hawk_row_long<T, 256, W, false>), grid, dim3(256), 0, s, a);
        }
    }
    return launched("row kernel launch");
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
