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
// Where a row does not fit the registers, (m, sum) run along in one pass and are
// rescaled as m grows: the published online softmax (Milakov and Gimelshein, Online
// normalizer calculation for softmax, 2018).

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
constexpr int64_t kUnits = 256;            // compute units
constexpr int64_t kWords = 4 * kUnits;     // parts of all rows that are split
constexpr int64_t kSplitRows = kUnits / 4; // those rows at most
static_assert(kWords * 8 + kSplitRows * 4 == HK_ROW_LOSS_STATE_BYTES, "a word a part, a counter a row");

struct PairArgs {
    const void *offsets, *target;
    const double* logp;       // before it is rounded
    const float *ref_logp, *weight, *bar_loss;
    float *margin, *pair_loss;
    int64_t rows, pairs;
    float beta, smoothing, even;
    int offsets64, target64;
};

__device__ __forceinline__ int64_t cut_of(const PairArgs& a, int64_t k) {
    const int64_t v = a.offsets64 ? static_cast<const int64_t*>(a.offsets)[k] : static_cast<const int32_t*>(a.offsets)[k];
    return v < 0 ? 0 : v > a.rows ? a.rows : v;
}

template <class T>
struct RowArgs {
    const T* logits;
    T* bar_logits;
    const void* target;
    float *logp, *lse;
    float* row_loss;          // each row's weighted loss, or NULL
    float* loss;              // their sum, taken by the last workgroup, or NULL
    double* wide;             // logp before it is rounded to 32 bits, or NULL
    uint32_t* counter;        // workgroups done, a word a row (the sum: the first word)
    uint64_t* run;            // the (m, s) of a row's parts, or NULL
    const float* bar_logp;    // the gradient's c (before scale), or NULL
    const float *bar_loss, *old_logp, *ref_logp, *advantage, *weight;
    int64_t rows, vocab, row_stride, bar_stride;
    float scale, low, high, kl, even;   // low, high: the ratio's bounds; even: the weight where weight is NULL
    int64_t each;             // vectors of a row that a workgroup takes, where rows are split
    int64_t first;            // the launch's first row
    int target64;
    PairArgs pairs;           // the preference loss's gradient
};

enum Work { kLogp, kPolicy, kGradient, kPolicyGradient, kPairGradient };

// exp2 that flushes results below 2^-126 to 0, and a log2 to 1 ulp: the
// hardware's own.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ int64_t target_of(const void* target, int wide, int64_t n) {
    return wide ? static_cast<const int64_t*>(target)[n] : static_cast<const int32_t*>(target)[n];
}

// What a row's loss reads beside its logits, asked for before they are reduced.
struct PolicyRow {
    float w, A, old, ref;
};
template <class T>
__device__ __forceinline__ PolicyRow policy_planes(const RowArgs<T>& a, int64_t n, bool read) {
    PolicyRow r{0.0f, 0.0f, 0.0f, 0.0f};
    if (read) {
        r.w = a.weight ? a.weight[n] : a.even;
        r.A = a.advantage[n];
        r.old = a.old_logp[n];
        if (a.kl != 0.0f) r.ref = a.ref_logp[n];
    }
    return r;
}

// The row's loss by its log-probability (times its weight) and the loss's
// derivative by it (times weight and bar_loss).  A weight of 0 gives 0.
template <class T>
__device__ __forceinline__ void policy_row(const RowArgs<T>& a, const PolicyRow& p, float logp, float& loss, float& slope) {
    loss = slope = 0.0f;
    if (p.w == 0.0f) return;
    const float r = expf(logp - p.old);
    const float plain = r * p.A, clipped = fminf(fmaxf(r, a.low), a.high) * p.A;
    // a NaN is the minimum (a NaN ratio or advantage, or an infinite one times 0):
    // fminf, fmaxf and the comparison would drop it
    if (!(plain == plain)) { loss = slope = plain; return; }
    loss = plain <= clipped ? -plain : -clipped;
    slope = plain <= clipped ? -plain : 0.0f;
    if (a.kl != 0.0f) {
        // e^d - 1 is an infinity before d is: a target without probability has both
        const float d = p.ref - logp, grown = expm1f(d);
        loss += a.kl * (grown == INFINITY ? grown : grown - d);
        slope -= a.kl * grown;
    }
    loss *= p.w;
    slope *= a.bar_loss ? p.w * *a.bar_loss : p.w;
}

// A run of a row: its largest logit m and the sum s of 2^((x - m) k).  The
// difference comes before the product, so a row of the type's lowest value is a
// row of equal logits.  m = -inf with s = 0 where no logit is above -inf, and
// m = s = inf where one is +inf.  What is subtracted is always a number, so that
// inf - inf comes up only for a target that is +inf itself.
constexpr float kLargest = 3.40282347e+38f;
__device__ __forceinline__ float floor_of(float m) { return m == -INFINITY ? 0.0f : fminf(m, kLargest); }
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

// A row is passed in vectors that start at 16-byte addresses, wherever the row
// itself starts: position p of it is element p - lead, and what lies before the
// row or past its end is -inf and neither read nor written.  (Vectors at the
// row's own address, 2 bytes off: 4096 rows of 50001 bfloat16 logits 87 us.)
template <class T>
__device__ __forceinline__ int lead_of(const T* row) {
    return static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
}
// The vector at position p of [low, high): from (the row's address less its lead).
template <class T, bool Stream>
__device__ __forceinline__ Words row_vector(const T* from, int64_t p, int low, int64_t high) {
    constexpr int V = kVec<T>;
    if (p >= low && p + V <= high) return __builtin_bit_cast(Words, (load_raw<T, V, Stream>(from + p)));
    Words x = __builtin_bit_cast(Words, (splat<T, V>(static_cast<T>(-INFINITY))));
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (p + j < low || p + j >= high) continue;
        if constexpr (sizeof(T) == 4) {
            x[j] = __builtin_bit_cast(uint32_t, from[p + j]);
        } else {
            const uint32_t bits = __builtin_bit_cast(uint16_t, from[p + j]);
            x[j / 2] = j & 1 ? (x[j / 2] & 0xffffu) | bits << 16 : (x[j / 2] & 0xffff0000u) | bits;
        }
    }
    return x;
}
template <class T, bool Stream>
__device__ __forceinline__ void put_vector(T* to, int64_t p, int low, int64_t high, const float (&x)[kVec<T>]) {
    constexpr int V = kVec<T>;
    if (p >= low && p + V <= high) {
        store<T, V, Stream>(to + p, x);
        return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (p + j >= low && p + j < high) to[p + j] = static_cast<T>(x[j]);
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
__device__ __forceinline__ void finish_row(const RowArgs<T>& a, const PolicyRow& planes, int64_t n, bool out, bool writes, float top, float s,
                                           float at, float& logs, float& c) {
    logs = log2f(s);
    float logp = 0.0f, lse = 0.0f, loss = 0.0f;
    c = 0.0f;
    if (!out) {
        const float ln = logs * kLn2;
        lse = fused(top, a.scale, ln);
        logp = fused(at - top, a.scale, -ln);
        if constexpr (W == kPolicy) policy_row(a, planes, logp, loss, c);
    }
    if (writes) {
        if (a.logp) a.logp[n] = logp;
        if (a.lse) a.lse[n] = lse;
        if (W == kPolicy && a.row_loss) a.row_loss[n] = loss;
        // A margin is a small difference of sums of these: rounding each to 32 bits
        // (5e-7 of a logp of -10) would be most of its error.
        if (W == kLogp && a.wide)
            a.wide[n] = out ? 0.0 : (static_cast<double>(at) - top) * a.scale - log(static_cast<double>(s));
    }
    c *= a.scale;
}

// The sum of rows' losses in 64 bits, each run of kRun numbers by one workgroup in a
// fixed order.  All of a lane's loads are out at once (one after another, 65536
// rows took 80 us).
constexpr int kTotalThreads = 1024, kEach = 8, kRun = kTotalThreads * kEach;
template <int Threads, class In>
__device__ __forceinline__ double sum_run(const In* x, int64_t count) {
    constexpr int each = kRun / Threads;
    __shared__ double lds[Threads / 64];
    double t = 0.0;
#pragma unroll 1
    for (int i0 = 0; i0 < each; i0 += kEach) {
        In v[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int64_t at = threadIdx.x + static_cast<int64_t>(i0 + i) * Threads;
            v[i] = at < count ? x[at] : In(0);
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) t += static_cast<double>(v[i]);
        if ((i0 + kEach) * static_cast<int64_t>(Threads) >= count) break;
    }
    for (int d = 32; d > 0; d >>= 1) t += __shfl_xor(t, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = t;
    __syncthreads();
    t = 0.0;
    for (int w = 0; w < Threads / 64; ++w) t += lds[w];
    return t;
}
template <class In, class Out>
__global__ void __launch_bounds__(kTotalThreads) hawk_row_total(const In* x, int64_t count, Out* out) {
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kRun;
    const double t = sum_run<kTotalThreads>(x + first, count - first < kRun ? count - first : kRun);
    if (threadIdx.x == 0) out[blockIdx.x] = static_cast<Out>(t);
}

// A number that is one for the L lanes of a row, told to the compiler where they
// are whole waves: rows are then addressed by a scalar and a lane's offset.
template <int L>
__device__ __forceinline__ int one_of(int x) {
    if constexpr (L >= 64) return __builtin_amdgcn_readfirstlane(x);
    else return x;
}

// Rows held whole in the registers of L lanes, NV vectors a lane: one read of the
// logits for the loss and, where asked, its gradient.  A workgroup goes from row
// to row, and a vector's register takes the next row's as soon as its gradient is
// stored, so loads run beside the second pass over the row.  The row has no fewer
// than half the vectors (NV > 1), so those before the half's last need no bounds.
// Rows of whole waves pass as a stream (with their gradient, 512 rows of 131072
// bfloat16 logits 58 us, 63 cached; 8192 of them 828 and 832).
template <class T, int L, int NV, Work W, bool Grad>
__global__ void __launch_bounds__((L > kThreads ? L : kThreads)) hawk_row_held(const RowArgs<T> a) {
    constexpr int V = kVec<T>, R = (L > kThreads ? L : kThreads) / L;
    constexpr bool Stream = L >= 256;
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
        const int lead = lead_of(row), rest = lead + vocab - i * L * V;   // the positions from lane 0's vector on
        const T* from = row - lead + i * L * V;
        if (i > 0 && i < NV / 2 - 1) x = __builtin_bit_cast(Words, (load_raw<T, V, Stream>(from + static_cast<unsigned>(mine))));
        else x = row_vector<T, Stream>(from, mine, i == 0 ? lead : 0, rest);
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
        const T* row = a.logits + n * a.row_stride;
        float at = out ? 0.0f : y < vocab ? static_cast<float>(row[y]) : NAN;
        const PolicyRow planes = policy_planes(a, n, W == kPolicy && !out);
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
        finish_row<W>(a, planes, n, out, real && lane == 0, top, s, at, logs, c);
        const T* ahead = a.logits + next * a.row_stride;
        if constexpr (Grad) {
            const int lead = lead_of(row);
            T* bar = a.bar_logits + n * a.bar_stride - lead;
            const bool zero = out || c == 0.0f;
            if (real) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int hit = lead + y - mine - i * L * V;
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
                    if (i > 0 && i < NV / 2 - 1) store<T, V, Stream>(bar + i * L * V + static_cast<unsigned>(mine), g);
                    else put_vector<T, Stream>(bar + i * L * V, mine, i == 0 ? lead : 0, lead + vocab - i * L * V, g);
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
    if constexpr (W == kPolicy && L < 256) {
        // few rows: the workgroup that is done last sums them all, instead of a
        // launch of its own
        if (a.loss) {
            __shared__ int last;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) last = atomicAdd(a.counter, 1u) == gridDim.x - 1;
            __syncthreads();
            if (!last) return;
            __threadfence();
            const double t = sum_run<kThreads>(a.row_loss, a.rows);
            if (threadIdx.x == 0) {
                *a.loss = static_cast<float>(t);
                *a.counter = 0;
            }
        }
    }
}

// A lane's running (m, s) over positions first, first + L*V .. below end of a row
// that starts at low, kAhead vectors at a time.
constexpr int kAhead = 4;
template <class T, int L>
__device__ __forceinline__ void run_of(const T* from, int64_t first, int low, int64_t end, float k, float& m, float& s) {
    constexpr int V = kVec<T>;
    for (int64_t p = first; p < end; p += kAhead * L * V) {
        Words x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) x[i] = row_vector<T, true>(from, p + i * L * V, low, end);
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

// Few long rows: `parts` workgroups a row, a.each vectors a part.  A part leaves
// its (m, s) in a word and counts itself; the last one counted joins the words in
// their order and finishes the row.  A word is 0 until its part has come (no pair
// is: s is 1 or more, a NaN, or 0 beside m = -inf), so nothing but the word itself
// orders it: with a release and an acquire at each part's count, whose fences
// write back and drop the caches, 64 rows of 262144 bfloat16 logits take 33 us
// instead of 13.  The word waited for was sent before its part counted itself; if it
// never shows (the state's words shared by two streams) the row is a NaN.
constexpr int kMostParts = 64, kLooks = 1 << 20;
template <class T, Work W>
__global__ void __launch_bounds__(kThreads) hawk_row_parts(const RowArgs<T> a, int parts) {
    constexpr int V = kVec<T>;
    const int64_t n = blockIdx.x / parts;
    const int part = static_cast<int>(blockIdx.x % parts), lane = threadIdx.x;
    const float k = a.scale * kLog2e;
    const int64_t y = target_of(a.target, a.target64, n);
    const bool out = y < 0;
    if (out && part > 0) return;
    const T* row = a.logits + n * a.row_stride;
    float at = out ? 0.0f : y < a.vocab ? static_cast<float>(row[y]) : NAN;
    const PolicyRow planes = policy_planes(a, n, W == kPolicy && !out);
    float m = -INFINITY, s = 0.0f;
    if (!out) {
        const int lead = lead_of(row);
        const int64_t high = lead + a.vocab, end = (part + 1) * a.each * V;
        run_of<T, kThreads>(row - lead, (part * a.each + lane) * V, lead, end < high ? end : high, k, m, s);
        asm volatile("" : "+v"(at));
        join_lanes<kThreads>(m, s, k, 0);
        if (lane >= 64) return;
        uint64_t* word = a.run + n * parts;
        int done = 0;
        if (lane == 0) {
            const uint64_t pair = static_cast<uint64_t>(__builtin_bit_cast(uint32_t, m)) << 32 | __builtin_bit_cast(uint32_t, s);
            __hip_atomic_store(word + part, pair, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            done = __hip_atomic_fetch_add(a.counter + n, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1u;
        }
        if (!__builtin_amdgcn_readfirstlane(done)) return;
        m = -INFINITY, s = 0.0f;
        if (lane < parts) {
            uint64_t pair = 0;
            for (int i = 0; pair == 0 && i < kLooks; ++i) pair = __hip_atomic_load(word + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            word[lane] = 0;
            m = __builtin_bit_cast(float, static_cast<uint32_t>(pair >> 32));
            s = pair == 0 ? NAN : __builtin_bit_cast(float, static_cast<uint32_t>(pair));
        }
        if (lane == 0) a.counter[n] = 0;
        join_lanes<64>(m, s, k, 0);
    }
    float logs, c;
    finish_row<W>(a, planes, n, out, lane == 0, floor_of(m), s, at, logs, c);
}

// Rows of any length, a workgroup of L lanes each.
template <class T, int L, Work W>
__global__ void __launch_bounds__(L) hawk_row_long(const RowArgs<T> a) {
    constexpr int V = kVec<T>;
    const int64_t n = a.first + blockIdx.x;
    const int lane = threadIdx.x;
    const float k = a.scale * kLog2e;
    const T* row = a.logits + n * a.row_stride;
    const int lead = lead_of(row);
    const int64_t y = target_of(a.target, a.target64, n);
    const bool out = y < 0;
    float at = out ? 0.0f : y < a.vocab ? static_cast<float>(row[y]) : NAN;
    const PolicyRow planes = policy_planes(a, n, W == kPolicy && !out);
    float m = -INFINITY, s = 0.0f;
    if (!out) run_of<T, L>(row - lead, static_cast<int64_t>(lane) * V, lead, lead + a.vocab, k, m, s);
    asm volatile("" : "+v"(at));
    join_lanes<L>(m, s, k, 0);
    const float top = floor_of(m);
    float logs, c;
    finish_row<W>(a, planes, n, out, lane == 0, top, s, at, logs, c);
}

// The derivative of the preference loss by a row's log-probability (times weight
// and bar_loss): its sequence is the last that starts at or before it.
__device__ __forceinline__ float pair_slope(const PairArgs& a, int64_t n) {
    int64_t low = 0, high = 2 * a.pairs - 1;
    while (low < high) {
        const int64_t mid = (low + high + 1) >> 1;
        if (cut_of(a, mid) <= n) low = mid;
        else high = mid - 1;
    }
    if (n < cut_of(a, low) || n >= cut_of(a, low + 1)) return 0.0f;      // a row that no sequence holds
    const int64_t p = low >> 1;
    const float w = a.weight ? a.weight[p] : a.even;
    if (w == 0.0f) return 0.0f;
    float up, down;
    sigmoid(a.beta * a.margin[p], up, down);
    float slope = a.beta * w * (a.smoothing * up - (1.0f - a.smoothing) * down);
    if (a.bar_loss) slope *= *a.bar_loss;
    return low & 1 ? -slope : slope;
}

// The gradient from a saved lse: L lanes a row, kAhead vectors a lane at a time.
template <class T, int L, Work W>
__global__ void __launch_bounds__((L > kThreads ? L : kThreads)) hawk_row_gradient(const RowArgs<T> a) {
    constexpr int V = kVec<T>, R = kThreads / L;
    constexpr bool Stream = L >= 256;
    const int64_t n = a.first + static_cast<int64_t>(blockIdx.x) * R + threadIdx.x / L;
    const int lane = threadIdx.x % L;
    if (n >= a.rows) return;
    const int64_t y = target_of(a.target, a.target64, n);
    const T* row = a.logits + n * a.row_stride;
    const int lead = lead_of(row);
    const int64_t last = lead + a.vocab, at_y = y < 0 ? -1 : lead + y;
    int64_t high = last, first = static_cast<int64_t>(lane) * V;
    if constexpr (L >= kThreads) {
        const int64_t part = blockIdx.y * a.each * V, end = part + a.each * V;
        first += part;
        high = end < last ? end : last;
    }
    T* bar = a.bar_logits + n * a.bar_stride - lead;
    float c = 0.0f, lse = 0.0f;
    if (y >= 0) {
        lse = a.lse[n];
        if constexpr (W == kGradient) {
            c = a.bar_logp[n];
        } else if constexpr (W == kPairGradient) {
            c = pair_slope(a.pairs, n);
        } else {
            float loss;
            policy_row(a, policy_planes(a, n, true), a.logp[n], loss, c);
        }
        // past the vocabulary, unless its weight leaves the row out
        if (y >= a.vocab && (W == kGradient || c != 0.0f)) c = NAN;
        c *= a.scale;
    }
    // A row without a gradient is not read, unless to know it takes longer than to
    // ask for the row's first vectors (a search for its pair).
    const bool zero = c == 0.0f, unread = W == kPairGradient ? y < 0 : zero;
    for (int64_t p0 = first; p0 < high; p0 += kAhead * L * V) {
        Words x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) x[i] = row_vector<T, Stream>(row - lead, p0 + i * L * V, lead, unread ? 0 : high);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t p = p0 + i * L * V;
            float g[V];
            forget(x[i]);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                // l - lse is rounded once, from the saved lse, before it is taken to base 2
                const float e = exp2_fast(fused(element<T>(x[i], j), a.scale, -lse) * kLog2e);
                g[j] = zero ? 0.0f : -c * e;
            }
            if (at_y >= p && at_y < p + V) {
#pragma unroll
                for (int j = 0; j < V; ++j) g[j] = p + j == at_y ? c + g[j] : g[j];
            }
            put_vector<T, Stream>(bar, p, lead, high, g);
            asm volatile("" ::: "memory");         // a vector is stored before the next one is widened
        }
    }
}

// One wave a pair: both sequences' log ratios summed in 64 bits, then the loss.
// A single workgroup takes all pairs and sums their losses too (Whole).
constexpr int kPairThreads = 1024, kPairWaves = kPairThreads / 64, kPairs = 128;
template <bool Whole>
__global__ void __launch_bounds__(kPairThreads) hawk_pair_loss(const PairArgs a, float* total) {
    const int lane = threadIdx.x & 63;
    double sum = 0.0;
    for (int64_t p = static_cast<int64_t>(blockIdx.x) * kPairWaves + (threadIdx.x >> 6); p < a.pairs;
         p += static_cast<int64_t>(gridDim.x) * kPairWaves) {
        const int64_t c0 = cut_of(a, 2 * p), c1 = cut_of(a, 2 * p + 1), c2 = cut_of(a, 2 * p + 2);
        double t = 0.0;
        for (int64_t n0 = c0 + lane; n0 < c2; n0 += 4 * 64) {
            double lp[4];
            float ref[4];
            int64_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t n = n0 + 64 * i;
                y[i] = n < c2 ? target_of(a.target, a.target64, n) : -1;
                lp[i] = n < c2 ? a.logp[n] : 0.0;
                ref[i] = n < c2 && a.ref_logp ? a.ref_logp[n] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const double r = lp[i] - static_cast<double>(ref[i]);
                if (y[i] >= 0) t += n0 + 64 * i < c1 ? r : -r;
            }
        }
        for (int d = 32; d > 0; d >>= 1) t += __shfl_xor(t, d);
        const float w = a.weight ? a.weight[p] : a.even;
        const double z = static_cast<double>(a.beta) * t;
        // -log sigma(z) and -log sigma(-z) = z - log sigma(z), neither overflowing
        const double soft = log1p(exp(-fabs(z)));
        const double lose = soft + (z < 0.0 ? -z : 0.0), win = soft + (z > 0.0 ? z : 0.0);
        // a side of weight 0 costs nothing, be it infinite
        const double one = a.smoothing < 1.0f ? (1.0 - a.smoothing) * lose : 0.0, other = a.smoothing > 0.0f ? a.smoothing * win : 0.0;
        const double loss = (z == z) ? one + other : z;
        const float weighted = w == 0.0f ? 0.0f : static_cast<float>(w * loss);
        sum += static_cast<double>(weighted);
        if (lane == 0) {
            if (a.margin) a.margin[p] = static_cast<float>(t);
            if (!Whole && a.pair_loss) a.pair_loss[p] = weighted;
        }
    }
    if constexpr (Whole) {
        __shared__ double lds[kPairWaves];
        if (lane == 0) lds[threadIdx.x >> 6] = sum;
        __syncthreads();
        if (threadIdx.x != 0 || !total) return;
        sum = 0.0;
        for (int w = 0; w < kPairWaves; ++w) sum += lds[w];
        *total = static_cast<float>(sum);
    }
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
    a.run = static_cast<uint64_t*>(j.state);
    a.counter = j.state ? reinterpret_cast<uint32_t*>(a.run + kWords) : nullptr;
    return a;
}

int launched(const char* what) {
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? HK_OK : hawk_internal::set_hip_error(what, err);
}

template <class T, int L, int NV, Work W, bool Grad>
void launch_held(const RowArgs<T>& a, hipStream_t s) {
    constexpr int threads = L > kThreads ? L : kThreads, R = threads / L;
    const int64_t blocks = (a.rows + R - 1) / R;
    // as many workgroups as the card holds at once, each taking row after row
    const int64_t most = kUnits * (L == 1024 ? 1 : L == 512 ? 2 : NV >= 16 ? 4 : NV >= 8 ? 6 : 8);
    hipLaunchKernelGGL((hawk_row_held<T, L, NV, W, Grad>), dim3(static_cast<unsigned>(blocks < most ? blocks : most)),
                       dim3(threads), 0, s, a);
}

template <int N> using Count = std::integral_constant<int, N>;

// A launch has fewer than 2^32 threads along an axis of its grid.  Rows of a
// workgroup each, or R to one, go in launches of at most that many: calls
// launch(blocks, first row).
template <class Launch>
void each_launch(int64_t rows, int64_t R, int threads, Launch&& launch) {
    const int64_t most = UINT32_MAX / threads * R;
    for (int64_t first = 0; first < rows; first += most) {
        const int64_t here = rows - first < most ? rows - first : most;
        launch(static_cast<unsigned>((here + R - 1) / R), first);
    }
}

// A row's vectors, the most that its lead can make them.
template <class T>
int64_t vectors_of(const RowArgs<T>& a) {
    constexpr int V = kVec<T>;
    const uint64_t apart = a.rows > 1 ? static_cast<uint64_t>(a.row_stride) * sizeof(T) : 0;
    const bool leads = (reinterpret_cast<uintptr_t>(a.logits) | apart) % 16 != 0;
    return (a.vocab + (leads ? V - 1 : 0) + V - 1) / V;
}
constexpr int64_t kHeldVectors = 16384;    // rows that a workgroup of 1024 lanes holds
constexpr int64_t kSplitVectors = 16384;
constexpr int64_t kShortVectors = 512;     // rows that at most a wave holds
constexpr int64_t kFewVectors = 16384;     // 256 KiB of logits

// The workgroups of a row: more than one where at most 64 rows have 16384 vectors
// or more (one row of 131072 floats 4.7 us a call against 9.7 by one workgroup,
// 52 of them 10.7 and 13.4, 52 of 200003 12.0 and 21.5), at most four a unit (eight:
// the 52 rows 14.5 and 18.3).  52 rows of 50001 floats lose 0.4 us by it, 256 of
// 131072 bfloat16 0.3.
template <class T>
int parts_of(const RowArgs<T>& a) {
    const int64_t vectors = vectors_of(a);
    if (a.rows == 0 || a.rows > kSplitRows || vectors < kSplitVectors || !a.run) return 1;
    const int64_t by_length = vectors / (kAhead * kThreads), by_rows = kWords / a.rows;
    const int64_t parts = by_length < by_rows ? by_length : by_rows;
    return static_cast<int>(parts < kMostParts ? parts : kMostParts);
}

// The lanes of a row by its vectors.  Its loss with the gradient holds rows of up
// to 16384 vectors; without, those of up to 512 (several rows a workgroup, whose
// reductions stay in a wave): a longer one needs no second pass, and a running
// (m, s) holds nothing.  Fewer rows than two a unit take 1024 lanes each.  A
// gradient from a saved lse takes a workgroup for each 1024 vectors of a row: 4096
// rows of 50001 floats 336 us against 368 with a workgroup a row, one row of 131072
// 4.6 against 40.
template <class T, Work W>
int rows_of(RowArgs<T> a, hipStream_t s) {
    if (a.rows == 0) return HK_OK;
    const int64_t vectors = vectors_of(a);
    const bool few = a.rows < 2 * kUnits;
    if constexpr (W == kGradient || W == kPolicyGradient || W == kPairGradient) {
        auto go = [&](auto lanes) {
            constexpr int L = decltype(lanes)::value, R = kThreads / L;
            const int64_t most = vectors / (kAhead * kThreads), parts = L < kThreads || most < 1 ? 1 : most < 65535 ? most : 65535;
            a.each = (vectors + parts - 1) / parts;
            each_launch(a.rows, R, kThreads, [&](unsigned blocks, int64_t first) {
                a.first = first;
                hipLaunchKernelGGL((hawk_row_gradient<T, L, W>), dim3(blocks, static_cast<unsigned>(parts)), dim3(kThreads), 0, s, a);
            });
        };
        if (vectors <= 32) go(Count<16>{});
        else if (vectors <= 256) go(Count<64>{});
        else go(Count<256>{});
    } else {
        const bool hold = W == kPolicy && a.bar_logits;
        const int parts = parts_of(a);
        a.each = (vectors + parts - 1) / parts;
        auto held = [&](auto lanes, auto count) {
            constexpr int L = decltype(lanes)::value, NV = decltype(count)::value;
            if (hold) launch_held<T, L, NV, W, W == kPolicy>(a, s);
            else if constexpr (L < 256) launch_held<T, L, NV, W, false>(a, s);
        };
        if (vectors <= 16) held(Count<16>{}, Count<1>{});
        else if (vectors <= 32) held(Count<16>{}, Count<2>{});
        else if (vectors <= 64) held(Count<16>{}, Count<4>{});
        else if (vectors <= 128) held(Count<64>{}, Count<2>{});
        else if (vectors <= 256) held(Count<64>{}, Count<4>{});
        else if (vectors <= kShortVectors) held(Count<64>{}, Count<8>{});
        else if (!hold && vectors <= 1024 && !few) launch_held<T, 64, 16, W, false>(a, s);
        else if (hold) {
            if constexpr (W == kPolicy) {
                if (vectors <= 1024) held(Count<256>{}, Count<4>{});
                else if (vectors <= 2048) held(Count<256>{}, Count<8>{});
                else if (vectors <= 4096 && few) held(Count<1024>{}, Count<4>{});
                else if (vectors <= 4096) held(Count<256>{}, Count<16>{});
                else if (vectors <= 8192) held(Count<512>{}, Count<16>{});
                else held(Count<1024>{}, Count<16>{});
            }
        } else if (parts > 1) {
            hipLaunchKernelGGL((hawk_row_parts<T, W>), dim3(static_cast<unsigned>(a.rows * parts)), dim3(kThreads), 0, s, a, parts);
        } else if (few) {
            hipLaunchKernelGGL((hawk_row_long<T, 1024, W>), dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, s, a);
        } else {
            each_launch(a.rows, 1, 256, [&](unsigned blocks, int64_t first) {
                a.first = first;
                hipLaunchKernelGGL((hawk_row_long<T, 256, W>), dim3(blocks), dim3(256), 0, s, a);
            });
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

// *out = the sum of x, which takes `partial`'s doubles (2 * runs(count)) on the way.
int64_t runs(int64_t count) { return (count + kRun - 1) / kRun; }
int total(const float* x, int64_t count, float* out, double* partial, hipStream_t s) {
    int64_t left = runs(count);
    const dim3 block(kTotalThreads);
    if (left <= 1) {
        hipLaunchKernelGGL((hawk_row_total<float, float>), dim3(1), block, 0, s, x, count, out);
        return launched("hawk_row_total launch");
    }
    hipLaunchKernelGGL((hawk_row_total<float, double>), dim3(static_cast<unsigned>(left)), block, 0, s, x, count, partial);
    while (left > kRun) {                 // more than 2^26 numbers
        double* next = partial + left;
        hipLaunchKernelGGL((hawk_row_total<double, double>), dim3(static_cast<unsigned>(runs(left))), block, 0, s,
                           static_cast<const double*>(partial), left, next);
        partial = next;
        left = runs(left);
    }
    hipLaunchKernelGGL((hawk_row_total<double, float>), dim3(1), block, 0, s, static_cast<const double*>(partial), left, out);
    return launched("hawk_row_total launch");
}

// Scratch: the sums' doubles, then a double a row and a float a pair (preference)
// or three floats a row (policy).
int64_t partial_count(const hk_row_loss_job& j) { return 2 * runs(j.rows > j.pairs ? j.rows : j.pairs); }
double* partials(void* scratch) { return static_cast<double*>(scratch); }
double* row_doubles(const hk_row_loss_job& j, void* scratch) { return partials(scratch) + partial_count(j); }
float* row_floats(const hk_row_loss_job& j, void* scratch) { return reinterpret_cast<float*>(row_doubles(j, scratch)); }
float* pair_floats(const hk_row_loss_job& j, void* scratch) { return reinterpret_cast<float*>(row_doubles(j, scratch) + j.rows); }

}  // namespace

extern "C" {

size_t hk_row_loss_scratch_bytes(const hk_row_loss_job* job) {
    if (!job || job->rows < 0 || job->pairs < 0) return 0;
    return sizeof(double) * static_cast<size_t>(partial_count(*job) + 2 * job->rows + (job->pairs + 1) / 2);
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
    if (job->rows > 0 && (job->loss || job->bar_logits) && !scratch) return hawk_internal::set_error(HK_EVALUE, "hk_policy_loss: scratch is required");
    hipStream_t s = static_cast<hipStream_t>(stream);
    bool summed = false;
    rc = typed(job->dtype, [&](auto t) {
        typedef decltype(t) T;
        RowArgs<T> a = args_of<T>(*job);
        a.row_loss = job->loss ? row_floats(*job, scratch) : nullptr;
        // in the rows' own launch where they are few: 200 rows of 48 floats 6.5 us a
        // call against 7.9 with a launch more, but the workgroups' fences wait for
        // what they stored: 4524 rows of 1660 float16 logits 126 us against 16
        summed = job->loss && job->state && job->rows > 0 && job->rows <= kRun && vectors_of(a) <= kShortVectors &&
                 job->rows * vectors_of(a) <= kFewVectors;
        if (summed) a.loss = job->loss;
        if (!a.bar_logits || vectors_of(a) <= kHeldVectors) return rows_of<T, kPolicy>(a, s);
        // longer rows twice: all their losses, then all their gradients (4096 rows of
        // 131072 floats 1077 us against 1091 with both in one workgroup's passes, 52 of
        // them 26 against 46)
        a.bar_logits = nullptr;
        if (!a.logp) a.logp = row_floats(*job, scratch) + job->rows;
        if (!a.lse) a.lse = row_floats(*job, scratch) + 2 * job->rows;
        const int rc = rows_of<T, kPolicy>(a, s);
        if (rc != HK_OK) return rc;
        a.bar_logits = static_cast<T*>(job->bar_logits);
        return rows_of<T, kPolicyGradient>(a, s);
    });
    if (rc != HK_OK || !job->loss || summed) return rc;
    return total(row_floats(*job, scratch), job->rows, job->loss, partials(scratch), s);
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

static int check_pairs(const hk_row_loss_job* j, const std::string& who) {
    using hawk_internal::set_error;
    const int rc = check_job(j, who);
    if (rc != HK_OK) return rc;
    if (j->pairs > 0 && !j->offsets) return set_error(HK_EVALUE, who + ": offsets are required");
    if (j->pairs == 0 && j->rows > 0) return set_error(HK_EVALUE, who + ": rows without a pair");
    return HK_OK;
}

int hk_preference_loss(const hk_row_loss_job* job, void* scratch, void* stream) {
    int rc = check_pairs(job, "hk_preference_loss");
    if (rc != HK_OK) return rc;
    if ((job->rows > 0 || job->pairs > 0) && !scratch)
        return hawk_internal::set_error(HK_EVALUE, "hk_preference_loss: scratch is required");
    hipStream_t s = static_cast<hipStream_t>(stream);
    float* pair_loss = pair_floats(*job, scratch);
    double* wide = row_doubles(*job, scratch);
    rc = typed(job->dtype, [&](auto t) {
        typedef decltype(t) T;
        RowArgs<T> a = args_of<T>(*job);
        a.wide = wide;
        return rows_of<T, kLogp>(a, s);
    });
    if (rc != HK_OK) return rc;
    if (job->pairs > 0) {
        PairArgs p = pairs_of(*job);
        p.logp = wide;
        p.pair_loss = pair_loss;
        if (job->pairs <= kPairs) {
            hipLaunchKernelGGL(hawk_pair_loss<true>, dim3(1), dim3(kPairThreads), 0, s, p, job->loss);
            return launched("hawk_pair_loss launch");
        }
        const int64_t blocks = (job->pairs + kPairWaves - 1) / kPairWaves, most = UINT32_MAX / kPairThreads;
        hipLaunchKernelGGL(hawk_pair_loss<false>, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(kPairThreads), 0, s,
                           p, nullptr);
        rc = launched("hawk_pair_loss launch");
        if (rc != HK_OK) return rc;
    }
    return job->loss ? total(pair_loss, job->pairs, job->loss, partials(scratch), s) : HK_OK;
}

int hk_preference_loss_vjp(const hk_row_loss_job* job, void* scratch, void* stream) {
    (void)scratch;
    const int rc = check_pairs(job, "hk_preference_loss_vjp");
    if (rc != HK_OK) return rc;
    if (job->rows == 0) return HK_OK;
    if (!job->lse || !job->margin || !job->bar_logits)
        return hawk_internal::set_error(HK_EVALUE, "hk_preference_loss_vjp: lse, margin and bar_logits are required");
    hipStream_t s = static_cast<hipStream_t>(stream);
    return typed(job->dtype, [&](auto t) {
        typedef decltype(t) T;
        RowArgs<T> a = args_of<T>(*job);
        a.pairs = pairs_of(*job);
        return rows_of<T, kPairGradient>(a, s);
    });
}

}  // extern "C"
