// hawk_sample.hip — a token drawn from each row of logits by a given random number:
// temperature, top-k, top-p, min-p and the inverse of the kept tokens' distribution.
//
// The mathematics.  w_v = exp((x_v - max) / T).  Order a row's tokens by logit, the
// highest first, equal ones by index; each filter keeps a prefix of that order, so all
// of them keep the shortest one, whose last token has the order code
// (descending key, index).  The token drawn is the first, by index, at which the kept
// tokens' running sum passes u times their whole sum.
//
// Which token that is is decided at borders between sums, of which a row has as many
// as tokens: with weights rounded to 32 bits one row in some thousands would draw
// another token.  The weights are taken in 64 bits and held as whole numbers of
// 2^-shift, shift = 62 - log2(vocabulary) (51 at most): their sums stay below 2^63 and
// are exact, so neither the order in which atomics add them nor the way a row is cut
// changes a bit.  A weight is off by half a unit, so a row's sum by up to vocabulary *
// 2^-(shift + 1) of the highest weight: 2^-29 of it at 2^17 tokens, 2^-19 at 2^22.  A
// token below half a unit weighs nothing.
//
// What bounds it: the weights' 64-bit arithmetic, some thirty instructions a token, in the
// pass that sums them (one before it finds the highest logit; the token is looked for along
// one run of one wave): 4096 rows of 50001 float16 logits take 218 us, their bytes 62.  And,
// where rows are few, four launches that wait for one another (64 rows of 131072 bfloat16
// with a top-p: 69.5 us, of which the largest kernels take 23 each; a workgroup a row took
// 156).

#include "hawk_core.h"
#include "hawk_internal.h"
#include "hawk_vec.h"

#include <hip/hip_runtime.h>
#include <cstdint>
#include <string>

namespace {

using namespace hawk_vec;

typedef unsigned long long u64;

constexpr int64_t kMostVocab = 1 << 22;
constexpr int kBins = 2048;
constexpr int kList = 1024;                // candidates that are ranked against each other
constexpr u64 kAll = ~0ull;
constexpr int64_t kUnits = 256;            // compute units

template <class T> constexpr int kVec = 16 / static_cast<int>(sizeof(T));

template <class T>
struct SampleArgs {
    const T* logits;
    const void* u;
    const float *temperature, *top_p, *min_p;   // of each row, or NULL
    const int32_t* top_k;
    void* token;
    float* logp;
    int64_t rows, vocab, row_stride;
    double temperature_all, top_p_all, min_p_all;
    int64_t top_k_all;
    int u64bits, token64, shift;
};

// How a row's weights are taken: exp((x - top) / T) = 2^((x - top) octaves), as a
// multiple of 2^-shift.
constexpr int kTable = 128;
struct Weights {
    double top, octaves;
    const double* table;       // 2^(shift + j / 128)
};

constexpr u64 kUnit = 0x4330000000000000ull;             // 2^52, whose last digit is 1, as bits

// The weight, a whole number.  The exponent (in octaves) is split into an octave, a 128th
// of one from the table and a rest r of at most 1/256, whose power is a Taylor polynomial:
// the first term left out is (r ln 2)^5 / 120 < 2^-49.  Below 2^-80 it is 0, for -inf too.
__device__ __forceinline__ u64 weight_of(const Weights& k, float x) {
    constexpr double ln2 = 0.6931471805599453094;
    const double y = fmax((static_cast<double>(x) - k.top) * k.octaves, -80.0);
    const double near = __builtin_fma(y, static_cast<double>(kTable), 0x1.8p52);
    const int n = static_cast<int>(__builtin_bit_cast(uint64_t, near));
    const double r = __builtin_fma(near - 0x1.8p52, -1.0 / kTable, y);
    double p = __builtin_fma(r, ln2 * ln2 * ln2 * ln2 / 24.0, ln2 * ln2 * ln2 / 6.0);
    p = __builtin_fma(r, p, ln2 * ln2 / 2.0);
    p = __builtin_fma(r, p, ln2);
    p = __builtin_fma(r, p, 1.0);
    // n / 128 octaves more: the numbers are normal, so their exponents are added to
    const uint64_t w = __builtin_bit_cast(uint64_t, p * k.table[n & (kTable - 1)]) + (static_cast<uint64_t>(static_cast<uint32_t>(n & -kTable) << 13) << 32);
    return __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, w) + 0x1p52) - kUnit;
}


// A logit's place in descending order: smaller is higher.  Both zeros are one.
__device__ __forceinline__ uint32_t place_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}

// Running sums over a wave's lanes, by moves between lanes that need no memory: within
// rows of 16 lanes by 1, 2, 4 and 8, then a row's last lane into the rows after it.
template <int Control, int Rows>
__device__ __forceinline__ u64 moved(u64 v) {
    const uint32_t low = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), Control, Rows, 0xf, false);
    const uint32_t high = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), Control, Rows, 0xf, false);
    return static_cast<u64>(high) << 32 | low;
}
__device__ __forceinline__ u64 wave_upto(u64 v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    v += moved<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ u64 last_lane(u64 v) {
    const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(v), 63), high = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), 63);
    return static_cast<u64>(high) << 32 | low;
}
// The sum of a wave's numbers, and of the lanes before this one.
__device__ __forceinline__ u64 wave_sum(u64 v) { return last_lane(wave_upto(v)); }
__device__ __forceinline__ u64 wave_before(u64 v) { return wave_upto(v) - v; }

constexpr int kFew = 256;                  // candidates that are ranked by counting
constexpr int kCells = 4;                  // of a wave: runs of its part of a row
template <int NT>
struct Sums {
    double table[kTable];
    u64 cells[NT / 64 * kCells], waves[NT / 64], low;
    float tops[NT / 64];
    int bad;
};
template <int NT, bool Filtered>
struct Shared : Sums<NT> {};
template <int NT>
struct Shared<NT, true> : Sums<NT> {
    u64 bins[kBins], code[kList], value[kList], ahead[kFew], base, inside, high;
    int rank[kFew], found, listed;
};

// The sum of the threads' numbers before this one, and of all.
template <int NT>
__device__ __forceinline__ u64 block_before(Sums<NT>& s, u64 own, u64& all) {
    u64 before = wave_before(own);
    if ((threadIdx.x & 63) == 63) s.waves[threadIdx.x >> 6] = before + own;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        if (w == static_cast<int>(threadIdx.x >> 6)) before += all;
        all += s.waves[w];
    }
    __syncthreads();
    return before;
}

// A row, or a part of one, read by NT threads: from vector `begin` on, wave w has the
// vectors [w, w + 1) * steps * 64, so the waves' shares, and a wave's steps, follow each
// other by index.  Every pass reads the row; all but the first find it in the caches.
template <class T, int NT>
struct Row {
    const T* at;               // the row's address less its lead, 16-byte aligned
    int low, high;             // the row's first position, and past its last
    int begin, steps;          // the part's first vector; vectors of a lane
    int wave;                  // whose share this is

    // `part` of the parts of row n, each of NT * steps vectors.
    __device__ __forceinline__ Row(const SampleArgs<T>& a, int64_t n, int part, int steps_, int wave_) : steps(steps_), wave(wave_) {
        const T* from = a.logits + n * a.row_stride;
        low = static_cast<int>(reinterpret_cast<uintptr_t>(from) % 16 / sizeof(T));
        at = from - low;
        high = low + static_cast<int>(a.vocab);
        begin = part * (NT * steps);
    }
    __device__ __forceinline__ int position(int i) const {
        return (begin + (wave * steps + i) * 64 + static_cast<int>(threadIdx.x & 63)) * kVec<T>;
    }
    // What lies before the row or past its end is -inf.
    __device__ __forceinline__ Raw<T, kVec<T>> vector(int p) const {
        constexpr int V = kVec<T>;
        if (p >= low && p + V <= high) return load_raw<T, V>(at + p);
        Raw<T, V> x = splat<T, V>(static_cast<T>(-INFINITY));
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (p + j >= low && p + j < high) put<T, V>(x, j, at[p + j]);
        return x;
    }
    // f(first index, vector) of every step from `from` up to `end`, kAhead loads at a time;
    // a wave whose vectors are all in the row asks that once.
    template <class F> __device__ __forceinline__ void each(int from, int end, F&& f) const {
        constexpr int V = kVec<T>, kAhead = 2;
        for (int i = from; i < end; i += kAhead) {
            Raw<T, V> x[kAhead];
            const int p = position(i), first = __builtin_amdgcn_readfirstlane(p);
            if (i + kAhead <= end && first >= low && first + kAhead * 64 * V <= high) {
#pragma unroll
                for (int b = 0; b < kAhead; ++b) x[b] = load_raw<T, V>(at + p + b * 64 * V);
            } else {
#pragma unroll
                for (int b = 0; b < kAhead; ++b)
                    if (i + b < end) x[b] = vector(p + b * 64 * V);
            }
#pragma unroll
            for (int b = 0; b < kAhead; ++b) {
                if (i + b < end) f(p + b * 64 * V - low, x[b]);
                __builtin_amdgcn_sched_barrier(0);         // a vector at a time: fewer registers, more waves
            }
        }
    }
    // f(index, number) of every token.
    template <class F> __device__ __forceinline__ void tokens(int vocab, F&& f) const {
        each(0, steps, [&](int first, const Raw<T, kVec<T>>& v) {
#pragma unroll
            for (int j = 0; j < kVec<T>; ++j) {
                const int i = first + j;
                if (i >= 0 && i < vocab) f(static_cast<uint32_t>(i), widen<T, kVec<T>>(v, j));
            }
        });
    }
};

// Bins of the tokens with codes in [low, high], smaller codes first: a 64th of an octave
// below the highest logit each (shift < 0), or runs of 2^shift codes.
struct Bins {
    u64 low, high;
    double top, octaves;
    int shift;
    __device__ __forceinline__ int of(u64 code, float x) const {
        if (code < low || code > high) return -1;
        if (shift >= 0) return static_cast<int>((code - low) >> shift);
        const double d = (top - static_cast<double>(x)) * octaves * 64.0;
        return d < kBins - 1 ? static_cast<int>(d) : kBins - 1;      // (a NaN, of -inf, is the last)
    }
};
__device__ __forceinline__ u64 code_of(uint32_t i, float x) { return static_cast<u64>(place_of(x)) << 32 | i; }

// Adds the tokens' weights (or 1 each) to their bins.
template <class T, int NT>
__device__ __forceinline__ void fill(u64* to, const Row<T, NT>& row, int vocab, const Weights& k, const Bins& bins, bool mass) {
    u64 rest = 0;                                         // the last bin's, which may have most of a row (what is barred)
    row.tokens(vocab, [&](uint32_t i, float x) {
        const int b = bins.of(code_of(i, x), x);
        if (b < 0) return;
        if (mass) {
            const u64 w = weight_of(k, x);
            if (b == kBins - 1) rest += w;
            else atomicAdd(&to[b], w);
        } else {
            if (b == kBins - 1) ++rest;
            else atomicAdd(reinterpret_cast<uint32_t*>(&to[b]), 1u);
        }
    });
    rest = wave_sum(rest);
    if ((threadIdx.x & 63) == 0 && rest) atomicAdd(&to[kBins - 1], rest);
}
__device__ __forceinline__ u64 share_of(double share, u64 all) {
    const double want = ceil(share * static_cast<double>(all));
    const u64 target = want < 1.0 ? 1 : static_cast<u64>(want);
    return target < all ? target : all;
}
// The first bin at which the running sum from `base` reaches the target: s.found (kBins:
// none), s.base the sum before it, s.inside its own.  With share >= 0 the target is that
// share of the sum.
template <int NT>
__device__ __forceinline__ void locate(Shared<NT, true>& s, const u64* bins, u64 base, u64& target, double share) {
    constexpr int Each = kBins / NT;
    u64 v[Each], own = 0, all;
#pragma unroll
    for (int b = 0; b < Each; ++b) own += v[b] = bins[threadIdx.x * Each + b];
    u64 before = block_before(s, own, all) + base;
    if (share >= 0.0) target = share_of(share, all);
    if (before < target && before + own >= target) {
#pragma unroll
        for (int b = 0; b < Each; ++b) {
            if (before < target && before + v[b] >= target) {
                s.found = threadIdx.x * Each + b;
                s.base = before;
                s.inside = v[b];
            }
            before += v[b];
        }
    }
    __syncthreads();
}
template <class T, int NT>
__device__ __forceinline__ void search(Shared<NT, true>& s, const Row<T, NT>& row, int vocab, const Weights& k, const Bins& bins, bool mass, u64 base,
                                       u64& target, double share) {
    for (int b = threadIdx.x; b < kBins; b += NT) s.bins[b] = 0;
    if (threadIdx.x == 0) s.found = kBins, s.listed = 0, s.low = kAll, s.high = 0;
    __syncthreads();
    fill(s.bins, row, vocab, k, bins, mass);
    __syncthreads();
    locate(s, s.bins, base, target, share);
}

// The list's first n entries in ascending order of their codes (their low 32 bits alone:
// Index).  A bitonic network (Batcher, Sorting networks and their applications, 1968).
template <int NT, bool Index>
__device__ __forceinline__ void sort(Shared<NT, true>& s, int n) {
    int size = 2;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += NT) s.code[i] = kAll, s.value[i] = 0;
    __syncthreads();
    for (int width = 2; width <= size; width *= 2)
        for (int d = width / 2; d > 0; d /= 2) {
            for (int t = threadIdx.x; t < size / 2; t += NT) {
                const int i = (t & ~(d - 1)) * 2 | (t & (d - 1)), k = i | d;
                const u64 a = s.code[i], b = s.code[k];
                const bool above = Index ? static_cast<uint32_t>(a) > static_cast<uint32_t>(b) : a > b;
                const bool below = Index ? static_cast<uint32_t>(a) < static_cast<uint32_t>(b) : a < b;
                if ((i & width) == 0 ? above : below) {
                    s.code[i] = b;
                    s.code[k] = a;
                    const u64 v = s.value[i];
                    s.value[i] = s.value[k];
                    s.value[k] = v;
                }
            }
            __syncthreads();
        }
}
// The sum of the sorted list's values before this thread's entries, which are Each after
// each other.
template <int NT> constexpr int kEach = kList >= NT ? kList / NT : 1;
template <int NT>
__device__ __forceinline__ u64 list_before(Shared<NT, true>& s, int n, u64& all) {
    u64 own = 0;
#pragma unroll
    for (int e = 0; e < kEach<NT>; ++e) {
        const int i = static_cast<int>(threadIdx.x) * kEach<NT> + e;
        if (i < n) own += s.value[i];
    }
    return block_before(s, own, all);
}

// The code of the last token of a prefix: of those with code <= limit, in order, the
// first at which the running sum (of 1 each, or of the weights) reaches the target.
template <class T, int NT>
__device__ __forceinline__ u64 last_of(Shared<NT, true>& s, const Row<T, NT>& row, int vocab, const Weights& k, u64 limit, bool mass, u64 target, double share) {
    Bins bins{0, limit, k.top, k.octaves, -1};
    u64 base = 0;
    for (;;) {
        search(s, row, vocab, k, bins, mass, base, target, share);
        share = -1.0;
        const int found = s.found;
        if (found >= kBins) return limit;                // less than the target in all: everything is kept
        base = s.base;
        u64 least = kAll, most = 0;
        row.tokens(vocab, [&](uint32_t i, float x) {
            const u64 code = code_of(i, x);
            if (bins.of(code, x) != found) return;
            const int at = atomicAdd(&s.listed, 1);
            if (at < kList) {
                s.code[at] = code;
                s.value[at] = mass ? weight_of(k, x) : 1;
            }
            least = code < least ? code : least;
            most = code > most ? code : most;
        });
        if (least != kAll) {
            atomicMin(&s.low, least);
            atomicMax(&s.high, most);
        }
        __syncthreads();
        const int n = s.listed;
        if (n <= kList) {
            sort<NT, false>(s, n);
            u64 all, before = list_before(s, n, all) + base;
#pragma unroll
            for (int e = 0; e < kEach<NT>; ++e) {
                const int i = static_cast<int>(threadIdx.x) * kEach<NT> + e;
                if (i >= n) break;
                if (before < target && before + s.value[i] >= target) s.low = s.code[i];
                before += s.value[i];
            }
            __syncthreads();
            const u64 cut = s.low;
            __syncthreads();
            return cut;
        }
        bins.low = s.low;
        bins.high = s.high;
        bins.shift = 0;
        while ((bins.high - bins.low) >> bins.shift >= kBins) ++bins.shift;
        __syncthreads();
    }
}

// The first running sum above u * all: at least one whole number above its floor.
__device__ __forceinline__ u64 aim(double u, u64 all) {
    const double want = u * static_cast<double>(all);
    const u64 target = want >= 0.0 ? (want < 0x1p63 ? static_cast<u64>(want) : kAll - 1) + 1 : 1;
    return target > all ? all : target;
}

// What a row asks for.
struct Asked {
    double heat, u, share;     // share: top_p, or -1 where it keeps everything
    u64 count, least;          // count: top_k, or kAll; least: the least weight that min_p keeps
    __device__ __forceinline__ bool every() const { return count == kAll && share < 0.0 && least == 0; }
};
template <class T>
__device__ __forceinline__ Asked asked(const SampleArgs<T>& a, int64_t n) {
    Asked q;
    q.heat = a.temperature ? static_cast<double>(a.temperature[n]) : a.temperature_all;
    q.u = a.u64bits ? static_cast<const double*>(a.u)[n] : static_cast<double>(static_cast<const float*>(a.u)[n]);
    const double top_p = a.top_p ? static_cast<double>(a.top_p[n]) : a.top_p_all;
    const double min_p = a.min_p ? static_cast<double>(a.min_p[n]) : a.min_p_all;
    // no weight is above 1: a larger min_p leaves the highest alone
    const int64_t top_k = min_p > 1.0 ? 1 : a.top_k ? static_cast<int64_t>(a.top_k[n]) : a.top_k_all;
    q.share = top_p < 1.0 ? fmax(top_p, 0.0) : -1.0;
    q.count = top_k > 0 && top_k < a.vocab ? static_cast<u64>(top_k) : kAll;
    q.least = min_p > 0.0 && min_p <= 1.0 ? static_cast<u64>(ceil(scaled(min_p, a.shift))) : 0;
    return q;
}
// A row's highest logit, NaN where one is: whether it has a token to draw, by its weights.
__device__ __forceinline__ bool drawn(const Asked& q, float top) { return q.heat > 0.0 && q.u == q.u && top > -INFINITY; }
__device__ __forceinline__ Weights weights_of(const Asked& q, float top, const double* table) {
    return Weights{static_cast<double>(top), fmin(1.4426950408889634074 / q.heat, 1e300), table};
}
template <class T>
__device__ __forceinline__ void answer(const SampleArgs<T>& a, int64_t n, int64_t token, float logp) {
    if (a.token) {
        if (a.token64) static_cast<int64_t*>(a.token)[n] = token;
        else static_cast<int32_t*>(a.token)[n] = static_cast<int32_t>(token);
    }
    if (a.logp) a.logp[n] = logp;
}
// The answer of a row that is not drawn by its weights; `first` its highest logit's first token.
template <class T>
__device__ __forceinline__ void answer_plain(const SampleArgs<T>& a, int64_t n, const Asked& q, float top, int64_t first) {
    const bool none = !(q.heat >= 0.0) || !(q.u == q.u) || !(top == top);
    if (none || top == -INFINITY) answer(a, n, -1, none ? NAN : -INFINITY);
    else answer(a, n, first, 0.0f);
}
template <class T>
__device__ __forceinline__ void answer_drawn(const SampleArgs<T>& a, int64_t n, const Asked& q, float top, u64 at, u64 all) {
    const int64_t token = at < static_cast<u64>(a.vocab) ? static_cast<int64_t>(at) : a.vocab - 1;
    const double x = static_cast<double>(static_cast<float>(a.logits[n * a.row_stride + token]));
    answer(a, n, token, static_cast<float>((top == INFINITY ? 0.0 : (x - top) / q.heat) - log(scaled(static_cast<double>(all), top == INFINITY ? 0 : -a.shift))));
}
// Of a row's infinities, which share the whole, how many are kept.
__device__ __forceinline__ u64 infinities(const Asked& q, u64 count) {
    const u64 some = q.count < count ? q.count : count;
    return q.share < 0.0 ? some : share_of(q.share, some);
}

// Every token that may be kept is in the list, n of them: the filters, and the one drawn.
// Few are ranked by counting those before each, which waits for nothing; more are sorted.
template <int NT>
__device__ __forceinline__ u64 from_list(Shared<NT, true>& s, int n, const Asked& q, u64& all) {
    constexpr int Mine = kEach<NT>, Few = kFew > NT ? kFew / NT : 1;
    const int tid = threadIdx.x, some = q.count < static_cast<u64>(n) ? static_cast<int>(q.count) : n;
    const bool few = n <= kFew;
    u64 before = 0, target = kAll;
    if (!few) {
        sort<NT, false>(s, n);
        before = list_before(s, some, all);
    } else {
        u64 own = 0;
#pragma unroll
        for (int e = 0; e < Few; ++e) {
            const int i = tid + e * NT;
            if (i >= n) break;
            const u64 code = s.code[i];
            u64 sum = 0;
            int rank = 0;
            for (int o = 0; o < n; ++o) {
                const bool ahead = s.code[o] < code;
                rank += ahead;
                sum += ahead ? s.value[o] : 0;
            }
            s.rank[i] = rank;
            s.ahead[i] = sum;
            if (rank < some) own += s.value[i];
        }
        block_before(s, own, all);
    }
    if (q.share >= 0.0) target = share_of(q.share, all);
    if (!few) {
#pragma unroll
        for (int e = 0; e < Mine; ++e) {
            const int i = tid * Mine + e;
            if (i >= n) break;
            const u64 v = s.value[i];
            if (i > 0 && (i >= some || before >= target || v < q.least)) s.value[i] = 0;
            before += v;
        }
        __syncthreads();
        sort<NT, true>(s, n);
        before = list_before(s, n, all);
        const u64 aimed = aim(q.u, all);
#pragma unroll
        for (int e = 0; e < Mine; ++e) {
            const int i = tid * Mine + e;
            if (i >= n) break;
            if (before < aimed && before + s.value[i] >= aimed) s.low = s.code[i] & 0xffffffffull;
            before += s.value[i];
        }
    } else {
        u64 own = 0;
#pragma unroll
        for (int e = 0; e < Few; ++e) {
            const int i = tid + e * NT;
            if (i >= n) break;
            if (s.rank[i] > 0 && (s.rank[i] >= some || s.ahead[i] >= target || s.value[i] < q.least)) s.value[i] = 0;
            own += s.value[i];
        }
        block_before(s, own, all);
        const u64 aimed = aim(q.u, all);
#pragma unroll
        for (int e = 0; e < Few; ++e) {
            const int i = tid + e * NT;
            if (i >= n) break;
            const uint32_t at = static_cast<uint32_t>(s.code[i]);
            u64 sum = 0;
            for (int o = 0; o < n; ++o) sum += static_cast<uint32_t>(s.code[o]) < at ? s.value[o] : 0;
            if (sum < aimed && sum + s.value[i] >= aimed) s.low = at;
        }
    }
    __syncthreads();
    return s.low;
}

// The sums of a wave's runs, kCells at most, of what `weight` (of an index and a number)
// gives; their sum.
template <class T, int NT, class F>
__device__ __forceinline__ u64 sum_runs(u64* cells, const Row<T, NT>& row, F&& weight) {
    constexpr int V = kVec<T>;
    const int run = (row.steps + kCells - 1) / kCells;
    u64 total = 0;
#pragma unroll 1
    for (int c = 0; c < kCells; ++c) {
        const int from = c * run, end = from + run < row.steps ? from + run : row.steps;
        u64 sum = 0;
        if (from < end) {
            row.each(from, end, [&](int first, const Raw<T, V>& v) {
#pragma unroll
                for (int j = 0; j < V; ++j) sum += weight(static_cast<uint32_t>(first + j), widen<T, V>(v, j));
            });
            sum = wave_sum(sum);
        }
        if ((threadIdx.x & 63) == 0) cells[c] = sum;
        total += sum;
    }
    return total;
}
// A wave goes along its run c, before which `before` has passed: the token at which the
// target is reached is put into `low`.
template <class T, int NT, class F>
__device__ __forceinline__ void go_along(u64& low, const Row<T, NT>& row, int c, u64 before, u64 target, F&& weight) {
    constexpr int V = kVec<T>;
    const int run = (row.steps + kCells - 1) / kCells, end = (c + 1) * run < row.steps ? (c + 1) * run : row.steps;
#pragma unroll 1
    for (int i = c * run; i < end; ++i) {
        const int p = row.position(i), first = p - row.low;
        const Raw<T, V> v = row.vector(p);
        u64 w[V], own = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) own += w[j] = weight(static_cast<uint32_t>(first + j), widen<T, V>(v, j));
        const u64 step = wave_sum(own);
        if (before + step >= target) {
            u64 upto = before + wave_before(own);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (upto < target && upto + w[j] >= target) low = static_cast<u64>(first + j);
                upto += w[j];
            }
            return;
        }
        before += step;
    }
}
// The token drawn from those that `weight` gives one: the waves' runs are summed, and the
// wave that has the one that is aimed at goes along it.  `some` says how much of the sum
// of all there is to draw from.
template <class T, int NT, class F, class G>
__device__ __forceinline__ u64 from_row(Sums<NT>& s, const Row<T, NT>& row, double u, F&& weight, G&& some, u64& all) {
    const int lane = threadIdx.x & 63, wave = row.wave;
    const u64 total = sum_runs(s.cells + wave * kCells, row, weight);
    if (lane == 0) s.waves[wave] = total;
    __syncthreads();
    all = 0;
    u64 before = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        if (w == wave) before = all;
        all += s.waves[w];
    }
    all = some(all);
    const u64 target = aim(u, all);
    if (before < target && before + total >= target) {
        int c = 0;
        while (before + s.cells[wave * kCells + c] < target) before += s.cells[wave * kCells + c++];
        go_along(s.low, row, c, before, target, weight);
    }
    __syncthreads();
    return s.low;
}

// The highest of the threads' numbers, NaN where one is.
template <class T, int NT>
__device__ __forceinline__ float top_of(Sums<NT>& s, const Row<T, NT>& row) {
    constexpr int V = kVec<T>;
    float m = -INFINITY;
    bool bad = false;
    row.each(0, row.steps, [&](int, const Raw<T, V>& v) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float x = widen<T, V>(v, j);
            m = fmaxf(m, x);
            bad |= !(x == x);
        }
    });
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (threadIdx.x == 0) s.bad = 0;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.tops[threadIdx.x >> 6] = m;
    if (bad) s.bad = 1;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) m = fmaxf(m, s.tops[w]);
    return s.bad ? NAN : m;
}
// The first token of the highest logit (kAll: not here), in s.low.
template <class T, int NT>
__device__ __forceinline__ void first_of(Sums<NT>& s, const Row<T, NT>& row, int vocab, float top) {
    if (threadIdx.x == 0) s.low = kAll;
    __syncthreads();
    u64 first = kAll;
    row.tokens(vocab, [&](uint32_t i, float x) { if (x == top && i < first) first = i; });
    if (first != kAll) atomicMin(&s.low, first);
    __syncthreads();
}
template <int NT>
__device__ __forceinline__ void make_table(Sums<NT>& s, int shift) {
    for (int j = threadIdx.x; j < kTable; j += NT) s.table[j] = scaled(exp2(static_cast<double>(j) / kTable), shift);
}

// A row of NT threads.  Filtered: it may have filters.  Listed: it fits the list.
template <bool Filtered, bool Listed, class T, int NT>
__device__ __forceinline__ u64 from_whole(Shared<NT, Filtered>& s, const Row<T, NT>& row, int vocab, const Asked& q, float top, u64& all) {
    const Weights k = weights_of(q, top, s.table);
    auto whole = [](u64 sum) { return sum; };
    if (top == INFINITY)
        return from_row(s, row, q.u, [](uint32_t, float x) -> u64 { return x == INFINITY; }, [&](u64 count) { return infinities(q, count); }, all);
    if (!Filtered || q.every()) return from_row(s, row, q.u, [&](uint32_t, float x) { return weight_of(k, x); }, whole, all);
    if constexpr (Filtered) {
        bool listed = Listed;
        if (Listed) {
            row.tokens(vocab, [&](uint32_t i, float x) {
                s.code[i] = code_of(i, x);
                s.value[i] = weight_of(k, x);
            });
            if (threadIdx.x == 0) s.listed = vocab;
        } else if (q.count <= kList) {
            // the tokens down to the bin that has the last of the top_k
            u64 target = q.count;
            const Bins bins{0, kAll, k.top, k.octaves, -1};
            search(s, row, vocab, k, bins, false, 0, target, -1.0);
            if (s.base + s.inside <= kList) {
                const int found = s.found;
                row.tokens(vocab, [&](uint32_t i, float x) {
                    const u64 code = code_of(i, x);
                    if (bins.of(code, x) > found) return;
                    const int to = atomicAdd(&s.listed, 1);
                    s.code[to] = code;
                    s.value[to] = weight_of(k, x);
                });
                listed = true;
            }
        }
        __syncthreads();
        if (listed) return from_list(s, s.listed, q, all);
        u64 cut = kAll;
        for (int f = 0; f < 2; ++f) {                    // top_k, then top_p of what it keeps
            if (f == 0 ? q.count == kAll : q.share < 0.0) continue;
            cut = last_of(s, row, vocab, k, cut, f == 1, q.count, f == 0 ? -1.0 : q.share);
        }
        return from_row(s, row, q.u, [&](uint32_t i, float x) -> u64 {
            if (code_of(i, x) > cut) return 0;
            const u64 w = weight_of(k, x);
            return w >= q.least ? w : 0;
        }, whole, all);
    }
    return 0;
}

// Rows of a workgroup each.
template <class T, int NT, bool Filtered, bool Listed>
__global__ void __launch_bounds__(NT, Filtered ? 4 : 6) hawk_sample(const SampleArgs<T> a) {
    __shared__ Shared<NT, Filtered> s;
    const int vocab = static_cast<int>(a.vocab);
    make_table(s, a.shift);
    for (int64_t n = blockIdx.x; n < a.rows; n += gridDim.x) {
        __syncthreads();
        Row<T, NT> row(a, n, 0, 0, threadIdx.x >> 6);
        row.steps = (row.high + kVec<T> * NT - 1) / (kVec<T> * NT);
        const Asked q = asked(a, n);
        const float top = top_of(s, row);
        if (drawn(q, top)) {
            u64 all;
            const u64 at = from_whole<Filtered, Listed>(s, row, vocab, q, top, all);
            if (threadIdx.x == 0) answer_drawn(a, n, q, top, at, all);
        } else {
            if (q.heat == 0.0 && top > -INFINITY) first_of(s, row, vocab, top);
            if (threadIdx.x == 0) answer_plain(a, n, q, top, static_cast<int64_t>(s.low));
        }
    }
}

// ---- few long rows: several workgroups a row, four launches --------------------------------
//
// Each workgroup has a part of a row.  The first launch finds the parts' highest logits,
// the second sums the parts' runs or, where a filter needs the order, fills the row's
// bins; the third sums what is above the bin that the filter ends in and lists that bin's
// tokens; the fourth, a workgroup a row, ranks the list and draws.  Sums of whole numbers
// are the same in any order.  A row whose list is too long, or whose top_k is, is taken
// whole by the fourth.

constexpr int kPart = 256, kMostParts = 64, kDraw = 1024;
struct Parts {
    float* tops;               // [row][part]
    u64* firsts;               // [row][part]: the first token of the part's highest logit, of rows at temperature 0
    u64 *bins, *cells;         // [row][kBins], [row][part][wave][kCells]
    u64 *code, *value;         // [row][kList]
    int* listed;               // [row]
    int parts, steps;
};
// What a row's parts do: nothing (its answer needs no sums, or the last launch takes it
// whole), sums of runs, bins of counts or of weights.
enum Way { kNothing, kRuns, kCounts, kMasses };
__device__ __forceinline__ Way way_of(const Asked& q, float top) {
    if (!drawn(q, top)) return kNothing;
    if (top == INFINITY || (q.count == kAll && q.share < 0.0)) return kRuns;
    return q.count == kAll ? kMasses : q.count <= kList ? kCounts : kNothing;
}
// The row's highest logit of its parts', NaN where one is.
__device__ __forceinline__ float joined_top(const Parts& p, int64_t n) {
    const int lane = threadIdx.x & 63;
    float m = lane < p.parts ? p.tops[n * p.parts + lane] : -INFINITY;
    const bool bad = __any(!(m == m));
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    return bad ? NAN : m;
}

template <class T>
__global__ void __launch_bounds__(kPart) hawk_sample_tops(const SampleArgs<T> a, const Parts p) {
    __shared__ Sums<kPart> s;
    const int part = blockIdx.x;
    const int64_t n = blockIdx.y;
    const Row<T, kPart> row(a, n, part, p.steps, threadIdx.x >> 6);
    for (int b = part * kPart + threadIdx.x; b < kBins; b += p.parts * kPart) p.bins[n * kBins + b] = 0;
    if (part == 0 && threadIdx.x == 0) p.listed[n] = 0;
    const float top = top_of(s, row);
    if (threadIdx.x == 0) p.tops[n * p.parts + part] = top;
    if (asked(a, n).heat != 0.0) return;
    first_of(s, row, static_cast<int>(a.vocab), top);
    if (threadIdx.x == 0) p.firsts[n * p.parts + part] = s.low;
}

template <class T>
__global__ void __launch_bounds__(kPart, 4) hawk_sample_bins(const SampleArgs<T> a, const Parts p) {
    __shared__ Shared<kPart, true> s;
    const int part = blockIdx.x, vocab = static_cast<int>(a.vocab);
    const int64_t n = blockIdx.y;
    const Asked q = asked(a, n);
    const float top = joined_top(p, n);
    const Way way = way_of(q, top);
    if (way == kNothing) return;
    make_table(s, a.shift);
    for (int b = threadIdx.x; b < kBins; b += kPart) s.bins[b] = 0;
    __syncthreads();
    const Row<T, kPart> row(a, n, part, p.steps, threadIdx.x >> 6);
    const Weights k = weights_of(q, top, s.table);
    if (way == kRuns) {
        u64* cells = p.cells + ((n * p.parts + part) * (kPart / 64) + row.wave) * kCells;
        if (top == INFINITY) sum_runs(cells, row, [](uint32_t, float x) -> u64 { return x == INFINITY; });
        else sum_runs(cells, row, [&](uint32_t, float x) -> u64 { const u64 w = weight_of(k, x); return w >= q.least ? w : 0; });
        return;
    }
    fill(s.bins, row, vocab, k, Bins{0, kAll, k.top, k.octaves, -1}, way == kMasses);
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kPart)
        if (s.bins[b]) atomicAdd(&p.bins[n * kBins + b], s.bins[b]);
}

template <class T>
__global__ void __launch_bounds__(kPart, 4) hawk_sample_keep(const SampleArgs<T> a, const Parts p) {
    __shared__ Shared<kPart, true> s;
    const int part = blockIdx.x, vocab = static_cast<int>(a.vocab);
    const int64_t n = blockIdx.y;
    const Asked q = asked(a, n);
    const float top = joined_top(p, n);
    const Way way = way_of(q, top);
    if (way != kCounts && way != kMasses) return;
    make_table(s, a.shift);
    if (threadIdx.x == 0) s.found = kBins;
    __syncthreads();
    u64 target = q.count;
    locate(s, p.bins + n * kBins, 0, target, way == kMasses ? q.share : -1.0);
    const int found = s.found;
    const Row<T, kPart> row(a, n, part, p.steps, threadIdx.x >> 6);
    const Weights k = weights_of(q, top, s.table);
    const Bins bins{0, kAll, k.top, k.octaves, -1};
    if (way == kCounts && s.base + s.inside > kList) return;
    // a part's tokens are listed here first, and take their places in the row's list at once
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    auto list = [&](u64 code, u64 w) {
        const int to = atomicAdd(&s.listed, 1);
        if (to < kList) {
            s.code[to] = code;
            s.value[to] = w;
        }
    };
    if (way == kCounts) {
        row.tokens(vocab, [&](uint32_t i, float x) {
            const u64 code = code_of(i, x);
            if (bins.of(code, x) <= found) list(code, weight_of(k, x));
        });
    } else {
        sum_runs(p.cells + ((n * p.parts + part) * (kPart / 64) + row.wave) * kCells, row, [&](uint32_t i, float x) -> u64 {
            if (i >= static_cast<uint32_t>(vocab)) return 0; // (beside the row)
            const u64 code = code_of(i, x);
            const int b = bins.of(code, x);
            if (b > found) return 0;
            const u64 w = weight_of(k, x);
            if (b == found) list(code, w);
            return b < found && w >= q.least ? w : 0;
        });
    }
    __syncthreads();
    const int own = s.listed;
    if (threadIdx.x == 0) s.found = atomicAdd(&p.listed[n], own);
    __syncthreads();
    const int to = s.found;
    if (own > kList || to > kList - own) return;         // too long: the row is taken whole
    for (int i = threadIdx.x; i < own; i += kPart) {
        p.code[n * kList + to + i] = s.code[i];
        p.value[n * kList + to + i] = s.value[i];
    }
}

template <class T>
__global__ void __launch_bounds__(kDraw, 4) hawk_sample_draw(const SampleArgs<T> a, const Parts p) {
    constexpr int Waves = kPart / 64, Most = kMostParts * Waves * kCells, Each = Most / kDraw;
    __shared__ Shared<kDraw, true> s;
    __shared__ u64 cells[Most];
    static_assert(Most % kDraw == 0, "whole cells a thread");
    const int tid = threadIdx.x, vocab = static_cast<int>(a.vocab), count = p.parts * Waves * kCells;
    const int64_t n = blockIdx.x;
    const Asked q = asked(a, n);
    const float top = joined_top(p, n);
    if (!drawn(q, top)) {
        u64 first = kAll;
        if (q.heat == 0.0 && top > -INFINITY)
            for (int i = p.parts - 1; i >= 0; --i)
                if (p.tops[n * p.parts + i] == top) first = p.firsts[n * p.parts + i];
        if (tid == 0) answer_plain(a, n, q, top, static_cast<int64_t>(first));
        return;
    }
    const Way way = way_of(q, top);
    make_table(s, a.shift);
    if (tid == 0) s.low = 0, s.found = kBins;
    __syncthreads();
    const Weights k = weights_of(q, top, s.table);
    u64 all, target = q.count, cut = kAll;
    bool whole = way == kNothing;
    if (way == kCounts || way == kMasses) {
        locate(s, p.bins + n * kBins, 0, target, way == kMasses ? q.share : -1.0);
        const int listed = p.listed[n];
        whole = way == kCounts ? s.base + s.inside > kList : listed > kList;
        if (!whole) {
            for (int i = tid; i < listed; i += kDraw) {
                s.code[i] = p.code[n * kList + i];
                s.value[i] = p.value[n * kList + i];
            }
            __syncthreads();
            if (way == kCounts) {
                const u64 at = from_list(s, listed, q, all);
                if (tid == 0) answer_drawn(a, n, q, top, at, all);
                return;
            }
        }
    }
    if (whole) {
        Row<T, kDraw> row(a, n, 0, 0, tid >> 6);
        row.steps = (row.high + kVec<T> * kDraw - 1) / (kVec<T> * kDraw);
        const u64 at = from_whole<true, false>(s, row, vocab, q, top, all);
        if (tid == 0) answer_drawn(a, n, q, top, at, all);
        return;
    }
    for (int c = tid; c < count; c += kDraw) cells[c] = p.cells[n * count + c];
    __syncthreads();
    const Row<T, kPart> first(a, n, 0, p.steps, 0);
    const int run = (p.steps + kCells - 1) / kCells, span = p.steps * 64 * kVec<T>;      // the tokens of a wave's share
    if (way == kMasses) {
        // the list's tokens up to the one that reaches the target join the runs that they are of
        const int listed = p.listed[n];
        u64 before = s.base;
        int rank = tid;
        if (listed <= kFew) {
            if (tid < listed) {
                rank = 0;
                for (int o = 0; o < listed; ++o) {
                    const bool ahead = s.code[o] < s.code[tid];
                    rank += ahead;
                    before += ahead ? s.value[o] : 0;
                }
            }
        } else {
            u64 sum;
            sort<kDraw, false>(s, listed);
            before += list_before(s, listed, sum);
        }
        if (tid < listed) {
            const u64 w = s.value[tid], code = s.code[tid];
            if (before < target) {
                if (before + w >= target || rank + 1 == listed) s.high = code;
                if (w >= q.least) {
                    const int at = static_cast<int>(static_cast<uint32_t>(code)) + first.low;
                    const int wave = at / span;
                    atomicAdd(&cells[wave * kCells + (at - wave * span) / (64 * kVec<T>) / run], w);
                }
            }
        }
        __syncthreads();
        cut = s.high;
    }
    u64 own = 0;
#pragma unroll
    for (int e = 0; e < Each; ++e) own += tid * Each + e < count ? cells[tid * Each + e] : 0;
    u64 before = block_before(s, own, all);
    if (top == INFINITY) all = infinities(q, all);
    const u64 aimed = aim(q.u, all);
    if (before < aimed && before + own >= aimed) {
#pragma unroll
        for (int e = 0; e < Each; ++e) {
            const u64 v = tid * Each + e < count ? cells[tid * Each + e] : 0;
            if (before < aimed && before + v >= aimed) {
                s.found = tid * Each + e;
                s.base = before;
            }
            before += v;
        }
    }
    __syncthreads();
    if (tid < 64) {
        const int found = s.found / kCells;
        const Row<T, kPart> row(a, n, found / Waves, p.steps, found % Waves);
        if (top == INFINITY) {
            go_along(s.low, row, s.found % kCells, s.base, aimed, [](uint32_t, float x) -> u64 { return x == INFINITY; });
        } else {
            go_along(s.low, row, s.found % kCells, s.base, aimed, [&](uint32_t i, float x) -> u64 {
                if (code_of(i, x) > cut) return 0;
                const u64 w = weight_of(k, x);
                return w >= q.least ? w : 0;
            });
        }
    }
    __syncthreads();
    if (tid == 0) answer_drawn(a, n, q, top, s.low, all);
}

// ---- host ----------------------------------------------------------------------------

// A row of up to kList tokens is ranked as it stands (200 rows of 48: 10.6 us, 17 by way of
// the bins).  A lane has eight vectors of a longer row or fewer where the threads allow it;
// of many rows, a unit has several at a time: 512 threads each from 257 rows on.
template <class T, bool Filtered>
void launch(const SampleArgs<T>& a, dim3 grid, hipStream_t stream) {
    const int64_t vectors = (a.vocab + 2 * kVec<T> - 2) / kVec<T>;
    if (a.vocab <= 128) hipLaunchKernelGGL((hawk_sample<T, 64, Filtered, true>), grid, dim3(64), 0, stream, a);
    else if (a.vocab <= kList) hipLaunchKernelGGL((hawk_sample<T, 256, Filtered, true>), grid, dim3(256), 0, stream, a);
    else if (vectors <= 256 * 8) hipLaunchKernelGGL((hawk_sample<T, 256, Filtered, false>), grid, dim3(256), 0, stream, a);
    else if (a.rows > kUnits) hipLaunchKernelGGL((hawk_sample<T, 512, Filtered, false>), grid, dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((hawk_sample<T, 1024, Filtered, false>), grid, dim3(1024), 0, stream, a);
}

// The parts of a row: with fewer rows than half the units, and rows of more than eight
// vectors a lane of a workgroup, as many as give the units four workgroups each, but no
// part below four vectors a lane (64 rows of 131072: 69.5 us, whole 156).
int parts_of(int64_t rows, int64_t vocab, int esize) {
    const int64_t each = 16 / esize, vectors = (vocab + 2 * each - 2) / each;
    if (rows >= kUnits / 2 || vectors <= 256 * 8) return 1;
    int64_t parts = 4 * kUnits / rows;
    parts = parts < kMostParts ? parts : kMostParts;
    return static_cast<int>(parts < vectors / (4 * kPart) ? parts : vectors / (4 * kPart));
}
int size_of(int dtype) { return dtype == HK_F32 ? 4 : 2; }
size_t row_bytes(int parts) {
    return static_cast<size_t>(parts) * (16 + kPart / 64 * kCells * 8) + kBins * 8 + kList * 16 + 16;
}

template <class T>
int sample(const hk_sample_job& j, void* scratch, hipStream_t stream) {
    SampleArgs<T> a;
    a.logits = static_cast<const T*>(j.logits);
    a.u = j.u;
    a.temperature = j.row_temperature;
    a.top_p = j.row_top_p;
    a.min_p = j.row_min_p;
    a.top_k = j.row_top_k;
    a.token = j.token;
    a.logp = j.logp;
    a.rows = j.rows;
    a.vocab = j.vocab;
    a.row_stride = j.row_stride;
    a.temperature_all = j.temperature;
    a.top_p_all = j.top_p;
    a.min_p_all = j.min_p;
    a.top_k_all = j.top_k;
    a.u64bits = j.u64bits;
    a.token64 = j.token64;
    a.shift = 62;
    while (a.shift > 51 || (j.vocab >> (62 - a.shift)) > 1) --a.shift;
    const bool filtered = j.row_temperature || j.row_top_p || j.row_min_p || j.row_top_k || j.top_k > 0 || j.top_p < 1.0 || j.min_p > 0.0;
    const int parts = parts_of(j.rows, j.vocab, sizeof(T));
    if (parts > 1) {
        const int64_t vectors = (j.vocab + 2 * kVec<T> - 2) / kVec<T>;
        Parts p;
        p.parts = parts;
        p.steps = static_cast<int>((vectors + parts * kPart - 1) / (parts * kPart));
        char* room = static_cast<char*>(scratch);
        auto take = [&](int64_t each) { char* at = room; room += each * j.rows; return at; };
        p.bins = reinterpret_cast<u64*>(take(kBins * 8));
        p.cells = reinterpret_cast<u64*>(take(int64_t{parts} * (kPart / 64) * kCells * 8));
        p.code = reinterpret_cast<u64*>(take(kList * 8));
        p.value = reinterpret_cast<u64*>(take(kList * 8));
        p.firsts = reinterpret_cast<u64*>(take(int64_t{parts} * 8));
        p.tops = reinterpret_cast<float*>(take(int64_t{parts} * 8));
        p.listed = reinterpret_cast<int*>(take(16));
        const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(j.rows));
        hipLaunchKernelGGL((hawk_sample_tops<T>), grid, dim3(kPart), 0, stream, a, p);
        hipLaunchKernelGGL((hawk_sample_bins<T>), grid, dim3(kPart), 0, stream, a, p);
        if (filtered) hipLaunchKernelGGL((hawk_sample_keep<T>), grid, dim3(kPart), 0, stream, a, p);
        hipLaunchKernelGGL((hawk_sample_draw<T>), dim3(static_cast<unsigned>(j.rows)), dim3(kDraw), 0, stream, a, p);
    } else {
        const int64_t most = 1 << 20;
        const dim3 grid(static_cast<unsigned>(j.rows < most ? j.rows : most));
        filtered ? launch<T, true>(a, grid, stream) : launch<T, false>(a, grid, stream);
    }
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? HK_OK : hawk_internal::set_hip_error("hawk_sample launch", err);
}

}  // namespace

extern "C" size_t hk_sample_scratch_bytes(const hk_sample_job* job) {
    if (!job || job->rows <= 0 || job->vocab <= 0 || job->vocab > kMostVocab) return 0;
    if (job->dtype != HK_F32 && job->dtype != HK_BF16 && job->dtype != HK_F16) return 0;
    const int parts = parts_of(job->rows, job->vocab, size_of(job->dtype));
    return parts > 1 ? static_cast<size_t>(job->rows) * row_bytes(parts) : 0;
}

extern "C" int hk_sample(const hk_sample_job* job, void* scratch, void* stream) {
    using hawk_internal::set_error;
    if (!job) return set_error(HK_EVALUE, "hk_sample: a job is required");
    if (job->rows < 0 || job->vocab < 0) return set_error(HK_EVALUE, "hk_sample: sizes must be >= 0");
    if (job->vocab > kMostVocab) return set_error(HK_EVALUE, "hk_sample: the vocabulary has at most 2^22 tokens");
    if (job->dtype != HK_F32 && job->dtype != HK_BF16 && job->dtype != HK_F16)
        return set_error(HK_EVALUE, "hk_sample: the logits' element type is 32-bit or 16-bit");
    if (job->rows == 0) return HK_OK;
    if ((job->vocab > 0 && !job->logits) || !job->u) return set_error(HK_EVALUE, "hk_sample: logits and u are required");
    if (hk_sample_scratch_bytes(job) && !scratch) return set_error(HK_EVALUE, "hk_sample: scratch is required for few long rows");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (job->dtype == HK_F32) return sample<float>(*job, scratch, s);
    return job->dtype == HK_BF16 ? sample<bf16>(*job, scratch, s) : sample<f16>(*job, scratch, s);
}
