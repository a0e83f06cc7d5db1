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
// changes a bit.

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
__device__ __forceinline__ float placed(uint32_t at) {
    return __builtin_bit_cast(float, at & 0x80000000u ? at : ~at & 0x7fffffffu);
}

// The sum of a wave's numbers, in every lane, and of the lanes before this one.
__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ u64 wave_before(u64 v) {
    u64 sum = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 t = __shfl_up(sum, d);
        if (static_cast<int>(threadIdx.x & 63) >= d) sum += t;
    }
    return sum - v;
}

constexpr int kFew = 256;                  // candidates that are ranked by counting
constexpr int kCells = 16;                 // of a wave: runs of its part of a row
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

    __device__ __forceinline__ int position(int i) const {
        return (begin + (static_cast<int>(threadIdx.x >> 6) * steps + i) * 64 + static_cast<int>(threadIdx.x & 63)) * kVec<T>;
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
        constexpr int V = kVec<T>, kAhead = 4;
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

// Fills the bins with the tokens' weights (or 1 each) and finds the first at which their
// running sum from `base` reaches the target: s.found (kBins: none), s.base the sum
// before it, s.inside its own.  With share >= 0 the target is that share of the sum.
template <class T, int NT>
__device__ __forceinline__ void fill(Shared<NT, true>& s, const Row<T, NT>& row, int vocab, const Weights& k, const Bins& bins, bool mass, u64 base,
                     u64& target, double share) {
    for (int b = threadIdx.x; b < kBins; b += NT) s.bins[b] = 0;
    if (threadIdx.x == 0) s.found = kBins, s.listed = 0, s.low = kAll, s.high = 0;
    __syncthreads();
    u64 rest = 0;                                         // the last bin's, which may have most of a row (what is barred)
    row.tokens(vocab, [&](uint32_t i, float x) {
        const int b = bins.of(code_of(i, x), x);
        if (b < 0) return;
        if (mass) {
            const u64 w = weight_of(k, x);
            if (b == kBins - 1) rest += w;
            else atomicAdd(&s.bins[b], w);
        } else {
            if (b == kBins - 1) ++rest;
            else atomicAdd(reinterpret_cast<uint32_t*>(&s.bins[b]), 1u);
        }
    });
    rest = wave_sum(rest);
    if ((threadIdx.x & 63) == 0 && rest) atomicAdd(&s.bins[kBins - 1], rest);
    __syncthreads();
    constexpr int Each = kBins / NT;
    u64 own = 0, all;
#pragma unroll
    for (int b = 0; b < Each; ++b) own += s.bins[threadIdx.x * Each + b];
    u64 before = block_before(s, own, all) + base;
    if (share >= 0.0) {
        const double want = ceil(share * static_cast<double>(all));
        target = want < 1.0 ? 1 : static_cast<u64>(want);
        if (target > all) target = all;
    }
    if (before < target && before + own >= target) {
#pragma unroll
        for (int b = 0; b < Each; ++b) {
            const u64 v = s.bins[threadIdx.x * Each + b];
            if (before < target && before + v >= target) {
                s.found = threadIdx.x * Each + b;
                s.base = before;
                s.inside = v;
            }
            before += v;
        }
    }
    __syncthreads();
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
        fill(s, row, vocab, k, bins, mass, base, target, share);
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
    double u, share;           // share: top_p, or -1 where it keeps everything
    u64 count, least;          // count: top_k, or kAll; least: the least weight that min_p keeps
};

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
    if (q.share >= 0.0) {
        const double want = ceil(q.share * static_cast<double>(all));
        target = want < 1.0 ? 1 : static_cast<u64>(want);
    }
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

// The token drawn from those that `kept` (of an index and a number) gives a weight: the
// waves' runs are summed, and the wave that has the one that is aimed at goes along it.
// `some` says of the sum of all how much of it, from the first index on, there is to draw.
template <class T, int NT, class F, class G>
__device__ __forceinline__ u64 from_row(Sums<NT>& s, const Row<T, NT>& row, double u, F&& weight, G&& some, u64& all) {
    constexpr int V = kVec<T>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, run = (row.steps + kCells - 1) / kCells;
    auto kept = [&](int first, const Raw<T, V>& v, int j) -> u64 { return weight(static_cast<uint32_t>(first + j), widen<T, V>(v, j)); };
    u64 total = 0;
#pragma unroll 1
    for (int c = 0, i = 0; i < row.steps; ++c) {
        const int end = i + run < row.steps ? i + run : row.steps;
        u64 sum = 0;
        row.each(i, end, [&](int first, const Raw<T, V>& v) {
#pragma unroll
            for (int j = 0; j < V; ++j) sum += kept(first, v, j);
        });
        sum = wave_sum(sum);
        if (lane == 0) s.cells[wave * kCells + c] = sum;
        total += sum;
        i = end;
    }
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
        const int end = (c + 1) * run < row.steps ? (c + 1) * run : row.steps;
#pragma unroll 1
        for (int i = c * run; i < end; ++i) {
            const Raw<T, V> v = row.vector(row.position(i));
            const int first = row.position(i) - row.low;
            u64 w[V], own = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) own += w[j] = kept(first, v, j);
            const u64 step = wave_sum(own);
            if (before + step >= target) {
                u64 upto = before + wave_before(own);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (upto < target && upto + w[j] >= target) s.low = static_cast<u64>(first + j);
                    upto += w[j];
                }
                break;
            }
            before += step;
        }
    }
    __syncthreads();
    return s.low;
}

// Filtered: a row may have filters.  Listed: every row fits the list.
template <class T, int NT, bool Filtered, bool Listed>
__global__ void __launch_bounds__(NT, 4) hawk_sample(const SampleArgs<T> a) {
    constexpr int V = kVec<T>, Waves = NT / 64;
    __shared__ Shared<NT, Filtered> s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, vocab = static_cast<int>(a.vocab);
    for (int j = tid; j < kTable; j += NT) s.table[j] = scaled(exp2(static_cast<double>(j) / kTable), a.shift);
    for (int64_t n = blockIdx.x; n < a.rows; n += gridDim.x) {
        __syncthreads();
        const T* from = a.logits + n * a.row_stride;
        Row<T, NT> row;
        row.low = static_cast<int>(reinterpret_cast<uintptr_t>(from) % 16 / sizeof(T));
        row.at = from - row.low;
        row.high = row.low + vocab;
        row.begin = 0;
        row.steps = static_cast<int>((row.high + V * NT - 1) / (V * NT));
        const double heat = a.temperature ? static_cast<double>(a.temperature[n]) : a.temperature_all;
        const double u = a.u64bits ? static_cast<const double*>(a.u)[n] : static_cast<double>(static_cast<const float*>(a.u)[n]);

        // the highest logit, and whether one is a NaN
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
        if (tid == 0) s.bad = 0, s.low = vocab > 0 ? vocab - 1 : 0;
        __syncthreads();
        if (lane == 0) s.tops[wave] = m;
        if (bad) s.bad = 1;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < Waves; ++w) m = fmaxf(m, s.tops[w]);
        int64_t token = -1;
        float logp = 0.0f;
        if (s.bad || !(heat >= 0.0) || !(u == u)) {
            logp = NAN;
        } else if (m == -INFINITY) {
            logp = -INFINITY;
        } else if (heat == 0.0) {
            u64 first = kAll;
            row.tokens(vocab, [&](uint32_t i, float x) { if (x == m && i < first) first = i; });
            if (first != kAll) atomicMin(&s.low, first);
            __syncthreads();
            token = static_cast<int64_t>(s.low);
        } else {
            const bool infinite = m == INFINITY;
            const Weights k{static_cast<double>(m), fmin(1.4426950408889634074 / heat, 1e300), s.table};
            const double top_p = a.top_p ? static_cast<double>(a.top_p[n]) : a.top_p_all;
            const double low_p = a.min_p ? static_cast<double>(a.min_p[n]) : a.min_p_all;
            // no weight is above 1: a larger min_p leaves the highest alone
            const int64_t top_k = low_p > 1.0 ? 1 : a.top_k ? static_cast<int64_t>(a.top_k[n]) : a.top_k_all;
            Asked q;
            q.u = u;
            q.share = top_p < 1.0 ? fmax(top_p, 0.0) : -1.0;
            q.count = top_k > 0 && top_k < a.vocab ? static_cast<u64>(top_k) : kAll;
            q.least = low_p > 0.0 && low_p <= 1.0 ? static_cast<u64>(ceil(scaled(low_p, a.shift))) : 0;
            u64 cut = kAll, all, at;
            const bool every = q.count == kAll && q.share < 0.0 && q.least == 0;
            auto whole = [](u64 sum) { return sum; };
            if (infinite) {                              // the infinities share the whole, the first of them what is kept
                at = from_row(s, row, q.u, [](uint32_t, float x) -> u64 { return x == INFINITY; }, [&](u64 sum) {
                    const u64 some = q.count < sum ? q.count : sum;
                    const double part = q.share < 0.0 ? 1e300 : ceil(q.share * static_cast<double>(some));
                    return part < 1.0 ? 1 : part < static_cast<double>(some) ? static_cast<u64>(part) : some;
                }, all);
                all <<= a.shift;
            } else if (!Filtered || every) {
                at = from_row(s, row, q.u, [&](uint32_t, float x) { return weight_of(k, x); }, whole, all);
            } else if constexpr (Filtered) {
                bool listed = Listed;
                if (Listed) {
                    row.tokens(vocab, [&](uint32_t i, float x) {
                        s.code[i] = code_of(i, x);
                        s.value[i] = weight_of(k, x);
                    });
                    if (tid == 0) s.listed = vocab;
                } else if (q.count <= kList) {
                    // the tokens down to the bin that has the last of the top_k
                    u64 target = q.count;
                    const Bins bins{0, kAll, k.top, k.octaves, -1};
                    fill(s, row, vocab, k, bins, false, 0, target, -1.0);
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
                if (listed) {
                    at = from_list(s, s.listed, q, all);
                } else {
                    for (int f = 0; f < 2; ++f) {        // top_k, then top_p of what it keeps
                        if (f == 0 ? q.count == kAll : q.share < 0.0) continue;
                        cut = last_of(s, row, vocab, k, cut, f == 1, q.count, f == 0 ? -1.0 : q.share);
                    }
                    at = from_row(s, row, q.u, [&](uint32_t i, float x) -> u64 {
                        if (code_of(i, x) > cut) return 0;
                        const u64 w = weight_of(k, x);
                        return w >= q.least ? w : 0;
                    }, whole, all);
                }
            }
            token = at < a.vocab ? static_cast<int64_t>(at) : a.vocab - 1;
            const float x = static_cast<float>(from[token]);
            logp = static_cast<float>((infinite ? 0.0 : (static_cast<double>(x) - k.top) / heat) - log(scaled(static_cast<double>(all), -a.shift)));
        }
        if (tid == 0) {
            if (a.token) {
                if (a.token64) static_cast<int64_t*>(a.token)[n] = token;
                else static_cast<int32_t*>(a.token)[n] = static_cast<int32_t>(token);
            }
            if (a.logp) a.logp[n] = logp;
        }
    }
}

// A lane has eight vectors of a row or fewer where the threads allow it; of many rows, a
// unit has several at a time.
template <class T, bool Filtered>
void launch(const SampleArgs<T>& a, dim3 grid, hipStream_t stream) {
    const int64_t vectors = (a.vocab + 2 * kVec<T> - 2) / kVec<T>;
    if (a.vocab <= 128) hipLaunchKernelGGL((hawk_sample<T, 64, Filtered, true>), grid, dim3(64), 0, stream, a);
    else if (a.vocab <= kList) hipLaunchKernelGGL((hawk_sample<T, 256, Filtered, true>), grid, dim3(256), 0, stream, a);
    else if (vectors <= 256 * 8) hipLaunchKernelGGL((hawk_sample<T, 256, Filtered, false>), grid, dim3(256), 0, stream, a);
    else if (a.rows > 2 * 256) hipLaunchKernelGGL((hawk_sample<T, 512, Filtered, false>), grid, dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((hawk_sample<T, 1024, Filtered, false>), grid, dim3(1024), 0, stream, a);
}

template <class T>
int sample(const hk_sample_job& j, hipStream_t stream) {
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
    const int64_t most = 1 << 20;
    const dim3 grid(static_cast<unsigned>(j.rows < most ? j.rows : most));
    const bool filtered = j.row_temperature || j.row_top_p || j.row_min_p || j.row_top_k || j.top_k > 0 || j.top_p < 1.0 || j.min_p > 0.0;
    filtered ? launch<T, true>(a, grid, stream) : launch<T, false>(a, grid, stream);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? HK_OK : hawk_internal::set_hip_error("hawk_sample launch", err);
}

}  // namespace

extern "C" size_t hk_sample_scratch_bytes(const hk_sample_job*) { return 0; }

extern "C" int hk_sample(const hk_sample_job* job, void* scratch, void* stream) {
    using hawk_internal::set_error;
    (void)scratch;
    if (!job) return set_error(HK_EVALUE, "hk_sample: a job is required");
    if (job->rows < 0 || job->vocab < 0) return set_error(HK_EVALUE, "hk_sample: sizes must be >= 0");
    if (job->vocab > kMostVocab) return set_error(HK_EVALUE, "hk_sample: the vocabulary has at most 2^22 tokens");
    if (job->dtype != HK_F32 && job->dtype != HK_BF16 && job->dtype != HK_F16)
        return set_error(HK_EVALUE, "hk_sample: the logits' element type is 32-bit or 16-bit");
    if (job->rows == 0) return HK_OK;
    if ((job->vocab > 0 && !job->logits) || !job->u) return set_error(HK_EVALUE, "hk_sample: logits and u are required");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (job->dtype == HK_F32) return sample<float>(*job, s);
    return job->dtype == HK_BF16 ? sample<bf16>(*job, s) : sample<f16>(*job, s);
}
