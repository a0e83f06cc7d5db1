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

// 2^(j / 128), each rounded to 64 bits, made by the workgroup.
constexpr int kTable = 128;

// How a row's weights are taken: exp((x - top) / T) = 2^((x - top) octaves), as a
// multiple of 2^-shift.
struct Weights {
    double top, octaves;
    const double* table;
    int shift;
};

// The weight before it is rounded to a whole one.  The exponent y (in octaves) is split into an octave, a 128th of one from the
// table and a rest r of at most 1/256, whose power is a Taylor polynomial: the
// first term left out is (r ln 2)^5 / 120 < 2^-49.
__device__ __forceinline__ double weight_of(const Weights& k, double x) {
    if (x == k.top) return scaled(1.0, k.shift);
    const double y = (x - k.top) * k.octaves;             // <= 0
    if (!(y > -64.0)) return 0.0;
    const double shifted = __builtin_fma(y, static_cast<double>(kTable), 0x1.8p52);
    const int n = static_cast<int>(__builtin_bit_cast(uint64_t, shifted));
    const double r = __builtin_fma(shifted - 0x1.8p52, -1.0 / kTable, y) * 0.6931471805599453094;
    double p = __builtin_fma(r, 1.0 / 24.0, 1.0 / 6.0);
    p = __builtin_fma(r, p, 0.5);
    p = __builtin_fma(r, p, 1.0);
    p = __builtin_fma(r, p, 1.0);
    return scaled(p * k.table[n & (kTable - 1)], (n >> 7) + k.shift);
}
__device__ __forceinline__ u64 whole(double w) {
    return __builtin_bit_cast(uint64_t, w + 0x1p52) & 0xfffffffffffffull;
}

// A logit's place in descending order: smaller is higher.  Both zeros are one.
__device__ __forceinline__ uint32_t place_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}

template <int NT>
struct Shared {
    double table[kTable];
    u64 mass[kBins], code[kList], value[kList];
    uint32_t count[kBins];
    u64 waves[16], bin_base, low, high, cut;
    float tops[16];
    int found, listed, bad;
};

__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
// The sum of the lanes before this one.
__device__ __forceinline__ u64 wave_before(u64 v) {
    u64 sum = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 t = __shfl_up(sum, d);
        if (static_cast<int>(threadIdx.x & 63) >= d) sum += t;
    }
    return sum - v;
}

// A row, read by NT threads: wave w has the vectors [w, w + 1) * per of it, so the
// waves' parts follow each other by index.
template <class T, int NT>
struct Row {
    const T* at;           // the row's address less its lead, 16-byte aligned
    int low;               // the row's first position
    int64_t high;          // past its last
    int64_t first, end;    // this wave's vectors
    template <class F> __device__ __forceinline__ void each(F&& f) const {
        constexpr int V = kVec<T>;
        for (int64_t v = first; v < end; v += 64) {
            const int64_t p = (v + (threadIdx.x & 63)) * V;
            float x[V];
            if (p >= low && p + V <= high) {
                load<T, V>(at + p, x);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) x[j] = p + j >= low && p + j < high ? static_cast<float>(at[p + j]) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (p + j >= low && p + j < high) f(static_cast<uint32_t>(p + j - low), x[j]);
        }
    }
};

// The code of the last token of a prefix: of those with code <= limit, in order, the
// first at which the running sum (of 1 each, or of the weights) is at least the
// target.  With the weights the target is `share` of their whole sum.
template <class T, int NT, bool Mass>
__device__ u64 select(Shared<NT>& s, const Row<T, NT>& row, const Weights& k, u64 limit, u64 target, double share) {
    const int tid = threadIdx.x, wave = tid >> 6;
    u64 base = 0, low = 0, high = limit;
    int shift = -1;                                      // -1: bins of a 64th of an octave below the highest logit
    auto bin_of = [&](uint32_t i, float x, u64& code) -> int {
        code = static_cast<u64>(place_of(x)) << 32 | i;
        if (code < low || code > high) return -1;
        if (shift >= 0) return static_cast<int>((code - low) >> shift);
        const double d = x == k.top ? 0.0 : (k.top - static_cast<double>(x)) * k.octaves * 64.0;
        return d < kBins - 1 ? static_cast<int>(d) : kBins - 1;
    };
    for (;;) {
        for (int b = tid; b < kBins; b += NT) {
            s.mass[b] = 0;
            s.count[b] = 0;
        }
        if (tid == 0) s.listed = 0, s.low = kAll, s.high = 0, s.found = kBins;
        __syncthreads();
        row.each([&](uint32_t i, float x) {
            u64 code;
            const int b = bin_of(i, x, code);
            if (b < 0) return;
            atomicAdd(&s.count[b], 1u);
            if (Mass) atomicAdd(&s.mass[b], whole(weight_of(k, x)));
        });
        __syncthreads();
        // the first bin whose running sum reaches the target
        constexpr int Each = kBins / NT;
        u64 own = 0;
#pragma unroll
        for (int b = 0; b < Each; ++b) own += Mass ? s.mass[tid * Each + b] : s.count[tid * Each + b];
        u64 before = wave_before(own);
        if ((tid & 63) == 63) s.waves[wave] = before + own;
        __syncthreads();
        u64 all = 0;
        for (int w = 0; w < NT / 64; ++w) {
            if (w == wave) before += all;
            all += s.waves[w];
        }
        if (Mass && share >= 0.0) {
            const double want = ceil(share * static_cast<double>(all));
            target = want < 1.0 ? 1 : static_cast<u64>(want);
            if (target > all) target = all;
            share = -1.0;
        }
        before += base;
        if (before < target && before + own >= target) {
#pragma unroll
            for (int b = 0; b < Each; ++b) {
                const u64 v = Mass ? s.mass[tid * Each + b] : s.count[tid * Each + b];
                if (before < target && before + v >= target) {
                    s.found = tid * Each + b;
                    s.bin_base = before;
                }
                before += v;
            }
        }
        __syncthreads();
        const int found = s.found;
        if (found >= kBins) return limit;                // less than the target in all: everything is kept
        base = s.bin_base;
        const bool few = s.count[found] <= kList;
        u64 least = kAll, most = 0;
        row.each([&](uint32_t i, float x) {
            u64 code;
            if (bin_of(i, x, code) != found) return;
            if (few) {
                const int at = atomicAdd(&s.listed, 1);
                s.code[at] = code;
                s.value[at] = Mass ? whole(weight_of(k, x)) : 1;
            } else {
                least = code < least ? code : least;
                most = code > most ? code : most;
            }
        });
        if (few) {
            __syncthreads();
            const int n = s.listed;
            for (int i = tid; i < n; i += NT) {
                const u64 code = s.code[i], value = s.value[i];
                u64 upto = base;
                for (int o = 0; o < n; ++o) upto += s.code[o] <= code ? s.value[o] : 0;
                if (upto >= target && upto - value < target) s.cut = code;
            }
            __syncthreads();
            const u64 cut = s.cut;
            __syncthreads();
            return cut;
        }
        if (least != kAll) {
            atomicMin(&s.low, least);
            atomicMax(&s.high, most);
        }
        __syncthreads();
        low = s.low;
        high = s.high;
        shift = 0;
        while ((high - low) >> shift >= kBins) ++shift;
        __syncthreads();
    }
}

template <class T, int NT>
__global__ void __launch_bounds__(NT) hawk_sample(const SampleArgs<T> a) {
    constexpr int V = kVec<T>, Waves = NT / 64;
    __shared__ Shared<NT> s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int j = tid; j < kTable; j += NT) s.table[j] = exp2(static_cast<double>(j) / kTable);
    for (int64_t n = blockIdx.x; n < a.rows; n += gridDim.x) {
        __syncthreads();
        const T* from = a.logits + n * a.row_stride;
        Row<T, NT> row;
        row.low = static_cast<int>(reinterpret_cast<uintptr_t>(from) % 16 / sizeof(T));
        row.at = from - row.low;
        row.high = row.low + a.vocab;
        const int64_t vectors = (row.high + V - 1) / V, per = ((vectors + Waves - 1) / Waves + 63) / 64 * 64;
        row.first = wave * per;
        row.end = row.first + per < vectors ? row.first + per : vectors;
        const double T_row = a.temperature ? static_cast<double>(a.temperature[n]) : a.temperature_all;
        const double u = a.u64bits ? static_cast<const double*>(a.u)[n] : static_cast<double>(static_cast<const float*>(a.u)[n]);

        // the highest logit, and whether one is a NaN
        float m = -INFINITY;
        bool bad = false;
        row.each([&](uint32_t, float x) {
            m = fmaxf(m, x);
            bad |= !(x == x);
        });
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
        if (tid == 0) s.bad = 0, s.low = kAll;
        __syncthreads();
        if (lane == 0) s.tops[wave] = m;
        if (bad) s.bad = 1;
        __syncthreads();
        for (int w = 0; w < Waves; ++w) m = fmaxf(m, s.tops[w]);
        const double top = static_cast<double>(m);
        int64_t token = -1;
        float logp = 0.0f;
        if (s.bad || !(T_row >= 0.0) || !(u == u)) {
            logp = NAN;
        } else if (m == -INFINITY) {
            logp = -INFINITY;
        } else if (T_row == 0.0) {
            u64 first = kAll;
            row.each([&](uint32_t i, float x) { if (x == m && i < first) first = i; });
            if (first != kAll) atomicMin(&s.low, first);
            __syncthreads();
            token = static_cast<int64_t>(s.low);
        } else {
            const Weights k{top, 1.4426950408889634074 / T_row, s.table, a.shift};
            const double top_p = a.top_p ? static_cast<double>(a.top_p[n]) : a.top_p_all;
            const double low_p = a.min_p ? static_cast<double>(a.min_p[n]) : a.min_p_all;
            // no weight is above 1: a larger min_p leaves the highest alone
            const int64_t top_k = low_p > 1.0 ? 1 : a.top_k ? static_cast<int64_t>(a.top_k[n]) : a.top_k_all;
            u64 cut = kAll;
            if (top_k > 0 && top_k < a.vocab)
                cut = select<T, NT, false>(s, row, k, cut, static_cast<u64>(top_k), -1.0);
            if (top_p < 1.0)
                cut = select<T, NT, true>(s, row, k, cut, 0, top_p > 0.0 ? top_p : 0.0);
            const double least = low_p > 0.0 && low_p <= 1.0 ? scaled(low_p, a.shift) : 0.0;
            auto kept = [&](uint32_t i, float x) -> u64 {
                if ((static_cast<u64>(place_of(x)) << 32 | i) > cut) return 0;
                const double w = weight_of(k, x);
                return w >= least ? whole(w) : 0;
            };
            u64 sum = 0;
            row.each([&](uint32_t i, float x) { sum += kept(i, x); });
            sum = wave_sum(sum);
            if (lane == 0) s.waves[wave] = sum;
            if (tid == 0) s.low = 0;
            __syncthreads();
            u64 all = 0, before = 0;
            for (int w = 0; w < Waves; ++w) {
                if (w == wave) before = all;
                all += s.waves[w];
            }
            // the first running sum above u * all: at least one whole number above its floor
            const double want = u * static_cast<double>(all);
            u64 target = want >= 0.0 ? (want < 0x1p63 ? static_cast<u64>(want) : kAll - 1) + 1 : 1;
            if (target > all) target = all;
            if (before < target && before + sum >= target) {         // one wave goes along its part
                for (int64_t v = row.first; v < row.end; v += 64) {
                    const int64_t p = (v + lane) * V;
                    u64 w[V], own = 0;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const bool real = p + j >= row.low && p + j < row.high;
                        w[j] = real ? kept(static_cast<uint32_t>(p + j - row.low), static_cast<float>(row.at[p + j])) : 0;
                        own += w[j];
                    }
                    const u64 step = wave_sum(own);
                    if (before + step >= target) {
                        u64 upto = before + wave_before(own);
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            if (upto < target && upto + w[j] >= target) s.low = static_cast<u64>(p + j - row.low);
                            upto += w[j];
                        }
                        break;
                    }
                    before += step;
                }
            }
            __syncthreads();
            token = static_cast<int64_t>(s.low);
            const float x = from[token];
            logp = static_cast<float>((x == m ? 0.0 : (static_cast<double>(x) - top) / T_row) -
                                      log(scaled(static_cast<double>(all), -a.shift)));
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
    if (j.vocab <= 4096) hipLaunchKernelGGL((hawk_sample<T, 256>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((hawk_sample<T, 1024>), grid, dim3(1024), 0, stream, a);
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
