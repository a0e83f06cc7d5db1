// hawk_dropout.hip — dropout whose mask is never stored: a counter-based
// generator gives an element's random bits from its index, so the forward and
// the derivative compute the same mask from (seed, offset).
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011): ten rounds of two
// 32 x 32 -> 64-bit products over four words.  One evaluation gives eight
// 16-bit numbers, so a mask's rate is a multiple of 2^-16.

#include "hawk_core.h"
#include "hawk_internal.h"
#include "hawk_vec.h"

#include <hip/hip_runtime.h>
#include <cstdint>
#include <string>

namespace {

using namespace hawk_vec;

constexpr int kThreads = 256;
constexpr int kNumbers = 8;      // 16-bit numbers of one evaluation

struct Words { uint32_t w[4]; };

__device__ __forceinline__ Words philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p = static_cast<uint64_t>(c0) * 0xD2511F53u, q = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
        c0 = static_cast<uint32_t>(q >> 32) ^ c1 ^ k0;
        c1 = static_cast<uint32_t>(q);
        c2 = static_cast<uint32_t>(p >> 32) ^ c3 ^ k1;
        c3 = static_cast<uint32_t>(p);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Words{{c0, c1, c2, c3}};
}

struct DropArgs {
    const int64_t* offset_cell;
    uint64_t seed, offset;
    int64_t rows, cols, x_stride, residual_stride, y_stride;
    uint32_t cut;
};

__device__ __forceinline__ Words numbers(const DropArgs& a, uint64_t offset, int64_t g) {
    return philox(static_cast<uint32_t>(g), static_cast<uint32_t>(g >> 32), static_cast<uint32_t>(offset),
                  static_cast<uint32_t>(offset >> 32), static_cast<uint32_t>(a.seed),
                  static_cast<uint32_t>(a.seed >> 32));
}
__device__ __forceinline__ uint64_t offset_of(const DropArgs& a) {
    return a.offset + (a.offset_cell ? static_cast<uint64_t>(*a.offset_cell) : 0);
}
template <class A>
__device__ __forceinline__ A dropped(const DropArgs& a, const Words& u, int j, A x, A factor) {
    const uint32_t word = j < 4 ? (j < 2 ? u.w[0] : u.w[1]) : (j < 6 ? u.w[2] : u.w[3]);
    const uint32_t number = j & 1 ? word >> 16 : word & 0xffffu;
    return number >= a.cut ? x * factor : A(0);
}

// Eight elements of one counter as vectors: kSets counters a thread, whose loads
// are issued together.  A row is whole counters (Rows), or the array one run.
constexpr int kSets = 2;
template <class T, bool Residual, bool Rows>
__global__ void __launch_bounds__(kThreads) hawk_dropout(const DropArgs a, const T* x, const T* residual, T* y,
                                                         const Acc<T> factor) {
    typedef Acc<T> A;
    constexpr int V = sizeof(T) == 8 ? 2 : sizeof(T) == 4 ? 4 : 8;
    constexpr bool Stream = sizeof(T) == 2;
    const int64_t groups = Rows ? a.rows * (a.cols / kNumbers) : a.cols / kNumbers;
    const int64_t g0 = static_cast<int64_t>(blockIdx.x) * (kThreads * kSets) + threadIdx.x;
    const int64_t per_row = a.cols / kNumbers;
    const uint64_t offset = offset_of(a);
    Raw<T, V> in[kSets][kNumbers / V], add[kSets][kNumbers / V];
    int64_t row[kSets], c[kSets];
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
        const int64_t g = g0 + s * kThreads;
        row[s] = Rows ? g / per_row : 0;
        c[s] = (Rows ? g - row[s] * per_row : g) * kNumbers;
        if (g >= groups) continue;
#pragma unroll
        for (int j = 0; j < kNumbers / V; ++j) {
            in[s][j] = load_raw<T, V, Stream>(x + row[s] * a.x_stride + c[s] + j * V);
            if (Residual) add[s][j] = load_raw<T, V, Stream>(residual + row[s] * a.residual_stride + c[s] + j * V);
        }
    }
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
        const int64_t g = g0 + s * kThreads;
        if (g >= groups) continue;
        const Words u = numbers(a, offset, g);
#pragma unroll
        for (int j = 0; j < kNumbers / V; ++j) {
            A out[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                out[v] = dropped(a, u, j * V + v, widen<T, V>(in[s][j], v), factor);
                if (Residual) out[v] += widen<T, V>(add[s][j], v);
            }
            store<T, V, Stream>(y + row[s] * a.y_stride + c[s] + j * V, out);
        }
    }
    if constexpr (!Rows) {                // the last counter's elements, of an array that is no whole counters
        const int64_t i = groups * kNumbers + threadIdx.x;
        if (blockIdx.x == 0 && i < a.cols) {
            A v = dropped(a, numbers(a, offset, groups), threadIdx.x, static_cast<A>(x[i]), factor);
            if (Residual) v += static_cast<A>(residual[i]);
            y[i] = static_cast<T>(v);
        }
    }
}

// Rows apart whose counters run on from one row into the next: a thread's eight
// elements of a row begin at any half of a counter, so it takes two of them and
// shifts.  (16384 rows of 4093 bfloat16 elements, 4096 apart, with a residual: 79 us;
// 222 an element at a time.)
template <class T, bool Residual>
__global__ void __launch_bounds__(kThreads) hawk_dropout_apart(const DropArgs a, const T* x, const T* residual, T* y,
                                                               const Acc<T> factor) {
    typedef Acc<T> A;
    const int64_t per_row = (a.cols + kNumbers - 1) / kNumbers;
    const int64_t v = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (v >= a.rows * per_row) return;
    const int64_t row = v / per_row, c = (v - row * per_row) * kNumbers;
    const int64_t left = a.cols - c, i = row * a.cols + c;
    x += row * a.x_stride + c;
    y += row * a.y_stride + c;
    if (Residual) residual += row * a.residual_stride + c;
    A in[kNumbers], add[kNumbers];
    if (left >= kNumbers) {
        load<T, kNumbers>(x, in);
        if (Residual) load<T, kNumbers>(residual, add);
    } else {
#pragma unroll
        for (int j = 0; j < kNumbers; ++j) {
            in[j] = j < left ? static_cast<A>(x[j]) : A(0);
            add[j] = Residual && j < left ? static_cast<A>(residual[j]) : A(0);
        }
    }
    const uint64_t offset = offset_of(a);
    const int shift = static_cast<int>(i % kNumbers);        // halves of the first counter that are not this thread's
    const Words one = numbers(a, offset, i / kNumbers), two = numbers(a, offset, i / kNumbers + 1);
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) { w[j] = one.w[j]; w[4 + j] = two.w[j]; }
    if (shift & 4) {
#pragma unroll
        for (int j = 0; j < 6; ++j) w[j] = w[j + 2];
    }
    if (shift & 2) {
#pragma unroll
        for (int j = 0; j < 5; ++j) w[j] = w[j + 1];
    }
    Words u;
#pragma unroll
    for (int j = 0; j < 4; ++j) u.w[j] = shift & 1 ? w[j] >> 16 | w[j + 1] << 16 : w[j];
    A out[kNumbers];
#pragma unroll
    for (int j = 0; j < kNumbers; ++j) {
        out[j] = dropped(a, u, j, in[j], factor);
        if (Residual) out[j] += add[j];
    }
    if (left >= kNumbers) {
        store<T, kNumbers>(y, out);
    } else {
#pragma unroll
        for (int j = 0; j < kNumbers; ++j)
            if (j < left) y[j] = static_cast<T>(out[j]);
    }
}

template <class T>
int dropout(const hk_dropout_job& j, hipStream_t stream) {
    const int64_t n = j.rows * j.cols;
    if (n == 0) return HK_OK;
    const bool whole = j.cols % kNumbers == 0, vectors = j.rows == 1 || whole;
    const int64_t groups = vectors ? (n + kNumbers - 1) / kNumbers : j.rows * ((j.cols + kNumbers - 1) / kNumbers);
    const int64_t per = vectors ? kThreads * kSets : kThreads;
    const int64_t blocks = (groups + per - 1) / per;
    if (blocks > UINT32_MAX / kThreads) return hawk_internal::set_error(HK_EVALUE, "hk_dropout: the planes exceed the grid limit");
    const DropArgs a{j.offset_cell, j.seed, j.offset, j.rows, j.cols, j.x_stride, j.residual_stride, j.y_stride,
                     static_cast<uint32_t>(j.cut)};
    const Acc<T> factor = j.cut < 65536 ? Acc<T>(65536) / Acc<T>(65536 - j.cut) : Acc<T>(0);
    const T *x = static_cast<const T*>(j.x), *residual = static_cast<const T*>(j.residual);
    T* y = static_cast<T*>(j.y);
    const dim3 grid(static_cast<unsigned>(blocks)), block(kThreads);
    if (!vectors && residual) hipLaunchKernelGGL((hawk_dropout_apart<T, true>), grid, block, 0, stream, a, x, residual, y, factor);
    else if (!vectors) hipLaunchKernelGGL((hawk_dropout_apart<T, false>), grid, block, 0, stream, a, x, residual, y, factor);
    else if (j.rows == 1 && residual) hipLaunchKernelGGL((hawk_dropout<T, true, false>), grid, block, 0, stream, a, x, residual, y, factor);
    else if (j.rows == 1) hipLaunchKernelGGL((hawk_dropout<T, false, false>), grid, block, 0, stream, a, x, residual, y, factor);
    else if (residual) hipLaunchKernelGGL((hawk_dropout<T, true, true>), grid, block, 0, stream, a, x, residual, y, factor);
    else hipLaunchKernelGGL((hawk_dropout<T, false, true>), grid, block, 0, stream, a, x, residual, y, factor);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? HK_OK : hawk_internal::set_hip_error("hawk_dropout launch", err);
}

}  // namespace

extern "C" int hk_dropout(const hk_dropout_job* job, void* stream) {
    using hawk_internal::set_error;
    if (!job) return set_error(HK_EVALUE, "hk_dropout: a job is required");
    if (job->rows < 0 || job->cols < 0) return set_error(HK_EVALUE, "hk_dropout: sizes must be >= 0");
    if (job->cut < 0 || job->cut > 65536) return set_error(HK_EVALUE, "hk_dropout: cut must be in [0, 65536]");
    if (job->cols > 0 && job->rows > INT64_MAX / 16 / job->cols)
        return set_error(HK_EVALUE, "hk_dropout: the planes exceed the grid limit");
    if (job->rows > 0 && job->cols > 0 && (!job->x || !job->y))
        return set_error(HK_EVALUE, "hk_dropout: x and y are required");
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (job->dtype) {
        case HK_F32: return dropout<float>(*job, s);
        case HK_F64: return dropout<double>(*job, s);
        case HK_BF16: return dropout<bf16>(*job, s);
        case HK_F16: return dropout<f16>(*job, s);
    }
    return set_error(HK_EVALUE, "hk_dropout: unknown element type");
}
