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

// One thread takes the eight elements of one counter.
template <class T>
__global__ void __launch_bounds__(kThreads) hawk_dropout(const DropArgs a, const T* x, const T* residual, T* y) {
    const int64_t n = a.rows * a.cols, groups = (n + kNumbers - 1) / kNumbers;
    const int64_t g = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (g >= groups) return;
    const uint64_t offset = a.offset + (a.offset_cell ? static_cast<uint64_t>(*a.offset_cell) : 0);
    const Words u = philox(static_cast<uint32_t>(g), static_cast<uint32_t>(g >> 32), static_cast<uint32_t>(offset),
                           static_cast<uint32_t>(offset >> 32), static_cast<uint32_t>(a.seed),
                           static_cast<uint32_t>(a.seed >> 32));
    const Acc<T> factor = a.cut < 65536u ? Acc<T>(65536) / Acc<T>(65536u - a.cut) : Acc<T>(0);
    for (int j = 0; j < kNumbers; ++j) {
        const int64_t i = g * kNumbers + j;
        if (i >= n) break;
        const int64_t row = i / a.cols, c = i - row * a.cols;
        const uint32_t number = j & 1 ? u.w[j / 2] >> 16 : u.w[j / 2] & 0xffffu;
        Acc<T> v = number >= a.cut ? static_cast<Acc<T>>(x[row * a.x_stride + c]) * factor : Acc<T>(0);
        if (residual) v += static_cast<Acc<T>>(residual[row * a.residual_stride + c]);
        y[row * a.y_stride + c] = static_cast<T>(v);
    }
}

template <class T>
int dropout(const hk_dropout_job& j, hipStream_t stream) {
    const int64_t groups = (j.rows * j.cols + kNumbers - 1) / kNumbers;
    if (groups == 0) return HK_OK;
    const int64_t blocks = (groups + kThreads - 1) / kThreads;
    if (blocks > INT32_MAX) return hawk_internal::set_error(HK_EVALUE, "hk_dropout: the planes exceed the grid limit");
    const DropArgs a{j.offset_cell, j.seed, j.offset, j.rows, j.cols, j.x_stride, j.residual_stride, j.y_stride,
                     static_cast<uint32_t>(j.cut)};
    hipLaunchKernelGGL(hawk_dropout<T>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream, a,
                       static_cast<const T*>(j.x), static_cast<const T*>(j.residual), static_cast<T*>(j.y));
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
