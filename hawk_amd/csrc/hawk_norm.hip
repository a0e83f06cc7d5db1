// hawk_norm.hip — layer norm over rows on gfx950, and its derivative with the
// reduction of the weight's and the bias's gradients.
//
// The mathematics.  y = xh w + b, xh = (x - mean) rstd, rstd = 1 / sqrt(var + eps);
// var is the mean of (x - mean)^2 about the row's own mean, taken in a second pass
// over registers, so no digits are lost where the mean is large.  With g = bar_y w,
//   bar_x = rstd (g - mean(g) - xh mean(g xh)),
//   bar_w = sum over rows of bar_y xh,  bar_b = sum over rows of bar_y.
// Everything is computed in 32 bits; a result is rounded once, to its plane's type.
//
// What bounds it: HBM.  A row is read once and kept in registers by L lanes.  The
// sums over rows run along in registers too: a workgroup takes many rows, leaves one
// partial sum a column, and a second launch adds those in a fixed order.  16384 rows of
// 4096 bfloat16 columns take 53.7 us forward (5.0 TB/s; a plain copy of 1 GiB reaches
// 5.1); the derivative of 16384 x 2048 with both sums 46 us, of which the second launch is
// 4: two workgroups a unit, each with its next row's loads under way; more of them
// leave more partial sums.

#include "hawk_core.h"
#include "hawk_internal.h"
#include "hawk_vec.h"

#include <hip/hip_runtime.h>
#include <cstdint>
#include <string>
#include <type_traits>

namespace {

using namespace hawk_vec;

constexpr int kThreads = 256;
constexpr int kMost = 1024;                // lanes of a row that is not held in registers
constexpr int64_t kUnits = 256;            // compute units

template <class T> constexpr int kVec = 16 / static_cast<int>(sizeof(T));
// Rows of 16-bit elements pass as a stream, which is not kept in the caches.
template <class T> constexpr bool kOnce = sizeof(T) == 2;

template <class T>
struct NormArgs {
    const T *x, *bar_y;
    T *y, *bar_x;                          // bar_x may be NULL
    const void *weight, *bias;             // of T, or float where wide; NULL: 1 and 0
    float *mean, *rstd;
    float* parts;                          // the workgroups' sums: [2][parts][cols], or NULL
    int64_t rows, x_stride, y_stride, bar_y_stride, bar_x_stride;
    int cols, wide;
    float eps, inverse;                    // inverse: 1 / cols
};

// A row of 16-bit columns whose last ones are no whole vector has its last whole vector read
// in their place; its first elements are another lane's too.  In the forward pass they count
// where they are that lane's and are written by both, the same; in the derivative, which
// keeps sums of the columns, the vector is ordered ahead and settled, moved into place, when
// it is used.  (144416 rows of 347 bfloat16 columns, element by element: 100 and 257 us;
// this way 81 and 180.  Of floats there are three at most, and element by element is as good.)
template <class T, bool Whole>
__device__ __forceinline__ bool shared_end(int c, int cols) {
    constexpr int V = kVec<T>;
    return !Whole && V == 8 && c < cols && c + V > cols && cols >= V;
}
template <class T, bool Whole>
__device__ __forceinline__ int begin_of(int c, int cols) {
    return shared_end<T, Whole>(c, cols) ? cols - kVec<T> : c;
}
// The V elements from column c of a row; what lies past the row is 0 and not read.
template <class T, bool Whole, bool Stream = false>
__device__ __forceinline__ Raw<T, kVec<T>> order(const T* row, int c, int cols) {
    constexpr int V = kVec<T>;
    if (c + V <= cols) return load_raw<T, V, Stream>(row + c);
    if (shared_end<T, Whole>(c, cols)) return load_raw<T, V, Stream>(row + cols - V);
    Raw<T, V> x = splat<T, V>(static_cast<T>(0.0f));
    if constexpr (!Whole) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j < cols) put<T, V>(x, j, row[c + j]);
    }
    return x;
}
template <class T, bool Whole>
__device__ __forceinline__ Raw<T, kVec<T>> settle(Raw<T, kVec<T>> x, int c, int cols) {
    constexpr int V = kVec<T>;
    if (shared_end<T, Whole>(c, cols)) {
        using Bits = unsigned __int128;
        static_assert(sizeof(x) == sizeof(Bits), "a vector is 16 bytes");
        x = __builtin_bit_cast(Raw<T, V>, __builtin_bit_cast(Bits, x) >> (c + V - cols) * static_cast<int>(8 * sizeof(T)));
    }
    return x;
}
template <class T, bool Whole, bool Stream = false>
__device__ __forceinline__ Raw<T, kVec<T>> fetch(const T* row, int c, int cols) {
    return settle<T, Whole>(order<T, Whole, Stream>(row, c, cols), c, cols);
}
template <class T, bool Whole, bool Stream = false>
__device__ __forceinline__ void leave(T* row, int c, int cols, const float (&x)[kVec<T>]) {
    constexpr int V = kVec<T>;
    if (c + V <= cols) {
        store<T, V, Stream>(row + c, x);
        return;
    }
    if constexpr (!Whole) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j < cols) row[c + j] = static_cast<T>(x[j]);
    }
}
// The weight's (or the bias's) V numbers at column c.
template <class T, bool Whole>
__device__ __forceinline__ void factors(const void* w, int wide, int c, int cols, float none, float (&out)[kVec<T>]) {
    constexpr int V = kVec<T>;
    if (!w) {
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = none;
    } else if (wide) {
        const float* at = static_cast<const float*>(w);
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const Raw<float, 4> v = fetch<float, Whole>(at, c + i, cols);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[i + j] = v[j];
        }
    } else {
        const Raw<T, V> v = fetch<T, Whole>(static_cast<const T*>(w), c, cols);
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = widen<T, V>(v, j);
    }
}

// The sums of L lanes' numbers in every lane: a fixed tree within a wave, the waves'
// sums in a fixed tree.  `turn` alternates, so one barrier a call is enough.
template <int L, int N>
__device__ __forceinline__ void sum_lanes(float (&v)[N], int turn) {
#pragma unroll
    for (int d = (L < 64 ? L : 64) / 2; d > 0; d >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], d);
    if constexpr (L > 64) {
        constexpr int W = L / 64;
        __shared__ float lds[2][N][W];
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) lds[turn][k][threadIdx.x >> 6] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float t = lds[turn][k][threadIdx.x & (W - 1)];
#pragma unroll
            for (int d = W / 2; d > 0; d >>= 1) t += __shfl_xor(t, d);
            v[k] = t;
        }
    }
}

// Rows held in the registers of L lanes, NV vectors a lane; several rows a workgroup
// where L is below it.
template <class T, int L, int NV, bool Whole>
__global__ void __launch_bounds__((L > kThreads ? L : kThreads)) hawk_norm(const NormArgs<T> a) {
    constexpr int V = kVec<T>, R = (L > kThreads ? L : kThreads) / L;
    const int lane = threadIdx.x % L, cols = a.cols;
    int turn = 0;
    for (int64_t n = static_cast<int64_t>(blockIdx.x) * R + threadIdx.x / L; n < a.rows; n += static_cast<int64_t>(gridDim.x) * R) {
        const T* row = a.x + n * a.x_stride;
        Raw<T, V> x[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) x[i] = fetch<T, Whole, kOnce<T> && Whole>(row, begin_of<T, Whole>((i * L + lane) * V, cols), cols);
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * L + lane) * V, at = begin_of<T, Whole>(c, cols);
#pragma unroll
            for (int j = 0; j < V; ++j) s[0] += Whole || at + j >= c ? widen<T, V>(x[i], j) : 0.0f;
        }
        sum_lanes<L>(s, turn);
        turn ^= 1;
        const float mean = s[0] * a.inverse;
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * L + lane) * V, at = begin_of<T, Whole>(c, cols);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = widen<T, V>(x[i], j) - mean;
                s[0] = fused(d, (Whole ? c < cols : at + j >= c && at + j < cols) ? d : 0.0f, s[0]);
            }
        }
        sum_lanes<L>(s, turn);
        turn ^= 1;
        const float rstd = 1.0f / sqrtf(s[0] * a.inverse + a.eps);
        if (lane == 0) {
            if (a.mean) a.mean[n] = mean;
            if (a.rstd) a.rstd[n] = rstd;
        }
        if (!a.y) continue;
        T* out = a.y + n * a.y_stride;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = begin_of<T, Whole>((i * L + lane) * V, cols);
            float w[V], b[V], y[V];
            factors<T, Whole>(a.weight, a.wide, c, cols, 1.0f, w);
            factors<T, Whole>(a.bias, a.wide, c, cols, 0.0f, b);
#pragma unroll
            for (int j = 0; j < V; ++j) y[j] = fused((widen<T, V>(x[i], j) - mean) * rstd, w[j], b[j]);
            leave<T, Whole, kOnce<T> && Whole>(out, c, cols, y);
        }
    }
}

// Rows past the registers: three passes over one, by a workgroup.  (The second and the
// third find it in the caches.)
template <class T>
__global__ void __launch_bounds__(kMost) hawk_norm_long(const NormArgs<T> a) {
    constexpr int V = kVec<T>, Step = kMost * V;
    const int cols = a.cols, mine = threadIdx.x * V;
    int turn = 0;
    for (int64_t n = blockIdx.x; n < a.rows; n += gridDim.x) {
        const T* row = a.x + n * a.x_stride;
        float s[1] = {0.0f};
        for (int c = mine; c < cols; c += Step) {
            const Raw<T, V> x = fetch<T, false>(row, c, cols);
#pragma unroll
            for (int j = 0; j < V; ++j) s[0] += widen<T, V>(x, j);
        }
        sum_lanes<kMost>(s, turn);
        turn ^= 1;
        const float mean = s[0] * a.inverse;
        s[0] = 0.0f;
        for (int c = mine; c < cols; c += Step) {
            const Raw<T, V> x = fetch<T, false>(row, c, cols);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = widen<T, V>(x, j) - mean;
                s[0] = fused(d, c + j < cols ? d : 0.0f, s[0]);
            }
        }
        sum_lanes<kMost>(s, turn);
        turn ^= 1;
        const float rstd = 1.0f / sqrtf(s[0] * a.inverse + a.eps);
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[n] = mean;
            if (a.rstd) a.rstd[n] = rstd;
        }
        if (!a.y) continue;
        T* out = a.y + n * a.y_stride;
        for (int c = mine; c < cols; c += Step) {
            const Raw<T, V> x = fetch<T, false>(row, c, cols);
            float w[V], b[V], y[V];
            factors<T, false>(a.weight, a.wide, c, cols, 1.0f, w);
            factors<T, false>(a.bias, a.wide, c, cols, 0.0f, b);
#pragma unroll
            for (int j = 0; j < V; ++j) y[j] = fused((widen<T, V>(x, j) - mean) * rstd, w[j], b[j]);
            leave<T, false>(out, c, cols, y);
        }
    }
}

// The derivative.  A lane's columns are the same in every row that its workgroup
// takes, so the sums over rows stay in its registers.
template <class T, int L, int NV, bool Whole>
__global__ void __launch_bounds__((L > kThreads ? L : kThreads)) hawk_norm_vjp(const NormArgs<T> a) {
    constexpr int V = kVec<T>, Block = L > kThreads ? L : kThreads, R = Block / L;
    const int lane = threadIdx.x % L, cols = a.cols;
    float w[NV][V], sw[NV][V], sb[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        factors<T, Whole>(a.weight, a.wide, (i * L + lane) * V, cols, 1.0f, w[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) sw[i][j] = sb[i][j] = 0.0f;
    }
    int turn = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * R;
    int64_t n = static_cast<int64_t>(blockIdx.x) * R + threadIdx.x / L;
    // the next row's loads are under way while a row is reduced
    Raw<T, V> nx[NV], nb[NV];
    float next_mean = 0.0f, next_rstd = 0.0f;
    auto ask = [&](int64_t row) {
        if (row >= a.rows) return;
        next_mean = a.mean[row];
        next_rstd = a.rstd[row];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            nx[i] = order<T, Whole, kOnce<T> && Whole>(a.x + row * a.x_stride, (i * L + lane) * V, cols);
            nb[i] = order<T, Whole, kOnce<T> && Whole>(a.bar_y + row * a.bar_y_stride, (i * L + lane) * V, cols);
        }
    };
    ask(n);
    for (; n < a.rows; n += step) {
        const float mean = next_mean, rstd = next_rstd;
        Raw<T, V> x[NV], b[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x[i] = settle<T, Whole>(nx[i], (i * L + lane) * V, cols);
            b[i] = settle<T, Whole>(nb[i], (i * L + lane) * V, cols);
        }
        ask(n + step);
        float s[2] = {0.0f, 0.0f};
        // bar_y is 0 past the row, and w is
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = (widen<T, V>(x[i], j) - mean) * rstd, by = widen<T, V>(b[i], j);
                const float g = by * w[i][j];
                const int c = (i * L + lane) * V + (Whole ? 0 : j);
                s[0] += g;
                s[1] = fused(g, c < cols ? xh : 0.0f, s[1]);
                sw[i][j] = fused(by, xh, sw[i][j]);
                sb[i][j] += by;
            }
        if (!a.bar_x) continue;
        sum_lanes<L>(s, turn);
        turn ^= 1;
        const float one = s[0] * a.inverse, two = s[1] * a.inverse;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float out[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = (widen<T, V>(x[i], j) - mean) * rstd;
                out[j] = rstd * (fused(widen<T, V>(b[i], j), w[i][j], -one) - xh * two);
            }
            leave<T, Whole, kOnce<T> && Whole>(a.bar_x + n * a.bar_x_stride, (i * L + lane) * V, cols, out);
        }
    }
    if (!a.parts) return;
    float* part = a.parts + static_cast<int64_t>(blockIdx.x) * cols;
    const int64_t other = static_cast<int64_t>(gridDim.x) * cols;
    if constexpr (R == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * L + lane) * V;
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const float u[4] = {sw[i][j], sw[i][j + 1], sw[i][j + 2], sw[i][j + 3]};
                const float v[4] = {sb[i][j], sb[i][j + 1], sb[i][j + 2], sb[i][j + 3]};
                leave<float, Whole>(part, c + j, cols, u);
                leave<float, Whole>(part + other, c + j, cols, v);
            }
        }
    } else {
        // the workgroup's rows are added in their order
        __shared__ float lds[Block * NV * V];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    lds[(threadIdx.x / L * NV + i) * (L * V) + lane * V + j] = k ? sb[i][j] : sw[i][j];
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += Block) {
                float t = 0.0f;
#pragma unroll
                for (int r = 0; r < R; ++r) t += lds[r * (NV * L * V) + c];
                part[k * other + c] = t;
            }
        }
    }
}

// The derivative of rows past the registers, by a workgroup each; the sums over rows
// are another launch's.
template <class T>
__global__ void __launch_bounds__(kMost) hawk_norm_vjp_long(const NormArgs<T> a) {
    constexpr int V = kVec<T>, Step = kMost * V;
    const int cols = a.cols, mine = threadIdx.x * V;
    int turn = 0;
    for (int64_t n = blockIdx.x; n < a.rows; n += gridDim.x, turn ^= 1) {
        const T *row = a.x + n * a.x_stride, *bar = a.bar_y + n * a.bar_y_stride;
        const float mean = a.mean[n], rstd = a.rstd[n];
        float s[2] = {0.0f, 0.0f}, w[V];
        for (int c = mine; c < cols; c += Step) {
            const Raw<T, V> x = fetch<T, false>(row, c, cols), b = fetch<T, false>(bar, c, cols);
            factors<T, false>(a.weight, a.wide, c, cols, 1.0f, w);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float g = widen<T, V>(b, j) * w[j];
                s[0] += g;
                s[1] = fused(g, c + j < cols ? (widen<T, V>(x, j) - mean) * rstd : 0.0f, s[1]);
            }
        }
        sum_lanes<kMost>(s, turn);
        const float one = s[0] * a.inverse, two = s[1] * a.inverse;
        for (int c = mine; c < cols; c += Step) {
            const Raw<T, V> x = fetch<T, false>(row, c, cols), b = fetch<T, false>(bar, c, cols);
            float out[V];
            factors<T, false>(a.weight, a.wide, c, cols, 1.0f, w);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = (widen<T, V>(x, j) - mean) * rstd;
                out[j] = rstd * (fused(widen<T, V>(b, j), w[j], -one) - xh * two);
            }
            leave<T, false>(a.bar_x + n * a.bar_x_stride, c, cols, out);
        }
    }
}
// Workgroup (column tile, part): its columns' sums over every gridDim.y-th row.
template <class T>
__global__ void __launch_bounds__(kThreads) hawk_norm_columns(const NormArgs<T> a) {
    constexpr int V = kVec<T>;
    const int c = (blockIdx.x * kThreads + threadIdx.x) * V, cols = a.cols;
    if (c >= cols) return;
    float sw[V], sb[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sw[j] = sb[j] = 0.0f;
    for (int64_t n = blockIdx.y; n < a.rows; n += gridDim.y) {
        const float mean = a.mean[n], rstd = a.rstd[n];
        const Raw<T, V> x = fetch<T, false>(a.x + n * a.x_stride, c, cols), b = fetch<T, false>(a.bar_y + n * a.bar_y_stride, c, cols);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            sw[j] = fused(widen<T, V>(b, j), (widen<T, V>(x, j) - mean) * rstd, sw[j]);
            sb[j] += widen<T, V>(b, j);
        }
    }
    float* part = a.parts + static_cast<int64_t>(blockIdx.y) * cols;
    const int64_t other = static_cast<int64_t>(gridDim.y) * cols;
#pragma unroll
    for (int j = 0; j < V; j += 4) {
        const float u[4] = {sw[j], sw[j + 1], sw[j + 2], sw[j + 3]}, v[4] = {sb[j], sb[j + 1], sb[j + 2], sb[j + 3]};
        leave<float, false>(part, c + j, cols, u);
        leave<float, false>(part + other, c + j, cols, v);
    }
}

// The workgroups' sums of kTile columns added in a fixed order, in 64 bits: 64 streams
// of parts by 16 columns, so a wave reads whole 64-byte lines.  A launch stays below 2^32
// threads: past kMostTiles * kTile columns a workgroup has several tiles.
constexpr int kTile = 16, kStreams = 64;
constexpr int64_t kMostTiles = 1 << 20;
template <class G>
__global__ void __launch_bounds__(kTile* kStreams) hawk_norm_total(const float* parts, int64_t count, int64_t cols, G* weight, G* bias) {
    __shared__ double lds[kStreams][kTile + 1];
    G* out = blockIdx.y ? bias : weight;
    if (!out) return;
    const int lane = threadIdx.x % kTile, stream = threadIdx.x / kTile;
    for (int64_t tile = blockIdx.x; tile * kTile < cols; tile += gridDim.x) {
        const int64_t c = tile * kTile + lane;
        double t = 0.0;
        if (c < cols) {
            const float* at = parts + blockIdx.y * count * cols + c;
#pragma unroll 4
            for (int64_t p = stream; p < count; p += kStreams) t += static_cast<double>(at[p * cols]);
        }
        lds[stream][lane] = t;
        __syncthreads();
        for (int d = kStreams / 2; d > 0; d >>= 1) {
            if (stream < d) lds[stream][lane] += lds[stream + d][lane];
            __syncthreads();
        }
        if (stream == 0 && c < cols) out[c] = static_cast<G>(static_cast<float>(lds[0][lane]));
        // (row 0 is written anew by the threads that read it here, the others' were read before the last barrier)
    }
}
template <class G>
__global__ void __launch_bounds__(kThreads) hawk_norm_none(int64_t cols, G* weight, G* bias) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (c >= cols) return;
    if (weight) weight[c] = static_cast<G>(0.0f);
    if (bias) bias[c] = static_cast<G>(0.0f);
}

// Rows without columns: the mean of no numbers.
__global__ void __launch_bounds__(kThreads) hawk_norm_empty(int64_t rows, float* mean, float* rstd) {
    for (int64_t n = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; n < rows; n += static_cast<int64_t>(gridDim.x) * kThreads) {
        if (mean) mean[n] = NAN;
        if (rstd) rstd[n] = NAN;
    }
}

int size_of(int dtype) { return dtype == HK_F32 ? 4 : 2; }

// How a row is held: `lanes` lanes of `vectors` vectors, or lanes = 0 for one that is
// not.  A row takes the fewest lanes that hold it in two vectors each; a wave four of them
// where those are 16 numbers, as it waits for no other wave (the derivative of 3001 rows of
// 777 floats with the sums: 14.9 us, 16.9 by four waves a row).  The wider the workgroup of a
// row is, the fewer rows are under way beside one that waits at its barrier, so long rows
// take few waves: 16384 x 8192 bfloat16 forward 122 us by 256 lanes of four, 165 by 1024 of
// one, its derivative 146 by 512 of two, 182 by 1024 of one; 4096 x 16384 forward 61 by 512 of four, 78 by
// 1024 of two.  The derivative's sums leave no registers for more vectors a lane.
struct Shape { int lanes, vectors; };
Shape shape_of(int64_t cols, int esize, bool vjp) {
    const int64_t vectors = (cols + 16 / esize - 1) / (16 / esize);
    if (vectors <= 16) return {16, 1};
    if (vectors <= 64) return {64, 1};
    if (vectors <= 128) return {64, 2};
    if (vectors <= 256) return esize == 4 ? Shape{64, 4} : Shape{256, 1};
    if (vectors <= 512) return {256, 2};
    if (vectors <= 1024) return vjp ? Shape{512, 2} : Shape{256, 4};
    if (vectors <= 2048) return vjp ? Shape{1024, 2} : Shape{512, 4};
    return {0, 0};
}
// The derivative's workgroups, each with a partial sum a column.
int64_t parts_of(int64_t rows, int64_t cols, int esize) {
    const Shape s = shape_of(cols, esize, true);
    if (s.lanes == 0) return rows < kUnits / 4 ? rows : kUnits / 4;
    const int64_t at_once = s.lanes > kThreads ? 1 : kThreads / s.lanes;
    const int64_t need = (rows + at_once - 1) / at_once, most = s.lanes > kThreads ? kUnits : 2 * kUnits;
    return need < most ? need : most;
}

int launched(const char* what) {
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? HK_OK : hawk_internal::set_hip_error(what, err);
}

// Four vectors a lane of a wave, which 16-bit rows do not take.
template <class T, class F>
void wave_of_four(F&& f) {
    if constexpr (sizeof(T) == 4) f(std::integral_constant<int, 4>());
}

template <class T>
NormArgs<T> args_of(const hk_layer_norm_job& j) {
    NormArgs<T> a;
    a.x = static_cast<const T*>(j.x);
    a.bar_y = static_cast<const T*>(j.bar_y);
    a.y = static_cast<T*>(j.y);
    a.bar_x = static_cast<T*>(j.bar_x);
    a.weight = j.weight;
    a.bias = j.bias;
    a.mean = j.mean;
    a.rstd = j.rstd;
    a.parts = nullptr;
    a.rows = j.rows;
    a.x_stride = j.x_stride;
    a.y_stride = j.y_stride;
    a.bar_y_stride = j.bar_y_stride;
    a.bar_x_stride = j.bar_x_stride;
    a.cols = static_cast<int>(j.cols);
    a.wide = j.weight_dtype == HK_F32 && j.dtype != HK_F32;
    a.eps = j.eps;
    a.inverse = static_cast<float>(1.0 / static_cast<double>(j.cols));
    return a;
}

template <class T, int L, int NV>
void launch_norm(const NormArgs<T>& a, hipStream_t stream) {
    constexpr int Block = L > kThreads ? L : kThreads, R = Block / L;
    const int64_t need = (a.rows + R - 1) / R, most = 1 << 20;
    const dim3 grid(static_cast<unsigned>(need < most ? need : most)), block(Block);
    if (a.cols % kVec<T> == 0) hipLaunchKernelGGL((hawk_norm<T, L, NV, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((hawk_norm<T, L, NV, false>), grid, block, 0, stream, a);
}
template <class T>
int norm(const hk_layer_norm_job& j, hipStream_t stream) {
    const NormArgs<T> a = args_of<T>(j);
    const Shape s = shape_of(j.cols, sizeof(T), false);
    if (s.lanes == 0) {
        const dim3 grid(static_cast<unsigned>(j.rows < 4 * kUnits ? j.rows : 4 * kUnits)), block(kMost);
        hipLaunchKernelGGL((hawk_norm_long<T>), grid, block, 0, stream, a);
    } else if (s.lanes == 16) launch_norm<T, 16, 1>(a, stream);
    else if (s.lanes == 64) s.vectors == 1 ? launch_norm<T, 64, 1>(a, stream) : s.vectors == 2 ? launch_norm<T, 64, 2>(a, stream) : wave_of_four<T>([&](auto four) { launch_norm<T, 64, decltype(four)::value>(a, stream); });
    else if (s.lanes == 256) s.vectors == 1 ? launch_norm<T, 256, 1>(a, stream) : s.vectors == 2 ? launch_norm<T, 256, 2>(a, stream) : launch_norm<T, 256, 4>(a, stream);
    else launch_norm<T, 512, 4>(a, stream);
    return launched("hawk_norm launch");
}

template <class T, int L, int NV>
void launch_vjp(const NormArgs<T>& a, int64_t blocks, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(blocks)), block(L > kThreads ? L : kThreads);
    if (a.cols % kVec<T> == 0) hipLaunchKernelGGL((hawk_norm_vjp<T, L, NV, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((hawk_norm_vjp<T, L, NV, false>), grid, block, 0, stream, a);
}
template <class T, class G>
int totals(const hk_layer_norm_job& j, const float* parts, int64_t count, hipStream_t stream) {
    G *weight = static_cast<G*>(j.bar_weight), *bias = static_cast<G*>(j.bar_bias);
    if (count == 0) {
        const dim3 grid(static_cast<unsigned>((j.cols + kThreads - 1) / kThreads)), block(kThreads);
        hipLaunchKernelGGL((hawk_norm_none<G>), grid, block, 0, stream, j.cols, weight, bias);
    } else {
        const int64_t tiles = (j.cols + kTile - 1) / kTile;
        const dim3 grid(static_cast<unsigned>(tiles < kMostTiles ? tiles : kMostTiles), 2), block(kTile * kStreams);
        hipLaunchKernelGGL((hawk_norm_total<G>), grid, block, 0, stream, parts, count, j.cols, weight, bias);
    }
    return launched("hawk_norm_total launch");
}
template <class T>
int norm_vjp(const hk_layer_norm_job& j, float* scratch, hipStream_t stream) {
    NormArgs<T> a = args_of<T>(j);
    const bool sums = j.bar_weight || j.bar_bias;
    const int64_t parts = j.rows ? parts_of(j.rows, j.cols, sizeof(T)) : 0;
    if (sums) a.parts = scratch;
    if (j.rows) {
        const Shape s = shape_of(j.cols, sizeof(T), true);
        if (s.lanes == 0) {
            if (sums) {                                    // first: bar_x may be x or bar_y
                const int64_t tile = kThreads * kVec<T>;
                const dim3 grid(static_cast<unsigned>((j.cols + tile - 1) / tile), static_cast<unsigned>(parts)), block(kThreads);
                hipLaunchKernelGGL((hawk_norm_columns<T>), grid, block, 0, stream, a);
            }
            if (a.bar_x) {
                const dim3 grid(static_cast<unsigned>(j.rows < 4 * kUnits ? j.rows : 4 * kUnits)), block(kMost);
                hipLaunchKernelGGL((hawk_norm_vjp_long<T>), grid, block, 0, stream, a);
            }
        } else if (s.lanes == 16) launch_vjp<T, 16, 1>(a, parts, stream);
        else if (s.lanes == 64) s.vectors == 1 ? launch_vjp<T, 64, 1>(a, parts, stream) : s.vectors == 2 ? launch_vjp<T, 64, 2>(a, parts, stream) : wave_of_four<T>([&](auto four) { launch_vjp<T, 64, decltype(four)::value>(a, parts, stream); });
        else if (s.lanes == 256) s.vectors == 1 ? launch_vjp<T, 256, 1>(a, parts, stream) : launch_vjp<T, 256, 2>(a, parts, stream);
        else if (s.lanes == 512) launch_vjp<T, 512, 2>(a, parts, stream);
        else launch_vjp<T, 1024, 2>(a, parts, stream);
        const int rc = launched("hawk_norm_vjp launch");
        if (rc != HK_OK) return rc;
    }
    if (!sums) return HK_OK;
    return j.weight_dtype == HK_F32 ? totals<T, float>(j, scratch, parts, stream) : totals<T, T>(j, scratch, parts, stream);
}

int refuse(const hk_layer_norm_job* j) {
    using hawk_internal::set_error;
    if (!j) return set_error(HK_EVALUE, "hk_layer_norm: a job is required");
    if (j->rows < 0 || j->cols < 0) return set_error(HK_EVALUE, "hk_layer_norm: sizes must be >= 0");
    if (j->dtype != HK_F32 && j->dtype != HK_BF16 && j->dtype != HK_F16)
        return set_error(HK_EVALUE, "hk_layer_norm: the planes' element type is 32-bit or 16-bit");
    if (j->weight_dtype != HK_F32 && j->weight_dtype != j->dtype)
        return set_error(HK_EVALUE, "hk_layer_norm: the weights' element type is 32-bit or the planes'");
    if (j->cols > INT32_MAX / 2 || (j->cols > 0 && j->rows > INT64_MAX / 16 / j->cols))
        return set_error(HK_EVALUE, "hk_layer_norm: the planes exceed the grid limit");
    auto crosses = [&](const void* out, int64_t out_stride, const void* in, int64_t in_stride) {
        return j->rows > 1 && j->cols > 0 && out && out == in && out_stride != in_stride;
    };
    if (crosses(j->y, j->y_stride, j->x, j->x_stride) || crosses(j->bar_x, j->bar_x_stride, j->x, j->x_stride) ||
        crosses(j->bar_x, j->bar_x_stride, j->bar_y, j->bar_y_stride))
        return set_error(HK_EVALUE, "hk_layer_norm: an output over an input has its row distance");
    if (!(j->eps >= 0.0f)) return set_error(HK_EVALUE, "hk_layer_norm: eps must be >= 0");
    return HK_OK;
}

}  // namespace

extern "C" size_t hk_layer_norm_scratch_bytes(const hk_layer_norm_job* job, int32_t vjp) {
    if (!job || !vjp || job->rows <= 0 || job->cols <= 0 || (!job->bar_weight && !job->bar_bias)) return 0;
    if (job->dtype != HK_F32 && job->dtype != HK_BF16 && job->dtype != HK_F16) return 0;
    return static_cast<size_t>(parts_of(job->rows, job->cols, size_of(job->dtype))) * static_cast<size_t>(job->cols) * 2 * sizeof(float);
}

extern "C" int hk_layer_norm(const hk_layer_norm_job* job, void* scratch, void* stream) {
    (void)scratch;
    const int rc = refuse(job);
    if (rc != HK_OK) return rc;
    if (job->rows == 0) return HK_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (job->cols == 0) {
        if (!job->mean && !job->rstd) return HK_OK;
        const int64_t need = (job->rows + kThreads - 1) / kThreads;
        hipLaunchKernelGGL(hawk_norm_empty, dim3(static_cast<unsigned>(need < 4 * kUnits ? need : 4 * kUnits)), dim3(kThreads), 0, s, job->rows,
                           job->mean, job->rstd);
        return launched("hawk_norm_empty launch");
    }
    if (!job->x) return hawk_internal::set_error(HK_EVALUE, "hk_layer_norm: x is required");
    if (job->dtype == HK_F32) return norm<float>(*job, s);
    return job->dtype == HK_BF16 ? norm<bf16>(*job, s) : norm<f16>(*job, s);
}

extern "C" int hk_layer_norm_vjp(const hk_layer_norm_job* job, void* scratch, void* stream) {
    using hawk_internal::set_error;
    const int rc = refuse(job);
    if (rc != HK_OK) return rc;
    if (job->cols == 0) return HK_OK;
    if (job->rows > 0 && (!job->x || !job->bar_y || !job->mean || !job->rstd))
        return set_error(HK_EVALUE, "hk_layer_norm_vjp: x, bar_y, mean and rstd are required");
    if (job->rows > 0 && (job->bar_weight || job->bar_bias) && !scratch)
        return set_error(HK_EVALUE, "hk_layer_norm_vjp: scratch is required for the sums over rows");
    hipStream_t s = static_cast<hipStream_t>(stream);
    float* work = static_cast<float*>(scratch);
    if (job->dtype == HK_F32) return norm_vjp<float>(*job, work, s);
    return job->dtype == HK_BF16 ? norm_vjp<bf16>(*job, work, s) : norm_vjp<f16>(*job, work, s);
}
