// hawk_vec.h — element types, vector loads and stores and small numerics the
// sequence, row and dropout kernels share (not part of the C-ABI).
#ifndef HAWK_VEC_H
#define HAWK_VEC_H

#include "hawk_core.h"

#include <hip/hip_runtime.h>
#include <cstdint>

namespace hawk_vec {

typedef __bf16 bf16;
typedef _Float16 f16;

// The type an element's arithmetic and states are held in: 32 bits for every
// type of 32 bits or fewer, 64 for double.
template <class T> struct AccOf { typedef float type; };
template <> struct AccOf<double> { typedef double type; };
template <class T> using Acc = typename AccOf<T>::type;

// N elements in one register group.  Loads and stores assume no more than an
// element's own alignment: gfx950 takes a 16-byte access at any 2-byte address,
// so a row that starts anywhere is read as wide as an aligned one.
template <class T, int N> struct VecOf {
    typedef T type __attribute__((ext_vector_type(N)));
    typedef type loose __attribute__((aligned(sizeof(T))));
};
template <class T> struct VecOf<T, 1> { typedef T type; typedef T loose; };

// A vector in the plane's type.  Stream: data that this pass touches once, so it
// is not kept in the caches.
template <class T, int N> using Raw = typename VecOf<T, N>::type;
template <class T, int N, bool Stream = false>
__device__ __forceinline__ Raw<T, N> load_raw(const T* p) {
    const auto* at = reinterpret_cast<const typename VecOf<T, N>::loose*>(p);
    if constexpr (Stream) return __builtin_nontemporal_load(at);
    else return *at;
}
template <class T, int N, bool Stream = false>
__device__ __forceinline__ void store_raw(T* p, const Raw<T, N>& x) {
    auto* at = reinterpret_cast<typename VecOf<T, N>::loose*>(p);
    if constexpr (Stream) __builtin_nontemporal_store(x, at);
    else *at = x;
}
template <class T, int N>
__device__ __forceinline__ Acc<T> widen(const Raw<T, N>& v, int j) {
    if constexpr (N == 1) return static_cast<Acc<T>>(v);
    else return static_cast<Acc<T>>(v[j]);
}
template <class T, int N>
__device__ __forceinline__ void put(Raw<T, N>& v, int j, T x) {
    if constexpr (N == 1) v = x;
    else v[j] = x;
}

template <class T, int N>
__device__ __forceinline__ Raw<T, N> splat(T x) {
    Raw<T, N> v;
#pragma unroll
    for (int j = 0; j < N; ++j) put<T, N>(v, j, x);
    return v;
}

// Vectors of narrow elements stay whole registers: chosen between as words, and
// (forget) what the compiler derived from one may not be carried past a point,
// so values held in a narrow type are converted again instead of held wide.
template <class R>
__device__ __forceinline__ R choose(bool first, const R& x, const R& y) {
    if constexpr (sizeof(R) % 4 == 0) {
        typedef uint32_t W __attribute__((ext_vector_type(sizeof(R) / 4)));
        if constexpr (sizeof(R) == 4) {
            return __builtin_bit_cast(R, first ? __builtin_bit_cast(uint32_t, x) : __builtin_bit_cast(uint32_t, y));
        } else {
            const W u = __builtin_bit_cast(W, x), v = __builtin_bit_cast(W, y);
            W w;
#pragma unroll
            for (unsigned j = 0; j < sizeof(R) / 4; ++j) w[j] = first ? u[j] : v[j];
            return __builtin_bit_cast(R, w);
        }
    } else {
        return first ? x : y;
    }
}
template <class R>
__device__ __forceinline__ void forget(R& v) {
    if constexpr (sizeof(R) == 16) {
        typedef uint32_t W __attribute__((ext_vector_type(4)));
        W w = __builtin_bit_cast(W, v);
        asm volatile("" : "+v"(w));
        v = __builtin_bit_cast(R, w);
    }
}

// The same widened, and rounded to nearest even, once, to the plane's type.
template <class T, int N, bool Stream = false>
__device__ __forceinline__ void load(const T* p, Acc<T> (&out)[N]) {
    const Raw<T, N> v = load_raw<T, N, Stream>(p);
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = widen<T, N>(v, j);
}
template <class T, int N, bool Stream = false>
__device__ __forceinline__ void store(T* p, const Acc<T> (&x)[N]) {
    Raw<T, N> v;
#pragma unroll
    for (int j = 0; j < N; ++j) put<T, N>(v, j, static_cast<T>(x[j]));
    store_raw<T, N, Stream>(p, v);
}

// a * b, and 0 where either is 0 whatever the other is.
__device__ __forceinline__ float cutmul(float a, float b) {
    float r;
    asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double cutmul(double a, double b) { return a == 0.0 || b == 0.0 ? 0.0 : a * b; }

// The product of two gates' products.  It is 0 only where one of them is (a
// cut): a product too small for the type stays the least normal number, so an
// infinity or a NaN that enters a long run of small gates also leaves it.
__device__ __forceinline__ float least_normal(float) { return 1.17549435e-38f; }
__device__ __forceinline__ double least_normal(double) { return 2.2250738585072014e-308; }
template <class A>
__device__ __forceinline__ A chain(A a, A b) {
    const A p = cutmul(a, b);
    return p == A(0) && a != A(0) && b != A(0) ? least_normal(A(0)) : p;
}
// The smaller of m and |g|; a NaN g leaves m.
__device__ __forceinline__ float smaller(float m, float g) { return __builtin_fminf(m, __builtin_fabsf(g)); }
__device__ __forceinline__ double smaller(double m, double g) { return __builtin_fmin(m, __builtin_fabs(g)); }

__device__ __forceinline__ float fused(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return __builtin_fma(a, b, c); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// sigma(z) and 1 - sigma(z), each to its own relative accuracy: e = exp(-|z|)
// never overflows and neither value is formed by a subtraction.
__device__ __forceinline__ void sigmoid(float z, float& a, float& rest) {
    const float e = __builtin_amdgcn_exp2f(-kLog2e * __builtin_fabsf(z));
    const float r = __builtin_amdgcn_rcpf(1.0f + e);
    const float small = e * r;
    a = z >= 0.0f ? r : small;           // a NaN z makes both values NaN
    rest = z >= 0.0f ? small : r;
}
__device__ __forceinline__ void sigmoid(double z, double& a, double& rest) {
    const double e = exp(-fabs(z));
    const double r = 1.0 / (1.0 + e), small = e * r;
    a = z >= 0.0 ? r : small;
    rest = z >= 0.0 ? small : r;
}

}  // namespace hawk_vec

#endif
