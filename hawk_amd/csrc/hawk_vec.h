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

// x = mantissa(x) 2^exponent(x) with 1/2 <= |mantissa| < 1; 0, an infinity and a NaN
// are their own mantissa, of exponent 0.
__device__ __forceinline__ float mantissa(float x) { return __builtin_amdgcn_frexp_mantf(x); }
__device__ __forceinline__ double mantissa(double x) { return __builtin_amdgcn_frexp_mant(x); }
__device__ __forceinline__ int exponent(float x) { return __builtin_amdgcn_frexp_expf(x); }
__device__ __forceinline__ int exponent(double x) { return __builtin_amdgcn_frexp_exp(x); }
__device__ __forceinline__ float scaled(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }
__device__ __forceinline__ double scaled(double x, int e) { return __builtin_amdgcn_ldexp(x, e); }

// The product of a run of gates as m 2^e, which never leaves its range: a run of
// gates may grow past the type's largest number, or fall below its least, and
// still meet a state for which the result is an ordinary number.  m is 0 only
// where a gate is (a cut), and it keeps its sign.
template <class A> struct Gain { A m; int e; };
template <class A>
__device__ __forceinline__ Gain<A> normal(const Gain<A>& p) { return {mantissa(p.m), p.e + exponent(p.m)}; }
template <class A>
__device__ __forceinline__ Gain<A> times(const Gain<A>& p, const Gain<A>& q) { return {cutmul(p.m, q.m), p.e + q.e}; }
template <class A>
__device__ __forceinline__ Gain<A> times(const Gain<A>& p, A g) { return times(p, Gain<A>{mantissa(g), exponent(g)}); }
// add + p h of a normal p, the product rounded as a state of its size is; a cut
// passes nothing.
template <class A>
__device__ __forceinline__ A passed(const Gain<A>& p, A h, A add) { return add + scaled(cutmul(p.m, h), p.e); }

__device__ __forceinline__ float fused(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return __builtin_fma(a, b, c); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// sigma(z) and 1 - sigma(z), each to its own relative accuracy: with e = exp(-z)
// they are 1 / (1 + e) and e / (1 + e), neither formed by a subtraction.  e is held
// at 2^125, where sigma is taken as 0 (z below -86.6): what is lost there and just
// above it is 2^-125 in absolute terms.  A NaN z makes both values NaN.
__device__ __forceinline__ void sigmoid(float z, float& a, float& rest) {
    const float e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(-kLog2e * z, 125.0f));
    const float r = __builtin_amdgcn_rcpf(1.0f + e);
    rest = e * r;
    a = r - 0x1p-125f;
}
__device__ __forceinline__ void sigmoid(double z, double& a, double& rest) {
    const double e = exp(-fabs(z));
    const double r = 1.0 / (1.0 + e), small = e * r;
    a = z >= 0.0 ? r : small;
    rest = z >= 0.0 ? small : r;
}

}  // namespace hawk_vec

#endif
