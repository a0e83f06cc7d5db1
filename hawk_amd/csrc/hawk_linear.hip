// hawk_linear.hip — linear attention with a decay for each head on gfx950, and its
// derivative.
//
// The mathematics.  S_t = g S_(t-1) + k_t v_t^T, o_t = scale q_t S_t.  Written out,
//   o_i = scale sum_(j <= i) g^(i-j) (q_i . k_j) v_j + scale g^(i+1) q_i h0,
// one form A(a, b, c) of three planes, whose derivative is the same form with the
// planes in other places: bar_q = A(bar_o, v, k), and with time reversed
// bar_k = A(v, bar_o, q), bar_v = A(k, q, bar_o).  One kernel computes all four.
//
// In chunks of C tokens, with X what the tokens before a chunk have left, as its
// first token sees it,
//   out_i = g^i (a_i X) + sum_(j <= i in the chunk) g^(i-j) (a_i . b_j) c_j,
//   X' = g^C X + sum_j g^(C-j) b_j c_j^T :
// products for the matrix cores.  A workgroup walks a run of chunks with its columns
// of X in registers: a wave has 16 columns of c.  X as the matrix cores leave it is
// an operand of the next chunk's product as it stands, if that product takes its
// terms in the order in which X lies in the lanes; a's columns are staged in that order.
//
// The numbers.  X and every sum are held in 32 bits.  The matrix cores multiply bf16;
// a number of more digits is a sum of bf16 parts (three make 24 bits), and a product is
// the sum of the parts' products down to 2^-25 of it wherever X is made or read.  Inside a
// chunk (a_i . b_j, and that times c_j) it is so for 32-bit planes; where the result is
// rounded to 16 bits, a_i . b_j is held as two parts, 2^-17 of it, which leaves 6e-5 of a
// bfloat16 result's norm in places that round the other way (three parts: 4e-5, and 340
// and 785 us where the two calls below take 270 and 566).
//
// What bounds it.  The eight waves of a workgroup share a chunk, in phases between four
// barriers; registers and LDS hold two workgroups a unit.  In the walk of 16 heads of 128
// bfloat16 columns LDS is active in 47 % of the units' busy cycles (44 % of those are bank
// conflicts), the vector units in 57 %, the matrix cores in 34 %.  One sequence of 32768 such
// tokens takes 270 us (states of its segments 76, their join 14, the walk 178; the bytes'
// time is 81); the derivative of 8 x 4096 tokens, whose 8 * 16 * 3 walks fill the chip
// uncut, 566 in one launch.  Waves of two column tiles, four to a workgroup, took a tenth
// longer; products of two tiles in turn were no faster.

#include "hawk_core.h"
#include "hawk_internal.h"
#include "hawk_vec.h"

#include <hip/hip_runtime.h>
#include <cstdint>
#include <string>
#include <type_traits>

namespace {

using namespace hawk_vec;

constexpr int kJoinThreads = 256;
constexpr int kMostWidth = 256, kMostWalks = 3;
constexpr int64_t kUnits = 256, kDies = 8;

typedef __bf16 Bf8 __attribute__((ext_vector_type(8)));
typedef float F4 __attribute__((ext_vector_type(4)));
typedef uint16_t H4 __attribute__((ext_vector_type(4)));
typedef uint16_t H8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ F4 product(const H8& a, const H8& b, const F4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Bf8, a), __builtin_bit_cast(Bf8, b), c, 0, 0, 0);
}

// What is written before is scheduled before: the reads of a loop that is unrolled are
// not all made first, which would take the registers of all of them.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// The N bf16 parts of a number, each the nearest to what the ones before leave: two are
// within 2^-17 of it, three are a number of 24 bits.  The first is no infinity where the
// number is none (Large: it may be above bf16's largest, and the nearest would be one).
constexpr float kMostPart = 0x1.fep127f;
template <int N, bool Large = true>
__device__ __forceinline__ void cut(float x, uint16_t (&out)[N]) {
#pragma unroll
    for (int p = 0; p < N; ++p) {
        const bf16 h = static_cast<bf16>(Large && p == 0 && N > 1 ? __builtin_amdgcn_fmed3f(x, -kMostPart, kMostPart) : x);
        out[p] = __builtin_bit_cast(uint16_t, h);
        if (p + 1 < N) x -= static_cast<float>(h);
    }
}
// Three parts that are x exactly, each what fits of the rest (its upper bits): as good as
// the nearest where no product of two of them is left out, and cheaper.
__device__ __forceinline__ void cut_down(float x, uint16_t (&out)[3]) {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        const uint32_t h = __builtin_bit_cast(uint32_t, x) & 0xffff0000u;
        out[p] = static_cast<uint16_t>(h >> 16);
        x -= __builtin_bit_cast(float, h);
    }
}
template <class T, int N>
__device__ __forceinline__ void parts_of(T x, uint16_t (&out)[N]) {
    if constexpr (N == 1) out[0] = __builtin_bit_cast(uint16_t, x);
    else cut<N, sizeof(T) == 4>(static_cast<float>(x), out);
}
__device__ __forceinline__ float part(uint16_t h) { return __builtin_bit_cast(float, static_cast<uint32_t>(h) << 16); }

// The parts of a type's elements, and of what a chunk computes from them.
template <class T> struct Parts;
template <> struct Parts<bf16> { static constexpr int in = 1, made = 2, reach = 2; };
template <> struct Parts<f16> { static constexpr int in = 2, made = 2, reach = 2; };
template <> struct Parts<float> { static constexpr int in = 3, made = 3, reach = 3; };
constexpr int kExact = 3;                  // X is kept, made and read to 24 bits

// The parts of what X is made of and read as, which meet N parts of a plane's element.
template <int N>
__device__ __forceinline__ void exact(float x, uint16_t (&out)[kExact]) {
    if constexpr (N == 1) cut_down(x, out);
    else cut<kExact>(x, out);
}

// sum over pairs of parts (p, q) with p + q < Reach
template <int Reach, int N, int M>
__device__ __forceinline__ F4 product(const H8 (&a)[N], const H8 (&b)[M], F4 c) {
#pragma unroll
    for (int s = Reach - 1; s >= 0; --s)   // the smallest first
#pragma unroll
        for (int p = 0; p < N; ++p)
            if (s - p >= 0 && s - p < M) c = product(a[p], b[s - p], c);
    return c;
}

template <class T>
struct Plane {
    T* at;
    int64_t seq, step, head;
};

template <class T>
struct LinearArgs {
    Plane<const T> a, b, c;
    Plane<T> out;              // at may be NULL
    const float* decay;
    const float* start;        // the state that enters, element (d, e) at d*state_d + e*state_e of a head's; or NULL
    float* end;                // the state that leaves, or NULL
    float* cuts;               // the states of sequences of several segments, [cut][head][width][columns], or NULL
    const void* offsets;
    int64_t seqs, steps, heads, slots, segment, segments;    // segments: of a dense sequence
    int state_d, state_e, width, columns, slices;
    float inner, outer;        // factors of b's products and of the result
    int offsets64, reverse;
};

struct Span {
    int64_t seq, first, length, begin, end;    // tokens [begin, end) of a sequence that starts at row `first`
    int64_t cut;                               // where its states are kept
    bool real, last, whole;                    // whole: the sequence is one segment, which needs none
};
template <class T>
__device__ __forceinline__ int64_t bound_of(const LinearArgs<T>& a, int64_t k) {
    const int64_t v = a.offsets64 ? static_cast<const int64_t*>(a.offsets)[k] : static_cast<const int32_t*>(a.offsets)[k];
    return v < 0 ? 0 : v > a.steps ? a.steps : v;
}
// Where a segment's states are kept.  Of packed sequences, at most one of several segments begins in each `segment` rows, and at
// most one has a later segment that does: two states for each of those runs of rows.
template <class T>
__device__ __forceinline__ int64_t cut_at(const LinearArgs<T>& a, int64_t seq, int64_t first, int64_t segment) {
    return a.offsets ? 2 * (first / a.segment + segment) + (segment == 0) : seq * a.segments + segment;
}
// A workgroup's segment, from its slot.  Packed sequence s's segments have the slots from
// bound(s) / segment + s on: more than it needs by one at most, and none of two sequences.
template <class T>
__device__ __forceinline__ Span span_of(const LinearArgs<T>& a, int64_t slot) {
    Span s;
    int64_t segment;
    if (!a.offsets) {
        s.seq = slot / a.segments;
        segment = slot - s.seq * a.segments;
        s.first = 0;
        s.length = a.steps;
    } else {
        int64_t low = 0, high = a.seqs - 1;
        while (low < high) {
            const int64_t mid = (low + high + 1) / 2;
            if (bound_of(a, mid) / a.segment + mid <= slot) low = mid;
            else high = mid - 1;
        }
        s.seq = low;
        s.first = bound_of(a, low);
        s.length = bound_of(a, low + 1) - s.first;
        if (s.length < 0) s.length = 0;
        segment = slot - (s.first / a.segment + low);
    }
    s.begin = segment * a.segment;
    s.real = segment >= 0 && (segment == 0 || s.begin < s.length);
    s.end = s.begin + a.segment < s.length ? s.begin + a.segment : s.length;
    s.last = s.end == s.length;
    s.whole = s.length <= a.segment;
    s.cut = cut_at(a, s.seq, s.first, segment);
    return s;
}

__device__ __forceinline__ float decay_of(float given) { return given >= 0.0f && given <= 1.0f ? given : NAN; }
// g^n in 64 bits.  A factor of the state that is applied chunk after chunk is held as a
// float and a rest: rounded alone, it would be off the same way every time, and a state that
// remembers n chunks by n roundings.
__device__ __forceinline__ double octaves_of(float g) { return g == 0.0f ? -1e30 : log2(static_cast<double>(g)); }
__device__ __forceinline__ double power(double octaves, int64_t n) { return exp2(octaves * static_cast<double>(n)); }
__device__ __forceinline__ float rest_of(double x) { return static_cast<float>(x - static_cast<double>(static_cast<float>(x))); }

// Where column d of a is staged: the order in which X's rows lie in the lanes, two
// tiles of 16 after each other.
__device__ __forceinline__ int staged(int d) { return (d & ~31) | (d >> 2 & 3) << 3 | (d >> 4 & 1) << 2 | (d & 3); }

// Eight tokens by four channels, a thread's share of a chunk's plane.  A load is always of
// tokens and channels that are there: past a chunk's last token it is that token's, past a
// row's last channels the row's last four.  settle() makes of it what the share is, when
// it is staged: the loads of the next chunk are under way meanwhile.
template <class T> struct Block { Raw<T, 4> x[8]; };
template <class T, int C, bool Narrow>
__device__ __forceinline__ void fetch(Block<T>& x, const T* at, int64_t step, int i, int count, int width) {
    if (Narrow && width < 4) {             // rows without four channels
        at += (i < count ? 0 : count - 1 - i) * step;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            x.x[r] = Raw<T, 4>{at[0], at[width > 1], at[width > 2 ? 2 : 0], static_cast<T>(0.0f)};
            at += i + r + 1 < count ? step : 0;
        }
    } else if (count == C) {
#pragma unroll
        for (int r = 0; r < 8; ++r) x.x[r] = load_raw<T, 4>(at + r * step);
    } else {
        at += (i < count ? 0 : count - 1 - i) * step;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            x.x[r] = load_raw<T, 4>(at);
            at += i + r + 1 < count ? step : 0;
            in_order();                    // this form's addresses are not the other's work
        }
    }
}
template <class R>
__device__ __forceinline__ R moved_down(const R& x, int n) {
    if constexpr (sizeof(R) == 8) {
        return __builtin_bit_cast(R, __builtin_bit_cast(uint64_t, x) >> (16 * n));
    } else {
        const R y = n & 1 ? R{x[1], x[2], x[3], 0.0f} : x;
        return n & 2 ? R{y[2], y[3], 0.0f, 0.0f} : y;
    }
}
// left: the channels of the share that are in the row, 4 at most.
template <class T>
__device__ __forceinline__ void settle(Block<T>& x, int i, int count, int left, int width) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const Raw<T, 4> v = width < 4 ? x.x[r] : moved_down(x.x[r], left > 0 ? 4 - left : 0);
        x.x[r] = i + r < count && left > 0 ? v : splat<T, 4>(static_cast<T>(0.0f));
        if (width < 4)
#pragma unroll
            for (int j = 1; j < 4; ++j)
                if (j >= width) x.x[r][j] = static_cast<T>(0.0f);
    }
}
// Whether a share holds what is no number: the largest of its magnitudes as whole numbers.
template <class T>
__device__ __forceinline__ bool no_number(const Block<T>& x) {
    if constexpr (sizeof(T) == 2) {
        typedef uint16_t H2 __attribute__((ext_vector_type(2)));
        typedef uint32_t W2 __attribute__((ext_vector_type(2)));
        constexpr uint16_t least = std::is_same_v<T, bf16> ? 0x7f80 : 0x7c00;
        H2 most = {0, 0};
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const W2 w = __builtin_bit_cast(W2, x.x[r]) & 0x7fff7fffu;
            const uint32_t one = w[0], two = w[1];
            most = __builtin_elementwise_max(most, __builtin_elementwise_max(__builtin_bit_cast(H2, one), __builtin_bit_cast(H2, two)));
        }
        return most[0] >= least || most[1] >= least;
    } else {
        uint32_t most = 0;
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) most = __builtin_elementwise_max(most, __builtin_bit_cast(uint32_t, static_cast<float>(x.x[r][j])) & 0x7fffffffu);
        return most >= 0x7f800000u;
    }
}
// The channel a share's load begins at, from the one it is of.
__device__ __forceinline__ int loaded(int d, int width) { return d + 4 <= width ? d : width < 4 ? 0 : width - 4; }
__device__ __forceinline__ int left_of(int d, int width) { return width - d < 4 ? width - d : 4; }

// A workgroup of W waves has 16 W columns of c.
template <class T, int DP, int C, int W>
struct Tiles {
    static constexpr int N = Parts<T>::in, M = Parts<T>::made;
    static constexpr int Wide = DP + 8, Long = C + 8;      // rows are 16 bytes apart in the banks
    uint16_t a[N][C][Wide];
    union {
        uint16_t b[N][C][Wide];                            // rows of tokens, until the products of a and b are made
        uint16_t turned[N][DP][Long];                      // rows of channels
    };
    uint16_t c[N][16 * W][Long];
    uint16_t inside[M][C][Long];                           // g^(i-j) a_i . b_j
    float power[C + 1];                                    // g^n
    float rest;                                            // what g^C has below its 24 bits
    float scaled[C];                                       // the same, times what inside is scaled by
    alignas(16) float weight[C];                           // what a token of the chunk has in X'
    int odd;                                               // c holds what is no number
};
// A number told to the compiler anew, so that what is computed from it (the tiles'
// addresses) is computed where it is used, and holds no registers through a loop.
__device__ __forceinline__ int afresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A thread's shares of the planes: of a and b, and of c.
template <int DP, int C, int W>
struct Shares {
    static constexpr int Threads = 64 * W, Slice = 16 * W, Blocks = C / 8 * (DP / 4), SliceBlocks = C / 8 * (Slice / 4);
    static_assert(Blocks <= Threads && SliceBlocks <= Threads, "a share a thread");
    // Where the waves are twice b's, the upper half has a's shares, in the same registers.
    static constexpr bool Halves = 2 * Blocks <= Threads && Blocks % 64 == 0;
    int eight, d, c_eight, c;      // the eight tokens and the four channels
    bool has, has_c;
    __device__ __forceinline__ Shares(int tid, int wave) {
        const int b = Halves ? tid % Blocks : tid, k = tid - (Threads - SliceBlocks);
        eight = b / (DP / 4);
        d = b % (DP / 4) * 4;
        c_eight = k / (Slice / 4);
        c = k % (Slice / 4) * 4;
        has = Blocks % 64 == 0 ? Halves ? wave * 64 < 2 * Blocks : wave * 64 < Blocks : b < Blocks;
        has_c = SliceBlocks % 64 == 0 ? wave * 64 >= Threads - SliceBlocks : k >= 0;
    }
};

// Where eight tokens' unit of a row of channels lies: so that eight lanes that read
// neighbouring rows, or write every fourth one, meet the banks once each.
__device__ __forceinline__ int unit(int d, int eight) { return (eight ^ (d >> 4 & 1)) * 8; }

template <class T, int DP, int C>
__device__ __forceinline__ void stage_rows(uint16_t (&to)[Parts<T>::in][C][DP + 8], const Block<T>& x, int eight, int d) {
    constexpr int N = Parts<T>::in;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        H4 h[N];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint16_t p[N];
            parts_of<T, N>(x.x[r][j], p);
#pragma unroll
            for (int n = 0; n < N; ++n) h[n][j] = p[n];
        }
#pragma unroll
        for (int n = 0; n < N; ++n) *reinterpret_cast<H4*>(&to[n][eight * 8 + r][staged(d)]) = h[n];
    }
}
template <class T, int R, int C>
__device__ __forceinline__ void stage_turned(uint16_t (&to)[Parts<T>::in][R][C + 8], const Block<T>& x, int eight, int d) {
    constexpr int N = Parts<T>::in;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        H8 h[N];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            uint16_t p[N];
            parts_of<T, N>(x.x[r][j], p);
#pragma unroll
            for (int n = 0; n < N; ++n) h[n][r] = p[n];
        }
#pragma unroll
        for (int n = 0; n < N; ++n) *reinterpret_cast<H8*>(&to[n][d + j][unit(d, eight)]) = h[n];
    }
}
template <int N, int R, int W>
__device__ __forceinline__ void take(H8 (&out)[N], const uint16_t (&from)[N][R][W], int row, int at) {
#pragma unroll
    for (int n = 0; n < N; ++n) out[n] = *reinterpret_cast<const H8*>(&from[n][row][at]);
}

template <class T>
struct Walks { LinearArgs<T> walk[kMostWalks]; };

// Workgroup (slot, head, slice) of a walk.  Whole: the walk over a segment; otherwise
// what the segment leaves of its own, for the sum over the segments before another.
template <class T, int DP, int C, int W, bool Whole>
__global__ void __launch_bounds__(64 * W, (DP < 256 && sizeof(T) == 2 && W == 8 ? 4 : 2)) hawk_linear(const Walks<T> walks, const int64_t before) {
    constexpr int N = Parts<T>::in, M = Parts<T>::made, Reach = Parts<T>::reach;
    typedef Shares<DP, C, W> Mine;
    constexpr int Threads = Mine::Threads, Slice = Mine::Slice;
    constexpr bool Halves = Mine::Halves;
    const LinearArgs<T>& a = walks.walk[blockIdx.y];
    __shared__ Tiles<T, DP, C, W> s;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 15, quad = lane >> 4;
    const int64_t pairs = a.slots * a.heads, group = kDies * a.slices;
    // a pair's slices go to one die, whose L2 has a and b for all of them
    const int64_t id = before + blockIdx.x, pair = id / group * kDies + id % kDies;
    const int slice = static_cast<int>(id / kDies % a.slices);
    if (pair >= pairs) return;
    const int64_t slot = pair / a.heads, head = pair - slot * a.heads;
    const Span span = span_of(a, slot);
    if (!span.real || (!Whole && span.last)) return;
    const float g = decay_of(a.decay[head]);
    const double octaves = octaves_of(g);
    const int e0 = slice * Slice, columns = a.columns - e0;
    const int64_t plane = static_cast<int64_t>(a.width) * a.columns;
    const int64_t state = (span.seq * a.heads + head) * plane, mark = (span.cut * a.heads + head) * plane;
    const int way = a.reverse ? -1 : 1;
    const int64_t row0 = a.reverse ? span.first + span.length - 1 : span.first;
    for (int n = tid; n <= C; n += Threads) {
        const double p = power(octaves, n);
        s.power[n] = static_cast<float>(p);
        if (n < C) s.scaled[n] = s.power[n] * (a.inner * a.outer);
        else s.rest = rest_of(p);
    }

    // X: tile i holds rows 16 i + 4 quad .. + 3 of column e
    F4 X[DP / 16];
    const int e = e0 + wave * 16 + col;
    const bool joined = Whole && !span.whole;              // (such a call has cuts)
    const float* enters = joined ? a.cuts + mark : Whole && a.start ? a.start + state : nullptr;
    const int enters_d = joined ? a.columns : a.state_d, enters_e = joined ? 1 : a.state_e;
    const float once = joined || a.reverse || span.length == 0 ? 1.0f : g;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) X[i] = F4{0.0f, 0.0f, 0.0f, 0.0f};
    if (enters)
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int d = i * 16 + quad * 4 + k;
                const float x = enters[(d < a.width ? d : 0) * enters_d + (e < a.columns ? e : 0) * enters_e];
                X[i][k] = d < a.width && e < a.columns ? x * once : 0.0f;
            }

    // this thread's shares, and where the chunk to be loaded has them
    const bool upper = Halves && wave * 64 >= Mine::Blocks;
    const Mine at_first(tid, wave);
    Block<T> xa, xb, xc;
    auto load_chunk = [&](const Mine& my, int64_t at) {
        const int count = static_cast<int>(span.end - at < C ? span.end - at : C);
        auto row = [&](const Plane<const T>& p) { return p.at + span.seq * p.seq + head * p.head + (row0 + way * at) * p.step; };
        if (my.has && (Whole || !upper)) {
            const int64_t step_a = way * a.a.step, step_b = way * (upper ? a.a.step : a.b.step);
            const int d = loaded(my.d, a.width);
            if (Whole && !Halves) fetch<T, C, DP == 32>(xa, row(a.a) + my.eight * 8 * step_a + d, step_a, my.eight * 8, count, a.width);
            fetch<T, C, DP == 32>(xb, row(upper ? a.a : a.b) + my.eight * 8 * step_b + d, step_b, my.eight * 8, count, a.width);
        }
        if (my.has_c) {
            const int64_t step = way * a.c.step;
            fetch<T, C, W == 4>(xc, row(a.c) + my.c_eight * 8 * step + loaded(e0 + my.c, a.columns), step, my.c_eight * 8, count, a.columns);
        }
    };
    if (span.begin < span.end) load_chunk(at_first, span.begin);
    for (int64_t at = span.begin; at < span.end; at += C) {
        const int count = static_cast<int>(span.end - at < C ? span.end - at : C);
        // the tokens that X' decays by; one less where the state leaves a forward walk
        const int n = count - (Whole && !a.reverse && span.last && at + C >= span.end ? 1 : 0);
        __syncthreads();
        if (tid == 0) s.odd = 0;
        if (at == span.begin || n < C)
            for (int j = tid; j < C; j += Threads) s.weight[j] = s.power[j < n ? n - j : 0] * a.inner;
        const int now = afresh(tid), col = now & 15, quad = now >> 4 & 3;
        const Mine my(now, wave);
        if (my.has && (Whole || !upper)) {
            if (count < C || a.width < DP) {
                if (Whole && !Halves) settle(xa, my.eight * 8, count, left_of(my.d, a.width), a.width);
                settle(xb, my.eight * 8, count, left_of(my.d, a.width), a.width);
            }
            if constexpr (Whole) {
                if (!Halves) stage_rows<T, DP, C>(s.a, xa, my.eight, my.d);
                stage_rows<T, DP, C>(upper ? s.a : s.b, xb, my.eight, my.d);
            } else {
                stage_turned<T, DP, C>(s.turned, xb, my.eight, my.d);
            }
        }
        bool odd = false;
        if (my.has_c) {
            if (count < C || columns < Slice) settle(xc, my.c_eight * 8, count, left_of(e0 + my.c, a.columns), a.columns);
            stage_turned<T, Slice, C>(s.c, xc, my.c_eight, my.c);
            if (Whole) odd = no_number(xc);
        }
        __syncthreads();
        if constexpr (Whole) {
            if (odd) s.odd = 1;
            // tiles of 16 x 16: inside = g^(i-j) a_i . b_j, rows j, columns i >= j
            constexpr int Side = C / 16, Pairs = Side * (Side + 1) / 2;
            for (int t = wave; t < Pairs; t += W) {
                int ti = 0;
                while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
                const int tj = t - ti * (ti + 1) / 2;
                F4 p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int d = 0; d < DP; d += 32) {
                    H8 fa[N], fb[N];
                    take(fa, s.a, ti * 16 + col, d + quad * 8);
                    take(fb, s.b, tj * 16 + col, d + quad * 8);
                    p = product<Reach>(fb, fa, p);
                    in_order();
                }
                const int i = ti * 16 + col, j = tj * 16 + quad * 4;
                H4 h[M];
                float v[4];
                if (ti > tj) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = p[k] * s.scaled[i - j - k];
                } else {                                   // what p is past the diagonal is not looked at
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = i >= j + k ? p[k] * s.scaled[i >= j + k ? i - j - k : 0] : 0.0f;
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint16_t q[M];
                    cut<M>(v[k], q);
#pragma unroll
                    for (int n = 0; n < M; ++n) h[n][k] = q[n];
                }
#pragma unroll
                for (int n = 0; n < M; ++n) *reinterpret_cast<H4*>(&s.inside[n][i][j]) = h[n];
                // a block of 32 tokens j is taken whole: its half past the diagonal is 0
                if (ti == tj && (ti & 1) == 0) {
#pragma unroll
                    for (int n = 0; n < M; ++n) *reinterpret_cast<H4*>(&s.inside[n][i][j + 16]) = H4{0, 0, 0, 0};
                }
            }
            __syncthreads();
            if (my.has && !upper) stage_turned<T, DP, C>(s.turned, xb, my.eight, my.d);
        }
        if (at + C < span.end) load_chunk(my, at + C);
        if constexpr (Whole) {
            // out^T: rows e, columns i.  First a X, in X's own order of channels.
            F4 o[C / 16];
#pragma unroll
            for (int t = 0; t < C / 16; ++t) o[t] = F4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int d = 0; d < DP; d += 32) {
                H8 fx[kExact];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    uint16_t q[kExact];
                    exact<N>(X[d / 16 + k / 4][k & 3], q);
#pragma unroll
                    for (int n = 0; n < kExact; ++n) fx[n][k] = q[n];
                }
#pragma unroll
                for (int t = 0; t < C / 16; ++t) {
                    H8 fa[N];
                    take(fa, s.a, t * 16 + col, d + quad * 8);
                    o[t] = product<kExact>(fx, fa, o[t]);
                }
                in_order();
            }
#pragma unroll
            for (int t = 0; t < C / 16; ++t) {
                const float g = s.power[t * 16 + col] * a.outer;
#pragma unroll
                for (int k = 0; k < 4; ++k) o[t][k] *= g;
            }
            if (!s.odd) {
#pragma unroll
                for (int j = 0; j < C; j += 32) {
                    H8 fc[N];
                    take(fc, s.c, wave * 16 + col, unit(wave * 16 + col, j / 8 + quad));
#pragma unroll
                    for (int t = j / 16; t < C / 16; ++t) {
                        H8 fp[M];
                        take(fp, s.inside, t * 16 + col, j + quad * 8);
                        o[t] = product<Reach>(fc, fp, o[t]);
                    }
                    in_order();
                }
            } else {
                // An infinity or a NaN in c, times the 0 of a token before it, would be a
                // NaN there: such a chunk is summed term by term.
#pragma unroll 1
                for (int j = 0; j < C; ++j) {
                    float c[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int r = wave * 16 + quad * 4 + k;
                        c[k] = 0.0f;
#pragma unroll
                        for (int n = N - 1; n >= 0; --n) c[k] += part(s.c[n][r][unit(r, j / 8) + (j & 7)]);
                    }
#pragma unroll
                    for (int t = 0; t < C / 16; ++t) {
                        float p = 0.0f;
#pragma unroll
                        for (int n = M - 1; n >= 0; --n) p += part(s.inside[n][t * 16 + col][j]);
                        if (j <= t * 16 + col)
#pragma unroll
                            for (int k = 0; k < 4; ++k) o[t][k] = fused(p, c[k], o[t][k]);
                    }
                }
            }
            const int left = columns - (wave * 16 + quad * 4);
            if (a.out.at && left > 0) {
                T* to = a.out.at + span.seq * a.out.seq + head * a.out.head + (row0 + way * (at + col)) * a.out.step + e0 + wave * 16 + quad * 4;
#pragma unroll
                for (int t = 0; t < C / 16; ++t) {
                    if (t * 16 + col >= count) continue;
                    const float x[4] = {o[t][0], o[t][1], o[t][2], o[t][3]};
                    T* here = to + (way * t * 16) * a.out.step;
                    if (left >= 4) {
                        store<T, 4>(here, x);
                    } else {
#pragma unroll
                        for (int k = 0; k < 3; ++k)
                            if (k < left) here[k] = static_cast<T>(x[k]);
                    }
                }
            }
            __syncthreads();
        }
        // X' = g^n X + sum_j g^(n-j) b_j c_j
        const float keep = s.power[n], rest = n == C ? s.rest : 0.0f;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) X[i][k] = fused(keep, X[i][k], rest * X[i][k]);
#pragma unroll
        for (int j = 0; j < C; j += 32) {
            H8 fc[N], fw[kExact];
            take(fc, s.c, wave * 16 + col, unit(wave * 16 + col, j / 8 + quad));
            F4 w[2];
            w[0] = *reinterpret_cast<const F4*>(&s.weight[j + quad * 8]);
            w[1] = *reinterpret_cast<const F4*>(&s.weight[j + quad * 8 + 4]);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                float c = part(fc[N - 1][k]);
#pragma unroll
                for (int p = N - 2; p >= 0; --p) c += part(fc[p][k]);
                uint16_t q[kExact];
                exact<N>(w[k / 4][k & 3] * c, q);
#pragma unroll
                for (int p = 0; p < kExact; ++p) fw[p][k] = q[p];
            }
            in_order();
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                H8 fb[N];
                take(fb, s.turned, i * 16 + col, unit(i * 16 + col, j / 8 + quad));
                X[i] = product<kExact>(fb, fw, X[i]);
                if (i & 1) in_order();
            }
        }
    }
    float* leaves = !Whole ? a.cuts + mark : a.end && span.last ? a.end + state : nullptr;
    const int leaves_d = Whole ? a.state_d : a.columns, leaves_e = Whole ? a.state_e : 1;
    if (leaves && e < a.columns)
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int d = i * 16 + quad * 4 + k;
                if (d < a.width) leaves[d * leaves_d + e * leaves_e] = X[i][k];
            }
}

// Each segment's own state becomes the one that enters it: kAhead segments are read at a
// time, before what waits for the one before.
template <class T>
__global__ void __launch_bounds__(kJoinThreads) hawk_linear_join(const Walks<T> walks) {
    constexpr int kAhead = 8;
    const LinearArgs<T>& a = walks.walk[blockIdx.y];
    const int plane = a.width * a.columns, blocks = (plane + kJoinThreads - 1) / kJoinThreads;
    const int64_t total = a.seqs * a.heads * blocks;
    for (int64_t id = blockIdx.x; id < total; id += gridDim.x) {
        const int64_t pair = id / blocks;
        const int i = static_cast<int>(id - pair * blocks) * kJoinThreads + static_cast<int>(threadIdx.x);
        if (i >= plane) continue;
        const int64_t seq = pair / a.heads, head = pair - seq * a.heads;
        const int64_t first = a.offsets ? bound_of(a, seq) : 0, length = (a.offsets ? bound_of(a, seq + 1) : a.steps) - first;
        if (length <= a.segment) continue;
        const int64_t segments = (length + a.segment - 1) / a.segment;
        const float g = decay_of(a.decay[head]);
        const double whole = power(octaves_of(g), a.segment);
        const float keep = static_cast<float>(whole), rest = rest_of(whole);
        auto joined = [&](float x, float own) { return fused(keep, x, fused(rest, x, own)); };
        const int d = i / a.columns, e = i - d * a.columns;
        float x = 0.0f;
        if (a.start) x = a.start[pair * plane + d * a.state_d + e * a.state_e] * (a.reverse ? 1.0f : g);
        float* at = a.cuts + (cut_at(a, seq, first, 0) * a.heads + head) * plane + i;
        const float leaves = *at;
        *at = x;
        x = joined(x, leaves);
        at = a.cuts + (cut_at(a, seq, first, 1) * a.heads + head) * plane + i;
        const int64_t step = (a.offsets ? 2 : 1) * a.heads * plane;
        for (int64_t t = 1; t < segments; t += kAhead, at += kAhead * step) {
            float own[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) own[k] = t + k + 1 < segments ? at[k * step] : 0.0f;   // (the last leaves nothing here)
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (t + k >= segments) break;
                at[k * step] = x;
                x = joined(x, own[k]);
            }
        }
    }
}

// ---- few tokens ------------------------------------------------------------------------
//
// S_t = g S_(t-1) + k_t v_t^T and o_t = scale q_t S_t as they stand: the states' traffic is
// the work.  A workgroup has 64 columns of a head's state in registers, 16 groups of 16
// lanes, each every 16th row, a lane four columns of it.

constexpr int kFewTokens = 8, kStepThreads = 256, kStepColumns = 64, kGroups = 16;
// The four numbers at column c of a row of `columns`, and the same written.
__device__ __forceinline__ F4 four(const float* row, int c, int columns) {
    F4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c + 4 <= columns) {
        x = load_raw<float, 4>(row + c);
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (c + j < columns) x[j] = row[c + j];
    }
    return x;
}
__device__ __forceinline__ void put_four(float* row, int c, int columns, const F4& x) {
    if (c + 4 <= columns) {
        store_raw<float, 4>(row + c, x);
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (c + j < columns) row[c + j] = x[j];
    }
}
template <class T, int Rows>
__global__ void __launch_bounds__(kStepThreads, Rows <= 8 ? 6 : 4) hawk_linear_steps(const LinearArgs<T> a, const int64_t before) {
    __shared__ float q[kMostWidth], k[kMostWidth], v[kStepColumns];
    __shared__ F4 sums[kGroups][kStepColumns / 4];
    const int tid = threadIdx.x, lane = tid % 16, group = tid / 16;
    const int64_t id = before + blockIdx.x, pair = id / a.slices, seq = pair / a.heads, head = pair - seq * a.heads;
    const int e0 = static_cast<int>(id - pair * a.slices) * kStepColumns, c = e0 + lane * 4;
    const int64_t state = pair * (static_cast<int64_t>(a.width) * a.columns);
    const float g = decay_of(a.decay[head]);
    F4 S[Rows];
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        const int d = group + r * kGroups;
        S[r] = F4{0.0f, 0.0f, 0.0f, 0.0f};
        if (a.start && d < a.width) S[r] = four(a.start + state + d * a.columns, c, a.columns);
    }
    for (int64_t t = 0; t < a.steps; ++t) {
        __syncthreads();
        if (tid < a.width) {
            q[tid] = static_cast<float>(a.a.at[seq * a.a.seq + t * a.a.step + head * a.a.head + tid]);
            k[tid] = static_cast<float>(a.b.at[seq * a.b.seq + t * a.b.step + head * a.b.head + tid]);
        }
        if (tid < kStepColumns) v[tid] = e0 + tid < a.columns ? static_cast<float>(a.c.at[seq * a.c.seq + t * a.c.step + head * a.c.head + e0 + tid]) : 0.0f;
        __syncthreads();
        const F4 x = *reinterpret_cast<const F4*>(&v[lane * 4]);
        F4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < Rows; ++r) {
            const int d = group + r * kGroups;
            if (d >= a.width) continue;
            const float kd = k[d], qd = q[d];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                S[r][j] = fused(g, S[r][j], kd * x[j]);
                sum[j] = fused(qd, S[r][j], sum[j]);
            }
        }
        if (!a.out.at) continue;
        sums[group][lane] = sum;
        __syncthreads();
        if (tid < kStepColumns && e0 + tid < a.columns) {
            float o = 0.0f;
#pragma unroll
            for (int r = 0; r < kGroups; ++r) o += reinterpret_cast<const float*>(sums[r])[tid];
            a.out.at[seq * a.out.seq + t * a.out.step + head * a.out.head + e0 + tid] = static_cast<T>(o * a.outer);
        }
    }
    if (!a.end) return;
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        const int d = group + r * kGroups;
        if (d < a.width) put_four(a.end + state + d * a.columns, c, a.columns, S[r]);
    }
}

// ---- host ----------------------------------------------------------------------------

// One walk: which planes it reads as a, b and c.
struct Walk {
    const hk_head_plane *a, *b, *c, *out;
    const float* start;
    float* end;
    int width, columns, state_d, state_e, reverse;
    float inner, outer;
};
int walks_of(const hk_linear_attention_job& j, int vjp, Walk (&w)[kMostWalks]) {
    const int K = j.keys, V = j.values;
    int n = 0;
    if (!vjp) {
        w[n++] = Walk{&j.q, &j.k, &j.v, &j.o, j.h0, j.last, K, V, V, 1, 0, 1.0f, j.scale};
        return n;
    }
    if (j.bar_q.data) w[n++] = Walk{&j.bar_o, &j.v, &j.k, &j.bar_q, j.h0, nullptr, V, K, 1, V, 0, 1.0f, j.scale};
    if (j.bar_k.data) w[n++] = Walk{&j.v, &j.bar_o, &j.q, &j.bar_k, j.bar_last, nullptr, V, K, 1, V, 1, j.scale, 1.0f};
    if (j.bar_v.data || j.bar_h0) w[n++] = Walk{&j.k, &j.q, &j.bar_o, &j.bar_v, j.bar_last, j.bar_h0, K, V, V, 1, 1, j.scale, 1.0f};
    return n;
}

// The columns of a workgroup: 128 where there are more than 64, which shares what is
// staged of a and b, and the products of the two, among twice the waves.
int slice_of(int columns) { return columns > 64 ? 128 : 64; }
int bucket_of(int width) { return width <= 32 ? 32 : width <= 64 ? 64 : width <= 128 ? 128 : 256; }

// Walks of one form are one launch: those like w[i] of the n.
bool alike(const Walk& a, const Walk& b) { return bucket_of(a.width) == bucket_of(b.width) && slice_of(a.columns) == slice_of(b.columns); }
int beside_of(const Walk* w, int n, int i) {
    int count = 0;
    for (int k = 0; k < n; ++k) count += alike(w[i], w[k]);
    return count;
}

// The tokens of a segment.  A launch whose whole walks are enough for most of the units
// goes uncut: what cutting costs, the segments' own states first, is about half a walk
// (4096 tokens of 128 bfloat16 channels: 192 walks whole 378 us, cut 436; 144: 376 and 420;
// 96: 373 and 213).
// Otherwise, and where sequences are of any length (up to eight times as many workgroups of
// them), as many segments as give each unit two workgroups of eight waves, or four of four,
// of two chunks at least.
struct Cut { int64_t segment, segments, slots, cuts; };
Cut cut_of(const hk_linear_attention_job& j, int columns, int walks) {
    const int64_t slices = (columns + slice_of(columns) - 1) / slice_of(columns), most = j.steps > 1 ? j.steps : 1;
    const int64_t tokens = j.offsets ? j.steps : j.seqs * j.steps, beside = j.heads * slices * walks;
    const int64_t full = (slice_of(columns) == 64 ? 4 : 2) * kUnits, least = j.dtype == HK_BF16 ? 128 : 64;
    int64_t each = tokens / full * beside + 1;
    each = each < least ? least : (each + 63) / 64 * 64;
    if (j.seqs * beside >= (j.offsets ? 8 * full : full * 3 / 8)) each = most;
    if (each >= most) return j.offsets ? Cut{most, 1, j.seqs + 1, 0} : Cut{most, 1, j.seqs, 0};
    if (j.offsets) return Cut{each, 0, j.steps / each + j.seqs, 2 * (j.steps / each + 1)};
    const int64_t n = (j.steps + each - 1) / each;
    return Cut{each, n, n * j.seqs, n * j.seqs};
}
size_t cuts_bytes(const hk_linear_attention_job& j, const Walk& w, int walks) {
    const Cut c = cut_of(j, w.columns, walks);
    return static_cast<size_t>(c.cuts) * static_cast<size_t>(j.heads) * w.width * w.columns * sizeof(float);
}

template <class T>
Plane<const T> in(const hk_head_plane& p) { return {static_cast<const T*>(p.data), p.seq, p.step, p.head}; }

int launched(const char* what) {
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? HK_OK : hawk_internal::set_hip_error(what, err);
}

template <class T, int DP, int C, int W>
void launch(const Walks<T>& walks, int n, hipStream_t stream) {
    int64_t total = 0, joins = 0;
    const bool cuts = walks.walk[0].cuts;                  // walks of one form have their sequences cut alike
    for (int i = 0; i < n; ++i) {
        const LinearArgs<T>& a = walks.walk[i];
        const int64_t each = (a.slots * a.heads + kDies - 1) / kDies * kDies * a.slices;
        const int64_t plane = static_cast<int64_t>(a.width) * a.columns, parts = a.seqs * a.heads * ((plane + kJoinThreads - 1) / kJoinThreads);
        total = each > total ? each : total;
        joins = parts > joins ? parts : joins;
    }
    const int64_t most = 1 << 20;
    auto each = [&](auto kernel) {                         // launches stay below 2^32 threads
        for (int64_t before = 0; before < total; before += most) {
            const int64_t left = total - before;
            hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(left < most ? left : most), static_cast<unsigned>(n)), dim3(64 * W), 0, stream,
                               walks, before);
        }
    };
    if (cuts) {
        each(hawk_linear<T, DP, C, W, false>);
        hipLaunchKernelGGL((hawk_linear_join<T>), dim3(static_cast<unsigned>(joins < most ? joins : most), static_cast<unsigned>(n)),
                           dim3(kJoinThreads), 0, stream, walks);
    }
    each(hawk_linear<T, DP, C, W, true>);
}
template <class T, int W>
void launch(const Walks<T>& walks, int n, int bucket, hipStream_t stream) {
    // more tokens a chunk cost more products inside it, fewer more passes over X
    constexpr int C = Parts<T>::in == 1 ? 64 : 32;
    if (bucket == 32) launch<T, 32, C, W>(walks, n, stream);
    else if (bucket == 64) launch<T, 64, C, W>(walks, n, stream);
    else if (bucket == 128) launch<T, 128, C, W>(walks, n, stream);
    else launch<T, 256, 32, W>(walks, n, stream);
}

template <class T>
LinearArgs<T> args_of(const hk_linear_attention_job& j, const Walk& w, int walks) {
    LinearArgs<T> a;
    a.a = in<T>(*w.a);
    a.b = in<T>(*w.b);
    a.c = in<T>(*w.c);
    a.out = Plane<T>{static_cast<T*>(w.out->data), w.out->seq, w.out->step, w.out->head};
    if (j.offsets) a.a.seq = a.b.seq = a.c.seq = a.out.seq = 0;    // packed planes have no such axis, whatever the job says
    a.decay = j.decay;
    a.start = w.start;
    a.end = w.end;
    a.offsets = j.offsets;
    a.seqs = j.seqs;
    a.steps = j.steps;
    a.heads = j.heads;
    const Cut c = cut_of(j, w.columns, walks);
    a.segment = c.segment;
    a.segments = c.segments;
    a.slots = c.slots;
    a.state_d = w.state_d;
    a.state_e = w.state_e;
    a.width = w.width;
    a.columns = w.columns;
    a.slices = (w.columns + slice_of(w.columns) - 1) / slice_of(w.columns);
    a.inner = w.inner;
    a.outer = w.outer;
    a.offsets64 = j.offsets64;
    a.reverse = w.reverse;
    a.cuts = nullptr;
    return a;
}

// Dense sequences of up to kFewTokens tokens, forward: as they stand, by vector arithmetic
// (64 x 16 heads of 128 x 128, one token: 29.7 us, 42.3 by chunks; its states take 20.7).
template <class T>
int steps(const hk_linear_attention_job& j, const Walk& w, hipStream_t stream) {
    LinearArgs<T> a = args_of<T>(j, w, 1);
    a.slices = (w.columns + kStepColumns - 1) / kStepColumns;
    const int64_t total = j.seqs * j.heads * a.slices, most = 1 << 22;
    auto each = [&](auto kernel) {
        for (int64_t before = 0; before < total; before += most) {
            const int64_t left = total - before;
            hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(left < most ? left : most)), dim3(kStepThreads), 0, stream, a, before);
        }
    };
    if (w.width <= 4 * kGroups) each(hawk_linear_steps<T, 4>);
    else if (w.width <= 8 * kGroups) each(hawk_linear_steps<T, 8>);
    else each(hawk_linear_steps<T, 16>);
    return launched("hawk_linear_steps launch");
}

// Every walk, those of one form in one launch.
template <class T>
int all(const hk_linear_attention_job& j, int vjp, void* scratch, hipStream_t stream) {
    Walk w[kMostWalks];
    const int n = walks_of(j, vjp, w);
    if (!vjp && !j.offsets && j.steps <= kFewTokens) return steps<T>(j, w[0], stream);
    char* room = static_cast<char*>(scratch);
    bool done[kMostWalks] = {};
    for (int i = 0; i < n; ++i) {
        if (done[i]) continue;
        Walks<T> walks = {};
        int count = 0;
        const int beside = beside_of(w, n, i);
        for (int k = i; k < n; ++k) {
            if (done[k] || !alike(w[i], w[k])) continue;
            done[k] = true;
            walks.walk[count] = args_of<T>(j, w[k], beside);
            const size_t bytes = cuts_bytes(j, w[k], beside);
            if (bytes) walks.walk[count].cuts = reinterpret_cast<float*>(room);
            room += bytes;
            ++count;
        }
        const int bucket = bucket_of(w[i].width);
        if (slice_of(w[i].columns) == 64) launch<T, 4>(walks, count, bucket, stream);
        else launch<T, 8>(walks, count, bucket, stream);
        const int rc = launched("hawk_linear launch");
        if (rc != HK_OK) return rc;
    }
    return HK_OK;
}

int run(const hk_linear_attention_job* job, int vjp, void* scratch, void* stream) {
    using hawk_internal::set_error;
    if (!job) return set_error(HK_EVALUE, "hk_linear_attention: a job is required");
    const hk_linear_attention_job& j = *job;
    if (j.seqs < 0 || j.steps < 0 || j.heads < 0) return set_error(HK_EVALUE, "hk_linear_attention: sizes must be >= 0");
    if (j.keys < 1 || j.keys > kMostWidth || j.values < 1 || j.values > kMostWidth)
        return set_error(HK_EVALUE, "hk_linear_attention: a head has 1 to 256 channels");
    if (j.dtype != HK_F32 && j.dtype != HK_BF16 && j.dtype != HK_F16)
        return set_error(HK_EVALUE, "hk_linear_attention: the planes' element type is 32-bit or 16-bit");
    if (j.seqs == 0 || j.heads == 0) return HK_OK;
    const bool tokens = j.steps > 0;
    if (!j.decay || (tokens && (!j.q.data || !j.k.data || !j.v.data || (vjp && !j.bar_o.data))))
        return set_error(HK_EVALUE, "hk_linear_attention: a plane is missing");
    if (j.steps > INT64_MAX / 16 / j.seqs / j.heads)
        return set_error(HK_EVALUE, "hk_linear_attention: the planes exceed the grid limit");
    if (hk_linear_attention_scratch_bytes(job, vjp) && !scratch)
        return set_error(HK_EVALUE, "hk_linear_attention: scratch is required");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (j.dtype == HK_F32) return all<float>(j, vjp, scratch, s);
    return j.dtype == HK_BF16 ? all<bf16>(j, vjp, scratch, s) : all<f16>(j, vjp, scratch, s);
}

}  // namespace

extern "C" size_t hk_linear_attention_scratch_bytes(const hk_linear_attention_job* job, int32_t vjp) {
    if (!job || job->seqs <= 0 || job->steps <= 0 || job->heads <= 0) return 0;
    if (job->keys < 1 || job->keys > kMostWidth || job->values < 1 || job->values > kMostWidth) return 0;
    Walk w[kMostWalks];
    const int n = walks_of(*job, vjp, w);
    size_t bytes = 0;
    for (int i = 0; i < n; ++i) bytes += cuts_bytes(*job, w[i], beside_of(w, n, i));
    return bytes;
}

extern "C" int hk_linear_attention(const hk_linear_attention_job* job, void* scratch, void* stream) { return run(job, 0, scratch, stream); }
extern "C" int hk_linear_attention_vjp(const hk_linear_attention_job* job, void* scratch, void* stream) { return run(job, 1, scratch, stream); }
