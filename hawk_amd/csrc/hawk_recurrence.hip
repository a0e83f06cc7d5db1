// hawk_recurrence.hip — gated linear recurrences h_t = a_t h_(t-1) + b_t over
// long sequences, and their reverse-mode derivative, on gfx950.
//
// The mathematics.  A run of steps maps the state before it to the state
// after it by h -> P h + H, with P the product of the run's gates and H its
// result from a zero state; two runs in order join to (P1 P2, H2 + P2 H1).  So
// a sequence is cut into tiles, every thread folds K steps of V channels in
// registers, the threads of a tile join theirs, the tiles join theirs, and a
// step's state is its local result plus its local product times the state that
// entered.  The derivative is the same recurrence run the other way: C_t =
// a_t (bar_h_t + C_(t+1)) has the gate a_t and the input a_t bar_h_t.
//
// The tiles join theirs in one pass over the data, by the published decoupled
// look-back (Merrill and Garland, Single-pass parallel prefix scan with decoupled
// look-back, 2016): each publishes its run, then folds those published before it.
//
// A gate of 0 cuts, and so does the first row of a packed sequence: products
// and their use take 0 times anything as 0 (cutmul), so neither an infinity
// nor a NaN passes a cut.  States are held in 32 bits (64 for double planes), and
// products as a mantissa of as many and an exponent of 32 (Gain), so that what a
// state passes on is right also where the gates' product alone is no number of the
// type: gates of 2 over 128 steps, or of 1/2 over 150.

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

// A workgroup's most threads.  Where lanes lie along the steps a long sequence
// takes large tiles, since each tile has one state to wait for (64 rows of 2^20
// float steps: 238 us in tiles of 256 threads, 211 of 512, 232 of 1024).
template <class T, int Dir> constexpr int kMost = Dir == 0 ? kThreads : 512;

template <class T>
struct Plane {
    T* data;
    int64_t seq, step, chan;
};

// What tiles tell each other goes through words that say themselves whether
// they are written: all bits set is "not yet", and a NaN is published as the
// one quiet NaN, which is not that.  So relaxed accesses at the GPU's scope are
// enough, with no order among them.
template <class A> struct Word;
template <> struct Word<float> { typedef uint32_t type; static constexpr uint32_t kNan = 0x7fc00000u; };
template <> struct Word<double> { typedef uint64_t type; static constexpr uint64_t kNan = 0x7ff8000000000000ull; };

template <class T>
struct RecArgs {
    Plane<T> gate, x, h, bar_h, bar_gate, bar_x;
    const Acc<T>* init;       // the state that enters the scan: h0, or bar_last
    const Acc<T>* h0;         // the derivative's h_(-1)
    Acc<T>* fin;              // the state that leaves it: last, or bar_h0
    const void* offsets;
    uint32_t* counter;        // a strip's: hands its chunks out in order
    uint64_t* agg;                         // [chunk][states]: each tile's (P's mantissa, H)
    uint16_t* agg_exp;                     // [chunk][states]: and P's exponent
    typename Word<Acc<T>>::type* state;    // [chunk][states]: the state that leaves each tile
    uint32_t* flag;                        // [strip][chunk]: 1 once that state is written
    int64_t seqs, chans, cols, states;   // states: those of one tile row, seqs * chans (packed: chans)
    int steps, groups;        // groups: threads across a row's channels
    int lcol, ncol, nt, strips, chunks;   // a tile: ncol columns (Dir 0: 2^lcol) by nt threads along the steps
    int counter_step;
    int rev, offsets64;       // rev: scan step i is row steps - 1 - i (packed planes)
};

// A packed sequence's first row; there are at most 2^30 rows.
__device__ __forceinline__ int cut_at(const void* offsets, int wide, int s) {
    return wide ? static_cast<int>(static_cast<const int64_t*>(offsets)[s]) : static_cast<const int32_t*>(offsets)[s];
}
// The same of an s that is one for the workgroup: a scalar load, which does not
// wait for the tile's loads.  (No kernel here writes offsets.)
__device__ __forceinline__ int cut_at_scalar(const void* offsets, int wide, int s) {
    typedef const __attribute__((address_space(4))) int64_t* Wide;
    typedef const __attribute__((address_space(4))) int32_t* Narrow;
    return wide ? static_cast<int>(((Wide)(offsets))[s]) : ((Narrow)(offsets))[s];
}

// The sequence of [low, high] whose rows hold `row`: the last one that starts at
// or before it.
template <class Cut>
__device__ __forceinline__ int sequence_of(Cut cut, int low, int high, int row) {
    while (low < high) {
        const int mid = low + (high - low + 1) / 2;
        if (cut(mid) <= row) low = mid;
        else high = mid - 1;
    }
    return low;
}

// One thread's K steps of V channels, left in the plane's type.  Dir 0: V
// consecutive channels a step, each step a load of its own; otherwise one
// channel, K steps in one load where the steps are contiguous (Dir 1, or -1
// where the scan runs down the axis).  A step past the end repeats the last
// one's address, so every load is issued without a branch.
template <class T, int V, int K, int Dir, bool Stream>
__device__ __forceinline__ void tile_load(const Plane<T>& p, int64_t s, int64_t c, int row0, int steps,
                                          Raw<T, V> (&out)[K]) {
    const T* base = p.data + s * p.seq + c * p.chan;
    if constexpr (Dir == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int row = row0 + k < steps ? row0 + k : steps - 1;
            out[k] = load_raw<T, V, Stream>(base + row * p.step);
        }
    } else {
        if (row0 + K <= steps) {
            const Raw<T, K> flat = load_raw<T, K>(Dir > 0 ? base + row0 : base - (row0 + K - 1));
#pragma unroll
            for (int k = 0; k < K; ++k) out[k] = flat[Dir > 0 ? k : K - 1 - k];
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int row = row0 + k < steps ? row0 + k : steps - 1;
                out[k] = Dir > 0 ? base[row] : base[-row];
            }
        }
    }
}

// Stores step k of a tile at p (the thread's first step) if it exists; `skip`
// leading channels belong to the neighbouring thread.
template <class T, int V, bool Stream>
__device__ __forceinline__ void row_store(T* p, int64_t step, int k, int rows, int skip, const Raw<T, V>& x) {
    if (k >= rows) return;
    T* to = p + k * step;
    if (skip == 0) {
        store_raw<T, V, Stream>(to, x);
    } else if constexpr (V > 1) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v >= skip) to[v] = x[v];
    }
}
// The same for all steps of a thread whose steps are contiguous.
template <class T, int K, int Dir>
__device__ __forceinline__ void run_store(T* p, int rows, const T (&x)[K]) {
    if (rows == K) {
        Raw<T, K> flat;
#pragma unroll
        for (int k = 0; k < K; ++k) flat[Dir > 0 ? k : K - 1 - k] = x[k];
        *reinterpret_cast<typename VecOf<T, K>::loose*>(Dir > 0 ? p : p - (K - 1)) = flat;
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k < rows) *(Dir > 0 ? p + k : p - k) = x[k];
    }
}

template <class A>
__device__ __forceinline__ void publish(typename Word<A>::type* at, A x) {
    typedef typename Word<A>::type W;
    W w = __builtin_bit_cast(W, x);
    if (!(x == x)) w = Word<A>::kNan;
    __hip_atomic_store(at, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class A>
__device__ __forceinline__ bool read(const typename Word<A>::type* at, A& x) {
    typedef typename Word<A>::type W;
    const W w = __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    x = __builtin_bit_cast(A, w);
    return w != ~W(0);
}
// A word that its tile has written, or is about to: that tile has begun (see
// the order of tiles below), so the wait ends.  Where it cannot (two streams
// worked in one scratch) it ends after kLooks looks, seconds, with the unwritten
// word, which is a NaN.
constexpr int kLooks = 1 << 22;
template <class A>
__device__ __forceinline__ A await(const typename Word<A>::type* at) {
    A x;
    for (int looks = kLooks; !read<A>(at, x) && looks > 0; --looks) __builtin_amdgcn_s_sleep(1);
    return x;
}

// A tile's run for those behind it: (m, H) side by side, one word for 32-bit states,
// and the exponent in 16 bits, none of them ever all bits.  (It is applied to a state
// and joined to nothing, and at 2^+-32000 every state is an infinity or 0.)
constexpr int kExponent = 1 << 15, kFar = 32000;
template <class A> struct Run { Gain<A> p; A h; };
__device__ __forceinline__ void publish_exponent(uint16_t* exps, int64_t at, int e) {
    const int held = e < -kFar ? -kFar : e > kFar ? kFar : e;
    __hip_atomic_store(exps + at, static_cast<uint16_t>(kExponent + held), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void publish_run(uint64_t* agg, uint16_t* exps, int64_t at, const Run<float>& r) {
    typedef Word<float> W;
    const uint32_t m = r.p.m == r.p.m ? __builtin_bit_cast(uint32_t, r.p.m) : W::kNan;
    const uint32_t h = r.h == r.h ? __builtin_bit_cast(uint32_t, r.h) : W::kNan;
    __hip_atomic_store(agg + at, static_cast<uint64_t>(h) << 32 | m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    publish_exponent(exps, at, r.p.e);
}
__device__ __forceinline__ void publish_run(uint64_t* agg, uint16_t* exps, int64_t at, const Run<double>& r) {
    publish<double>(agg + 2 * at, r.p.m);
    publish<double>(agg + 2 * at + 1, r.h);
    publish_exponent(exps, at, r.p.e);
}
__device__ __forceinline__ bool read_exponent(const uint16_t* exps, int64_t at, int& e) {
    const uint32_t w = __hip_atomic_load(exps + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    e = static_cast<int>(w) - kExponent;
    return w != 0xffffu;
}
__device__ __forceinline__ bool read_run(const uint64_t* agg, const uint16_t* exps, int64_t at, Run<float>& r) {
    const uint64_t w = __hip_atomic_load(agg + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const bool known = read_exponent(exps, at, r.p.e);
    r.p.m = __builtin_bit_cast(float, static_cast<uint32_t>(w));
    r.h = __builtin_bit_cast(float, static_cast<uint32_t>(w >> 32));
    return (w != ~uint64_t(0)) & known;
}
__device__ __forceinline__ bool read_run(const uint64_t* agg, const uint16_t* exps, int64_t at, Run<double>& r) {
    return read<double>(agg + 2 * at, r.p.m) & read<double>(agg + 2 * at + 1, r.h) & read_exponent(exps, at, r.p.e);
}
// As await; a run of which a part never shows is a NaN.
template <class A>
__device__ __forceinline__ void await_run(const uint64_t* agg, const uint16_t* exps, int64_t at, Run<A>& r) {
    bool known = false;
    for (int looks = kLooks; !known && looks > 0; --looks) {
        known = read_run(agg, exps, at, r);
        if (!known) __builtin_amdgcn_s_sleep(1);
    }
    if (!known) r.h = NAN;
}

// Aggregates read at once.  Eight hide more of a wait, but cost 32-bit planes, and
// lanes along the steps, a wave a SIMD: 1 x 65536 x 1024 bfloat16 101 us in eights,
// 102 in fours; 64 x 2^20 float steps, derivative, 375 and 368.
template <class T, int Dir> constexpr int kBatch = Dir == 0 && sizeof(T) == 2 ? 8 : 4;

// Workgroups go to the dies in turn, each with an L2 of its own.  So tiles are
// dealt out in windows in which a die takes some strips that lie beside each
// other: what two of them share of a line is fetched once (every grid's last part
// window in plain order; which die takes a tile does not matter to what it waits
// for).  One, 2, 4, 8, 16 strips, forward in us: 37 sequences, 65793 x 1001 bfloat16
// 151, 142, 138, 141, 143; 5, 30000 x 997 float 118, 111, 107, 109, 114; 64,
// 100000 x 511 125, 119, 117, 116, 116.  Streams share no line, but words that their
// tiles wait for: 1 x 65536 x 1024 103, 103, 103, 101, 102 and its derivative 164,
// 167, 165, 156, 157; 16 x 4096 x 2048 156, 155, 160, 156, 156.
constexpr unsigned kDies = 8, kBeside = 4, kBesideStream = 8;

template <class T, int V, int K, int Dir, bool Sigmoid, bool Vjp, bool Packed, bool Stream>
__global__ void __launch_bounds__((kMost<T, Dir>)) hawk_recurrence_tile(const RecArgs<T> a) {
    typedef Acc<T> A;
    __shared__ A lds_m[kMost<T, Dir> * V], lds_h[kMost<T, Dir> * V];
    __shared__ int lds_e[kMost<T, Dir> * V];
    __shared__ int lds_chunk, lds_from;
    const int tid = threadIdx.x, lane = tid & 63;
    const int ncol = Dir == 0 ? 1 << a.lcol : a.ncol, nt = a.nt;

    // A strip's chunks are taken in the order of the strip's counter: whatever a
    // tile waits for has begun before it.  (One counter for all would hand out
    // a tile in 10 ns: longer than a small tile takes.)
    constexpr unsigned beside = Stream ? kBesideStream : kBeside, window = kDies * beside;
    const unsigned into = blockIdx.x % window, base = blockIdx.x - into;
    const unsigned tile = base + window <= gridDim.x ? base + into % kDies * beside + into / kDies : blockIdx.x;
    const int strip = static_cast<int>(tile % static_cast<unsigned>(a.strips));
    int chunk = 0;
    if (a.chunks > 1) {
        if (tid == 0) lds_chunk = static_cast<int>(atomicAdd(a.counter + strip * a.counter_step, 1u));
        __syncthreads();
        chunk = __builtin_amdgcn_readfirstlane(lds_chunk);
        if (chunk >= a.chunks) return;             // only where two streams worked in one scratch
    }
    const int64_t col0 = static_cast<int64_t>(strip) * ncol;
    const int here = Dir == 0 ? tid & (ncol - 1) : tid / nt;
    const int tl = Dir == 0 ? tid >> a.lcol : tid - here * nt;
    // a column's sequence and first channel; the row's last channels are a full
    // vector that ends with them, whose first `skip` are the neighbour's
    auto place = [&](int64_t col, int64_t& s, int64_t& c, int& skip) {
        const uint32_t q = static_cast<uint32_t>(col) / static_cast<uint32_t>(a.groups);   // at most 2^31 states
        s = q;
        c = (static_cast<uint32_t>(col) - q * a.groups) * static_cast<uint32_t>(V);
        skip = 0;
        if (c + V > a.chans) {
            skip = static_cast<int>(c + V - a.chans);
            c = a.chans - V;
        }
    };
    const bool live = here < ncol && col0 + here < a.cols;
    int64_t s = 0, c0 = 0;
    int skip = 0;
    if (live) place(col0 + here, s, c0, skip);
    const int row0 = chunk * (nt * K) + tl * K;
    const int left = a.steps - row0;
    const int rows = !live || left < 0 ? 0 : left < K ? left : K;
    const int64_t first_state = s * a.chans + c0;    // dense planes: this thread's states

    const int at = row0 < a.steps ? row0 : a.steps - 1;
    Raw<T, V> gate[K], in[K], x[K], prior[K];
    tile_load<T, V, K, Dir, Stream>(a.gate, s, c0, at, a.steps, gate);
    tile_load<T, V, K, Dir, Stream>(Vjp ? a.bar_h : a.x, s, c0, at, a.steps, in);
    if constexpr (Vjp) {
        // h a step earlier in the primal's direction, a step later in the scan's
        tile_load<T, V, K, Dir, Stream>(a.h, s, c0, at + 1 < a.steps ? at + 1 : a.steps - 1, a.steps, prior);
        if constexpr (Sigmoid) tile_load<T, V, K, Dir, Stream>(a.x, s, c0, at, a.steps, x);
    }
    if (rows < K) {                       // steps that do not exist leave the state as it is
#pragma unroll
        for (int k = 0; k < K; ++k) {
            gate[k] = choose(k < rows, gate[k], splat<T, V>(static_cast<T>(Sigmoid ? INFINITY : 1.0f)));
            in[k] = choose(k < rows, in[k], splat<T, V>(static_cast<T>(0.0f)));
        }
    }

    // packed rows: which of this thread's begin a sequence in the scan's
    // direction, which end one, and the sequence the first is in.  The tile's
    // own sequences are found once; most tiles lie within one or two.
    unsigned begins = 0, ends = 0;
    int seq_at = 0, seq_low = 0, seq_high = 0;
    auto cut = [&](int q) -> int { return cut_at(a.offsets, a.offsets64, q); };
    if constexpr (Packed) {
        const int tile0 = chunk * (nt * K), tile1 = tile0 + nt * K < a.steps ? tile0 + nt * K - 1 : a.steps - 1;
        const int row_a = a.rev ? a.steps - 1 - tile1 : tile0, row_b = a.rev ? a.steps - 1 - tile0 : tile1;
        auto scalar = [&](int q) -> int { return cut_at_scalar(a.offsets, a.offsets64, q); };
        seq_low = sequence_of(scalar, 0, static_cast<int>(a.seqs) - 1, row_a);
        seq_high = seq_low;
        if (scalar(seq_low + 1) <= row_b) seq_high = sequence_of(scalar, seq_low, static_cast<int>(a.seqs) - 1, row_b);
        int low = scalar(seq_low), high = scalar(seq_low + 1);
        if (rows > 0) {
            const int row = a.rev ? a.steps - 1 - row0 : row0;
            int q = seq_low;
            if (seq_low != seq_high) {
                q = sequence_of(cut, seq_low, seq_high, row);
                low = cut(q);
                high = cut(q + 1);
            }
            seq_at = q;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (k >= rows) continue;
                const int r = a.rev ? row - k : row + k;
                while (!a.rev && r >= high && q < seq_high) {
                    ++q;
                    low = high;
                    high = cut(q + 1);
                }
                while (a.rev && r < low && q > seq_low) {
                    --q;
                    high = low;
                    low = cut(q);
                }
                begins |= static_cast<unsigned>(r == (a.rev ? high - 1 : low)) << k;
                ends |= static_cast<unsigned>(r == (a.rev ? low : high - 1)) << k;
            }
        }
    }
    // The sequence of the k-th row where it begins one.
    auto moved = [&](int k, int q) -> int {
        return k == 0 ? q : sequence_of(cut, seq_low, seq_high, a.rev ? a.steps - 1 - row0 - k : row0 + k);
    };
    auto begin = [&](int64_t q, int v) -> A { return a.init ? a.init[q * a.chans + c0 + v] : A(0); };

    // Gates and inputs cost less to convert twice than to hold twice as wide: the
    // bfloat16 forward of 8 steps keeps 64 registers of them instead of 128, and three
    // waves a SIMD win back even the sigmoid's second evaluation (16 x 4096 x 2048:
    // 178 us; 356 with both its values kept, at one wave).
    auto coefficients = [&](int k, int v, A& g, A& rest, A& b) {
        g = widen<T, V>(gate[k], v);
        if constexpr (Sigmoid) sigmoid(g, g, rest);
        b = widen<T, V>(in[k], v);
        if constexpr (!Vjp && Sigmoid) b *= rest;
    };
    // one step: the state after it, of the state before it.  (A sigmoid gate that is
    // NaN makes its step's outputs NaN by itself, so a product that takes 0 times
    // anything as 0 is enough.)
    auto through = [&](A g, A G) -> A { return Sigmoid ? cutmul(g, G) : g == A(0) ? A(0) : g * G; };
    auto step = [&](A g, A b, A h) -> A {
        if constexpr (Vjp) return through(g, b + h);
        else if constexpr (Sigmoid) return cutmul(g, h) + b;
        else return g == A(0) ? b : fused(g, h, b);
    };
    auto join = [&](const Gain<A>& p, const Gain<A>& q) -> Gain<A> { return normal(times(p, q)); };

    // fold this thread's steps from a zero state
    Gain<A> P[V];
    A H[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { P[v] = {A(1), 0}; H[v] = A(0); }
    int q = seq_at;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if constexpr (Packed) {
            if (begins >> k & 1) {
                q = moved(k, q);
#pragma unroll
                for (int v = 0; v < V; ++v) { P[v] = {A(0), 0}; H[v] = begin(q, v); }
            }
        }
        forget(gate[k]);                  // values are widened a step at a time
        forget(in[k]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            A g, rest, b;
            coefficients(k, v, g, rest, b);
            H[v] = step(g, b, H[v]);
            P[v] = times(P[v], g);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) asm volatile("" : "+v"(P[v].m), "+v"(P[v].e), "+v"(H[v]));
    }
#pragma unroll
    for (int v = 0; v < V; ++v) P[v] = normal(P[v]);

    A enter[V];
#pragma unroll
    for (int v = 0; v < V; ++v) enter[v] = !Packed && a.init && live ? a.init[first_state + v] : A(0);
    if (nt > 1 || a.chunks > 1) {
        // join the tile's threads: within a wave, then across its waves
        const int wt = Dir == 0 ? (ncol < 64 ? 64 >> a.lcol : 1) : 64;    // a wave's threads along the steps
        const int spacing = Dir == 0 ? ncol : 1;
        const int in_wave = Dir == 0 ? (ncol < 64 ? lane >> a.lcol : 0) : lane < tl ? lane : tl;
        for (int d = 1; d < wt; d <<= 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const Gain<A> p{__shfl_up(P[v].m, d * spacing), __shfl_up(P[v].e, d * spacing)};
                const A h = __shfl_up(H[v], d * spacing);
                const A joined_h = passed(P[v], h, H[v]);
                const Gain<A> joined_p = join(P[v], p);
                H[v] = in_wave >= d ? joined_h : H[v];
                P[v].m = in_wave >= d ? joined_p.m : P[v].m;
                P[v].e = in_wave >= d ? joined_p.e : P[v].e;
            }
        }
        // Runs of a wave, in order: Dir 0, run r of a column is its threads r wt
        // to r wt + wt - 1; otherwise a column's run in a wave ends with the
        // wave or with the column.
        const int run = Dir == 0 ? tl / wt : tid >> 6;
        const int first_run = Dir == 0 ? 0 : (tid - tl) >> 6;
        auto slot = [&](int r, int column, int v) -> int {
            return Dir == 0 ? (r * V + v) * ncol + column : r;
        };
        if (Dir == 0 ? tl % wt == wt - 1 || tl == nt - 1 : lane == 63) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                lds_m[slot(run, here, v)] = P[v].m;
                lds_e[slot(run, here, v)] = P[v].e;
                lds_h[slot(run, here, v)] = H[v];
            }
        }
        __syncthreads();
        Gain<A> earlier_p[V];
        A earlier_h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { earlier_p[v] = {A(1), 0}; earlier_h[v] = A(0); }
        for (int r = first_run; r < run; ++r) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int at = slot(r, here, v);
                const Gain<A> p{lds_m[at], lds_e[at]};
                earlier_h[v] = passed(p, earlier_h[v], lds_h[at]);
                earlier_p[v] = times(p, earlier_p[v]);        // at most eight runs
            }
        }
        if (a.chunks > 1) {
            // the tile's own (P, H): its last time lanes hold them
            __syncthreads();
            if (tl == nt - 1 && here < ncol) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const Gain<A> p = join(P[v], earlier_p[v]);
                    lds_h[here * V + v] = passed(P[v], earlier_h[v], H[v]);
                    lds_m[here * V + v] = p.m;
                    lds_e[here * V + v] = p.e;
                }
            }
        }
        // what lies between the tile's first step and this thread's: the runs before
        // its own, then the threads of its own
        auto before = [&] {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (wt > 1) {
                    const Gain<A> p{__shfl_up(P[v].m, spacing), __shfl_up(P[v].e, spacing)};
                    const A joined_h = passed(p, earlier_h[v], __shfl_up(H[v], spacing));
                    const Gain<A> joined_p = times(p, earlier_p[v]);
                    earlier_h[v] = in_wave > 0 ? joined_h : earlier_h[v];
                    earlier_p[v].m = in_wave > 0 ? joined_p.m : earlier_p[v].m;
                    earlier_p[v].e = in_wave > 0 ? joined_p.e : earlier_p[v].e;
                }
                earlier_p[v] = normal(earlier_p[v]);
            }
        };
        if (a.chunks <= 1) before();
        if (a.chunks > 1) {
            __syncthreads();
            typedef typename Word<A>::type W;
            const bool more = chunk + 1 < a.chunks;
            uint32_t* flags = a.flag + static_cast<int64_t>(strip) * a.chunks;
            auto raise = [&] { __hip_atomic_store(flags + chunk, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
            bool cut_all = true;
            if (more) {
                for (int i = tid; i < ncol * V; i += blockDim.x) {
                    const int64_t col = col0 + i / V;
                    int64_t cs, cc;
                    int cskip;
                    if (col >= a.cols) break;
                    place(col, cs, cc, cskip);
                    if (i % V < cskip) continue;
                    const int64_t state = chunk * a.states + cs * a.chans + cc + i % V;
                    publish_run(a.agg, a.agg_exp, state, Run<A>{{lds_m[i], lds_e[i]}, lds_h[i]});
                    // a cut in the tile: nothing before it matters to what leaves it
                    if (lds_m[i] == A(0)) publish<A>(a.state + state, lds_h[i]);
                    else cut_all = false;
                }
            }
            before();                         // while the words are on their way
            // a packed sequence that begins in the tile cuts every channel, so the
            // tiles after it wait for nothing before it
            if constexpr (Packed) {
                if (more && __syncthreads_and(cut_all) && tid == 0) raise();
            }
            // How far back a state is known.  One wave looks at the strip's flags of
            // the 64 chunks before this one: two lines a look, since every waiting
            // tile looks again and again (at the states' own words, 64 lines a look,
            // they took a third of the card's bandwidth).  A flag only says where to
            // look; the words it is about are awaited for themselves.
            if (chunk > 0 && tid < 64) {
                const int look = chunk - 1 - lane;
                uint64_t known = 0;
                for (int looks = kLooks; looks > 0; --looks) {
                    known = __ballot(look < 0 || __hip_atomic_load(flags + look, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 1u);
                    if (known) break;
                    __builtin_amdgcn_s_sleep(4);
                }
                // -1: the state before the first chunk
                if (lane == 0) lds_from = chunk - 1 - (known ? __builtin_ctzll(known) : 0);
            }
            __syncthreads();
            // The state that enters: the known one, then the chunks since in
            // order, so the bits do not depend on how far back that was.
            const int from = chunk > 0 ? lds_from : -1;
            for (int i = tid; i < ncol * V; i += blockDim.x) {
                const int64_t col = col0 + i / V;
                int64_t cs, cc;
                int cskip;
                if (col >= a.cols) break;
                place(col, cs, cc, cskip);
                if (i % V < cskip) continue;
                const int64_t state = cs * a.chans + cc + i % V;
                A carry;
                const W* known = a.state + (from < 0 ? 0 : from) * a.states + state;
                bool here_yet = true;             // asked for with the first aggregates, not before them
                if (from >= 0) here_yet = read<A>(known, carry);
                else carry = !Packed && a.init ? a.init[state] : A(0);
                for (int k = from + 1; k < chunk; k += kBatch<T, Dir>) {
                    Run<A> run_of[kBatch<T, Dir>];
                    bool ok[kBatch<T, Dir>];
#pragma unroll
                    for (int b = 0; b < kBatch<T, Dir>; ++b)
                        ok[b] = read_run(a.agg, a.agg_exp, (k + b < chunk ? k + b : k) * a.states + state, run_of[b]);
                    if (!here_yet) {
                        carry = await<A>(known);
                        here_yet = true;
                    }
#pragma unroll
                    for (int b = 0; b < kBatch<T, Dir>; ++b) {
                        if (k + b >= chunk) continue;
                        if (!ok[b]) await_run<A>(a.agg, a.agg_exp, (k + b) * a.states + state, run_of[b]);
                        carry = passed(run_of[b].p, carry, run_of[b].h);
                    }
                }
                if (!here_yet) carry = await<A>(known);
                if (more) {
                    if (lds_m[i] != A(0))
                        publish<A>(a.state + chunk * a.states + state, passed({lds_m[i], lds_e[i]}, carry, lds_h[i]));
                    if (i == V - 1) raise();      // the first column's last channel, which every strip has
                }
                lds_h[i] = carry;                 // this thread's alone until the barrier
            }
            __syncthreads();
#pragma unroll
            for (int v = 0; v < V; ++v) enter[v] = lds_h[(here < ncol ? here : 0) * V + v];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) enter[v] = passed(earlier_p[v], enter[v], earlier_h[v]);
    }

    // the steps again, from the state that enters them
    if (rows > 0) {
        const Plane<T>& to = Vjp ? a.bar_x : a.h;
        T* out = to.data + s * to.seq + c0 * to.chan + row0 * to.step;
        T* out_gate = Vjp ? a.bar_gate.data + s * a.bar_gate.seq + c0 * a.bar_gate.chan + row0 * a.bar_gate.step : nullptr;
        const bool has_end = Packed ? ends != 0 : row0 + rows == a.steps;
        q = seq_at;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if constexpr (Packed) {
                if (begins >> k & 1) {
                    q = moved(k, q);
#pragma unroll
                    for (int v = 0; v < V; ++v) enter[v] = begin(q, v);
                }
            }
            const bool last = (Packed || Vjp) && has_end && k < rows && (Packed ? (ends >> k & 1) : k == rows - 1);
            const int64_t state = Packed ? q * a.chans + c0 : first_state;
            forget(gate[k]);
            forget(in[k]);
            if constexpr (Vjp) {
                forget(prior[k]);
                if constexpr (Sigmoid) forget(x[k]);
                A h[V];
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = widen<T, V>(prior[k], v);
                if (last) {
#pragma unroll
                    for (int v = 0; v < V; ++v) h[v] = a.h0 ? a.h0[state + v] : A(0);
                }
                Raw<T, V> to_gate, to_x;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    A g, rest, b;
                    coefficients(k, v, g, rest, b);
                    const A G = b + enter[v];
                    A bar_gate = G * h[v], bar_x = G;
                    if constexpr (Sigmoid) {
                        bar_x = rest * G;
                        bar_gate = bar_x * ((h[v] - widen<T, V>(x[k], v)) * g);
                    }
                    put<T, V>(to_gate, v, static_cast<T>(bar_gate));
                    put<T, V>(to_x, v, static_cast<T>(bar_x));
                    enter[v] = through(g, G);
                }
                if constexpr (Dir == 0) {
                    if (a.bar_gate.data) row_store<T, V, Stream>(out_gate, a.bar_gate.step, k, rows, skip, to_gate);
                    if (a.bar_x.data) row_store<T, V, Stream>(out, a.bar_x.step, k, rows, skip, to_x);
                } else {
                    gate[k] = to_gate;
                    in[k] = to_x;
                }
            } else {
                Raw<T, V> h;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    A g, rest, b;
                    coefficients(k, v, g, rest, b);
                    enter[v] = step(g, b, enter[v]);
                    put<T, V>(h, v, static_cast<T>(enter[v]));
                }
                if constexpr (Dir == 0) row_store<T, V, Stream>(out, a.h.step, k, rows, skip, h);
                else in[k] = h;
            }
            if (Packed && last && a.fin) {
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (v >= skip) a.fin[state + v] = enter[v];
            }
        }
        if (!Packed && has_end && a.fin) {     // the steps past the end left the state as it was
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v >= skip) a.fin[first_state + v] = enter[v];
        }
        if constexpr (Dir != 0) {
            if (Vjp && a.bar_gate.data) run_store<T, K, Dir>(out_gate, rows, gate);
            if (!Vjp || a.bar_x.data) run_store<T, K, Dir>(out, rows, in);
        }
    }
    if constexpr (Packed) {               // a sequence without rows: its state passes through
        if (chunk == 0 && a.fin && live) {
            for (int e = tl; e < a.seqs; e += nt) {
                if (cut(e) < cut(e + 1)) continue;
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (v >= skip) a.fin[e * a.chans + c0 + v] = begin(e, v);
            }
        }
    }
}

// Before tiles that tell each other states: the counters at 0, no word written.
__global__ void __launch_bounds__(256) hawk_recurrence_clear(uint32_t* at, int64_t counters, int64_t count) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += 256LL * gridDim.x) {
        const uint32_t w = i < counters ? 0u : ~0u;
        store_raw<uint32_t, 4, true>(at + 4 * i, Raw<uint32_t, 4>{w, w, w, w});
    }
}

// A few steps (a token at a time, or some): one thread takes V channels of a
// sequence from step to step, with nothing to join.  Bounded by a launch and one
// round trip to memory.  bfloat16, us a call, against a tile: 64 x 1 x 2048 4.7 and
// 8.4, 512 x 4 x 8192 15.7 and 21.5, 512 x 8 x 2048 8.7 and 9.7; the other way from
// 8 steps of 512 x 8192 on (39 and 35; 16 steps 80 and 68).
constexpr int kShort = 8, kShortThreads = 64;
template <class T, int V, bool Sigmoid>
__global__ void __launch_bounds__(kShortThreads) hawk_recurrence_short(const RecArgs<T> a) {
    typedef Acc<T> A;
    const uint32_t col = blockIdx.x * kShortThreads + threadIdx.x;
    if (col >= a.cols) return;
    const uint32_t s = col / static_cast<uint32_t>(a.groups);
    int64_t c = (col - s * a.groups) * static_cast<uint32_t>(V);
    int skip = 0;
    if (c + V > a.chans) {
        skip = static_cast<int>(c + V - a.chans);
        c = a.chans - V;
    }
    const T *gate = a.gate.data + s * a.gate.seq + c * a.gate.chan, *x = a.x.data + s * a.x.seq + c * a.x.chan;
    T* out = a.h.data + s * a.h.seq + c * a.h.chan;
    const int64_t state = s * a.chans + c;
    Raw<T, V> g = load_raw<T, V>(gate), in = load_raw<T, V>(x);
    A h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = a.init ? a.init[state + v] : A(0);
    for (int t = 0; t < a.steps; ++t) {
        const Raw<T, V> g_now = g, in_now = in;
        if (t + 1 < a.steps) {
            g = load_raw<T, V>(gate + (t + 1) * a.gate.step);
            in = load_raw<T, V>(x + (t + 1) * a.x.step);
        }
        Raw<T, V> h_now;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            A ga = widen<T, V>(g_now, v), b = widen<T, V>(in_now, v), rest;
            if constexpr (Sigmoid) {
                sigmoid(ga, ga, rest);
                b *= rest;
            }
            h[v] = Sigmoid ? cutmul(ga, h[v]) + b : ga == A(0) ? b : fused(ga, h[v], b);
            put<T, V>(h_now, v, static_cast<T>(h[v]));
        }
        row_store<T, V, false>(out, a.h.step, t, a.steps, skip, h_now);
    }
    if (a.fin) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v >= skip) a.fin[state + v] = h[v];
    }
}

// States as they are: of no steps at all, or aside before they are written over.
template <class A>
__global__ void __launch_bounds__(256) hawk_recurrence_pass(const A* init, A* fin, int64_t states) {
    const int64_t j = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (j < states) fin[j] = init ? init[j] : A(0);
}

int log2_up(int64_t n) {
    int l = 0;
    while ((int64_t(1) << l) < n) ++l;
    return l;
}

// How a call is cut.  Dir 0: a wave's lanes lie along the channels first, so
// its loads are runs of a row; what is left of the workgroup lies along the
// steps, and across sequences where the steps are few.  Otherwise lanes lie
// along the steps, as many as a sequence needs, and what is left takes further
// sequences.
struct Shape {
    int v, k, dir;
    int lcol, ncol, nt, chunks, threads;
    int groups;
    int64_t cols, strips, states;
    bool stream;
};

template <class T, bool Vjp> struct Tile {
    static constexpr int kVec = 16 / static_cast<int>(sizeof(T));
    // steps a thread: the derivative holds twice the forward's registers
    static constexpr int kSteps = Vjp ? 4 : 8;
    static constexpr int kAlong = 8;              // steps a thread where they are contiguous
};

// Log2 of the lanes across a long row.  32 lanes of 16 bytes (512-byte runs) pass
// the planes of 16 x 4096 x 2048 bfloat16 elements at 6.07 TB/s, 16 lanes at
// 4.84, 64 at 5.88 (a copy of the pattern), but give half the steps a tile, and
// where few strips fill the card a tile waits for a state many tiles back:
// forward of 1 x 65536 x 1024 152 us in 4 strips of 32 lanes, 111 in 8 of 16, 101
// in 16 of 8; 8 x 2048 x 1536 44 us in 48 of 32, 42 in 96 of 16 and in 192 of 8;
// 16 x 4096 x 2048 157 us in 128 of 32, 168 in 256 of 16.
constexpr int kAcross = 5, kAcrossFew = 4, kAcrossLeast = 3;
constexpr int64_t kManyStrips = 64, kFewStrips = 16;

template <class T, bool Vjp>
Shape shape_of(const hk_recurrence_job& j) {
    Shape s{};
    const hk_plane* planes[6] = {&j.gate, &j.h, &j.x, &j.bar_h, &j.bar_gate, &j.bar_x};
    bool chan = true, along = !j.offsets;
    for (const hk_plane* p : planes) {
        if (!p->data) continue;
        chan &= p->chan == 1;
        along &= p->step == 1;
    }
    const int64_t seqs = j.offsets ? 1 : j.seqs;
    if (along && j.steps > 1 && (j.chans == 1 || !chan)) {
        s.dir = (j.reverse != 0) != Vjp ? -1 : 1;
        s.v = 1;
        s.k = Tile<T, Vjp>::kAlong;
        s.groups = static_cast<int>(j.chans);
        s.cols = seqs * s.groups;
        const int64_t need = (j.steps + s.k - 1) / s.k;
        constexpr int most = kMost<T, 1>;
        s.chunks = static_cast<int>((need + most - 1) / most);
        s.nt = static_cast<int>((need + s.chunks - 1) / s.chunks);
        s.ncol = s.nt < kThreads ? kThreads / s.nt : 1;
        if (s.ncol > s.cols) s.ncol = static_cast<int>(s.cols);
    } else {
        s.dir = 0;
        s.v = chan && j.chans >= Tile<T, Vjp>::kVec ? Tile<T, Vjp>::kVec : 1;
        s.k = Tile<T, Vjp>::kSteps;
        s.groups = static_cast<int>((j.chans + s.v - 1) / s.v);
        s.cols = seqs * s.groups;
        const int across = (s.cols >> kAcross) >= kManyStrips ? kAcross : (s.cols >> kAcrossFew) >= kFewStrips ? kAcrossFew : kAcrossLeast;
        s.lcol = log2_up(s.groups);
        if (s.lcol > across) s.lcol = across;
        const int64_t need = (j.steps + s.k - 1) / s.k;
        int most = kThreads >> s.lcol;
        // few steps: the lanes they leave take more columns
        while (need <= most / 2 && (int64_t(1) << s.lcol) < s.cols && s.lcol < 8) {
            ++s.lcol;
            most /= 2;
        }
        const int wt = s.lcol < 6 ? 64 >> s.lcol : 1;
        s.chunks = static_cast<int>((need + most - 1) / most);
        s.nt = static_cast<int>((need + s.chunks - 1) / s.chunks);
        s.nt = (s.nt + wt - 1) / wt * wt;          // whole waves
        s.chunks = static_cast<int>((need + s.nt - 1) / s.nt);
        s.ncol = 1 << s.lcol;
    }
    // Whole lines: a strip's part of a row begins and ends with a 128-byte line in
    // every plane, so nothing is read twice and it need not stay in the caches
    // (16 x 4096 x 2048 forward 157 us as a stream, 170 cached).  Otherwise the
    // neighbouring strip finds its share of a line there (65793 packed rows of
    // 1001 bfloat16 channels: 138 us cached, 168 as a stream).
    s.stream = s.dir == 0 && s.v > 1;
    for (const hk_plane* p : planes) {
        if (!p->data) continue;
        s.stream &= (p->seq * static_cast<int64_t>(sizeof(T))) % 128 == 0 && (p->step * static_cast<int64_t>(sizeof(T))) % 128 == 0 &&
                    reinterpret_cast<uintptr_t>(p->data) % 128 == 0;
    }
    s.threads = (s.nt * s.ncol + 63) / 64 * 64;
    s.strips = (s.cols + s.ncol - 1) / s.ncol;
    s.states = seqs * j.chans;
    return s;
}

int check_job(const hk_recurrence_job* j, bool vjp, const std::string& who) {
    using hawk_internal::set_error;
    if (!j) return set_error(HK_EVALUE, who + ": a job is required");
    if (j->seqs < 0 || j->steps < 0 || j->chans < 0) return set_error(HK_EVALUE, who + ": sizes must be >= 0");
    if (j->dtype < HK_F32 || j->dtype > HK_F16) return set_error(HK_EVALUE, who + ": unknown element type");
    if (j->seqs > INT32_MAX / 2 || j->steps > INT32_MAX / 2 || j->chans > INT32_MAX / 2 ||
        (j->chans > 0 && j->seqs > INT32_MAX / j->chans))
        return set_error(HK_EVALUE, who + ": more than 2^30 steps, or 2^31 states");
    const bool any = j->seqs > 0 && j->steps > 0 && j->chans > 0;
    if (any && (!j->gate.data || !j->h.data || (!vjp && !j->x.data) || (vjp && !j->bar_h.data)))
        return set_error(HK_EVALUE, who + ": a plane is missing");
    if (any && vjp && j->sigmoid && !j->x.data)
        return set_error(HK_EVALUE, who + ": the sigmoid form's gradient reads x");
    if (j->offsets && j->seqs == 0 && j->steps > 0)
        return set_error(HK_EVALUE, who + ": rows without a sequence");
    return HK_OK;
}

template <class T>
Plane<T> plane_of(const hk_plane& p, int64_t steps, bool flip) {
    Plane<T> q{static_cast<T*>(p.data), p.seq, p.step, p.chan};
    if (flip && q.data) {                 // scan step 0 is the last row
        q.data += (steps - 1) * q.step;
        q.step = -q.step;
    }
    return q;
}

// A strip's counter lies on a line of its own unless there are many.
int counter_step(const Shape& s) { return s.strips > 1024 ? 1 : 32; }
size_t counter_bytes(const Shape& s) { return (4 * static_cast<size_t>(s.strips) * counter_step(s) + 255) / 256 * 256; }
// The mantissa of P and H and the state of every (chunk, state), the flags, then P's
// exponents, in whole 16-byte words
size_t word_bytes(const Shape& s, size_t word) {
    return ((3 * word + 2) * static_cast<size_t>(s.states) * s.chunks + 4 * static_cast<size_t>(s.strips) * s.chunks + 15) / 16 * 16;
}

size_t tile_bytes(const Shape& s, size_t word) { return s.chunks > 1 ? counter_bytes(s) + word_bytes(s, word) : 0; }

// States that leave may be written over those that enter.  One tile a sequence
// has read these before a barrier; but a tile may still be to read them when the
// last one, which took what lies between from the tiles' (P, H), has finished, and
// packed rows read a sequence's state twice.  Such calls read a copy, which costs a
// launch and only they pay.
template <bool Vjp>
bool may_copy(const hk_recurrence_job& j, const Shape& s) {
    return (Vjp ? j.bar_last && j.bar_h0 : j.h0 && j.last) && (s.chunks > 1 || j.offsets);
}

template <class T, bool Vjp>
size_t scratch_of(const hk_recurrence_job& j) {
    if (j.seqs <= 0 || j.steps <= 0 || j.chans <= 0) return 0;
    const Shape s = shape_of<T, Vjp>(j);
    return tile_bytes(s, sizeof(Acc<T>)) + (may_copy<Vjp>(j, s) ? sizeof(Acc<T>) * static_cast<size_t>(j.seqs * j.chans) : 0);
}

int launched(const char* what) {
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? HK_OK : hawk_internal::set_hip_error(what, err);
}

template <class T, int V, int K, int Dir, bool Vjp, bool Stream>
void launch_tile(const hk_recurrence_job& j, const RecArgs<T>& a, const Shape& s, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(s.strips * s.chunks)), block(s.threads);
    auto go = [&](auto sigmoid, auto packed) {
        hipLaunchKernelGGL((hawk_recurrence_tile<T, V, K, Dir, sigmoid.value, Vjp, packed.value, Stream>), grid, block, 0,
                           stream, a);
    };
    typedef std::true_type Yes;
    typedef std::false_type No;
    if constexpr (Dir == 0) {
        if (j.offsets) return j.sigmoid ? go(Yes{}, Yes{}) : go(No{}, Yes{});
    }
    j.sigmoid ? go(Yes{}, No{}) : go(No{}, No{});
}

template <class T, bool Vjp>
int recurrence(const hk_recurrence_job& j, void* scratch, hipStream_t stream, const std::string& who) {
    typedef Acc<T> A;
    const A* init = static_cast<const A*>(Vjp ? j.bar_last : j.h0);
    A* fin = static_cast<A*>(Vjp ? j.bar_h0 : j.last);
    if (j.seqs == 0 || j.chans == 0) return HK_OK;
    if (j.steps == 0) {
        if (!fin) return HK_OK;
        const int64_t states = j.seqs * j.chans;
        hipLaunchKernelGGL(hawk_recurrence_pass<A>, dim3(static_cast<unsigned>((states + 255) / 256)), dim3(256), 0,
                           stream, init, fin, states);
        return launched("hawk_recurrence_pass launch");
    }
    const Shape s = shape_of<T, Vjp>(j);
    if (s.strips * s.chunks > UINT32_MAX / s.threads) return hawk_internal::set_error(HK_EVALUE, who + ": the planes exceed the grid limit");
    const int64_t entering = j.seqs * j.chans;
    const bool copy = may_copy<Vjp>(j, s) && init < fin + entering && fin < init + entering;
    if ((s.chunks > 1 || copy) && !scratch) return hawk_internal::set_error(HK_EVALUE, who + ": scratch is required");
    if (copy) {
        A* held = reinterpret_cast<A*>(static_cast<unsigned char*>(scratch) + tile_bytes(s, sizeof(A)));
        hipLaunchKernelGGL(hawk_recurrence_pass<A>, dim3(static_cast<unsigned>((entering + 255) / 256)), dim3(256), 0,
                           stream, init, held, entering);
        const int rc = launched("hawk_recurrence_pass launch");
        if (rc != HK_OK) return rc;
        init = held;
    }
    const bool flip = (j.reverse != 0) != Vjp;
    RecArgs<T> a{};
    a.gate = plane_of<T>(j.gate, j.steps, flip);
    a.x = plane_of<T>(j.x, j.steps, flip);
    a.h = plane_of<T>(j.h, j.steps, flip);
    a.bar_h = plane_of<T>(j.bar_h, j.steps, flip);
    a.bar_gate = plane_of<T>(j.bar_gate, j.steps, flip);
    a.bar_x = plane_of<T>(j.bar_x, j.steps, flip);
    a.init = init;
    a.h0 = static_cast<const A*>(j.h0);
    a.fin = fin;
    a.offsets = j.offsets;
    a.offsets64 = j.offsets64;
    a.seqs = j.seqs;
    a.chans = j.chans;
    a.cols = s.cols;
    a.steps = static_cast<int>(j.steps);
    a.groups = s.groups;
    a.lcol = s.lcol;
    a.ncol = s.ncol;
    a.nt = s.nt;
    a.strips = static_cast<int>(s.strips);
    a.chunks = s.chunks;
    a.states = s.states;
    a.rev = flip;
    if (s.chunks > 1) {
        typedef typename Word<A>::type W;
        a.counter = static_cast<uint32_t*>(scratch);
        a.counter_step = counter_step(s);
        const int64_t words_each = s.states * s.chunks;
        a.agg = reinterpret_cast<uint64_t*>(static_cast<unsigned char*>(scratch) + counter_bytes(s));
        a.state = reinterpret_cast<W*>(a.agg) + 2 * words_each;
        a.flag = reinterpret_cast<uint32_t*>(a.state + words_each);
        a.agg_exp = reinterpret_cast<uint16_t*>(a.flag + s.strips * s.chunks);
        const int64_t counters = static_cast<int64_t>(counter_bytes(s) / 16);
        const int64_t words = counters + static_cast<int64_t>(word_bytes(s, sizeof(A)) / 16);
        const int64_t blocks = (words + 1023) / 1024;
        hipLaunchKernelGGL(hawk_recurrence_clear, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), dim3(256),
                           0, stream, static_cast<uint32_t*>(scratch), counters, words);
        const int rc = launched("hawk_recurrence_clear launch");
        if (rc != HK_OK) return rc;
    }
    constexpr int VV = Tile<T, Vjp>::kVec, KC = Tile<T, Vjp>::kSteps, KT = Tile<T, Vjp>::kAlong;
    if constexpr (!Vjp) {
        if (!j.offsets && j.steps <= kShort && s.dir == 0) {
            const dim3 grid(static_cast<unsigned>((s.cols + kShortThreads - 1) / kShortThreads)), block(kShortThreads);
            auto go = [&](auto v) {
                if (j.sigmoid) hipLaunchKernelGGL((hawk_recurrence_short<T, decltype(v)::value, true>), grid, block, 0, stream, a);
                else hipLaunchKernelGGL((hawk_recurrence_short<T, decltype(v)::value, false>), grid, block, 0, stream, a);
            };
            if (s.v > 1) go(std::integral_constant<int, VV>{});
            else go(std::integral_constant<int, 1>{});
            return launched("hawk_recurrence_short launch");
        }
    }
    if (s.dir > 0) launch_tile<T, 1, KT, 1, Vjp, false>(j, a, s, stream);
    else if (s.dir < 0) launch_tile<T, 1, KT, -1, Vjp, false>(j, a, s, stream);
    else if (s.stream) launch_tile<T, VV, KC, 0, Vjp, true>(j, a, s, stream);
    else if (s.v > 1) launch_tile<T, VV, KC, 0, Vjp, false>(j, a, s, stream);
    else launch_tile<T, 1, KC, 0, Vjp, false>(j, a, s, stream);
    return launched("hawk_recurrence_tile launch");
}

}  // namespace

extern "C" {

size_t hk_recurrence_scratch_bytes(const hk_recurrence_job* job, int32_t vjp) {
    if (!job) return 0;
    switch (job->dtype) {
        case HK_F32: return vjp ? scratch_of<float, true>(*job) : scratch_of<float, false>(*job);
        case HK_F64: return vjp ? scratch_of<double, true>(*job) : scratch_of<double, false>(*job);
        case HK_BF16: return vjp ? scratch_of<bf16, true>(*job) : scratch_of<bf16, false>(*job);
        case HK_F16: return vjp ? scratch_of<f16, true>(*job) : scratch_of<f16, false>(*job);
    }
    return 0;
}

int hk_recurrence(const hk_recurrence_job* job, void* scratch, void* stream) {
    const int rc = check_job(job, false, "hk_recurrence");
    if (rc != HK_OK) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (job->dtype) {
        case HK_F32: return recurrence<float, false>(*job, scratch, s, "hk_recurrence");
        case HK_F64: return recurrence<double, false>(*job, scratch, s, "hk_recurrence");
        case HK_BF16: return recurrence<bf16, false>(*job, scratch, s, "hk_recurrence");
        default: return recurrence<f16, false>(*job, scratch, s, "hk_recurrence");
    }
}

int hk_recurrence_vjp(const hk_recurrence_job* job, void* scratch, void* stream) {
    const int rc = check_job(job, true, "hk_recurrence_vjp");
    if (rc != HK_OK) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (job->dtype) {
        case HK_F32: return recurrence<float, true>(*job, scratch, s, "hk_recurrence_vjp");
        case HK_F64: return recurrence<double, true>(*job, scratch, s, "hk_recurrence_vjp");
        case HK_BF16: return recurrence<bf16, true>(*job, scratch, s, "hk_recurrence_vjp");
        default: return recurrence<f16, true>(*job, scratch, s, "hk_recurrence_vjp");
    }
}

}  // extern "C"
