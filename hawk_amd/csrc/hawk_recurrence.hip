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
// A gate of 0 cuts, and so does the first row of a packed sequence: products
// and their use take 0 times anything as 0 (cutmul), so neither an infinity
// nor a NaN passes a cut; a product of gates is 0 only where one is (chain).  States and products are held in 32 bits (64 for
// double planes).

#include "hawk_core.h"
#include "hawk_internal.h"
#include "hawk_vec.h"

#include <hip/hip_runtime.h>
#include <cstdint>
#include <string>

namespace {

using namespace hawk_vec;

constexpr int kThreads = 256;

template <class T>
struct Plane {
    T* data;
    int64_t seq, step, chan;
};

template <class T>
struct RecArgs {
    Plane<T> gate, x, h, bar_h, bar_gate, bar_x;
    const Acc<T>* init;       // the state that enters the scan: h0, or bar_last
    const Acc<T>* h0;         // the derivative's h_(-1)
    Acc<T>* fin;              // the state that leaves it: last, or bar_h0
    const void* offsets;
    Acc<T>*agg_p, *agg_h;     // [chunk][seqs * chans]: each tile's (P, H)
    Acc<T>* carry;            // [chunk][seqs * chans]: the state that enters each tile
    int64_t seqs, chans, cols, states;   // states: those of one tile row, seqs * chans (packed: chans)
    int steps, groups;        // groups: threads across a row's channels
    int lcol, lt, chunks;     // log2 of a tile's columns and of its time lanes
    int rev, offsets64;       // rev: scan step i is row steps - 1 - i (packed planes)
};

enum Phase { kSingle, kAggregate, kApply };

__device__ __forceinline__ int64_t cut_at(const void* offsets, int wide, int64_t s) {
    return wide ? static_cast<const int64_t*>(offsets)[s] : static_cast<const int32_t*>(offsets)[s];
}

// The sequence whose rows hold `row`: the last one that starts at or before it.
__device__ __forceinline__ int64_t sequence_of(const void* offsets, int wide, int64_t seqs, int64_t row) {
    int64_t low = 0, high = seqs - 1;
    while (low < high) {
        const int64_t mid = (low + high + 1) >> 1;
        if (cut_at(offsets, wide, mid) <= row) low = mid;
        else high = mid - 1;
    }
    return low;
}

// One thread's K steps of V channels.  Chan: V consecutive channels a step,
// each step a load of its own; otherwise one channel, K steps in one load where
// the steps are contiguous (Dir 1, or -1 where the scan runs down the axis).
// A step past the end repeats the last one's address, so every load is issued
// without a branch; its value is replaced afterwards.
template <class T, int V, int K, int Dir>
__device__ __forceinline__ void tile_load(const Plane<T>& p, const T* base, int row0, int steps, Acc<T> (&out)[K][V]) {
    if constexpr (Dir == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int row = row0 + k < steps ? row0 + k : steps - 1;
            load<T, V>(base + row * p.step, out[k]);
        }
    } else {
        if (row0 + K <= steps) {
            Acc<T> flat[K];
            load<T, K>(Dir > 0 ? base + row0 : base - (row0 + K - 1), flat);
#pragma unroll
            for (int k = 0; k < K; ++k) out[k][0] = flat[Dir > 0 ? k : K - 1 - k];
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int row = row0 + k < steps ? row0 + k : steps - 1;
                load<T, 1>(Dir > 0 ? base + row : base - row, out[k]);
            }
        }
    }
}

// Stores the tile's steps that exist; `skip` leading channels belong to the
// neighbouring thread.
template <class T, int V, int K, int Dir>
__device__ __forceinline__ void tile_store(const Plane<T>& p, T* base, int row0, int rows, int skip,
                                           const Acc<T> (&x)[K][V]) {
    if constexpr (Dir == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            T* to = base + (row0 + k) * p.step;
            if (k >= rows) continue;
            if (skip == 0) {
                store<T, V>(to, x[k]);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (v >= skip) to[v] = static_cast<T>(x[k][v]);
            }
        }
    } else {
        if (rows == K) {
            Acc<T> flat[K];
#pragma unroll
            for (int k = 0; k < K; ++k) flat[Dir > 0 ? k : K - 1 - k] = x[k][0];
            store<T, K>(Dir > 0 ? base + row0 : base - (row0 + K - 1), flat);
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (k < rows) *(Dir > 0 ? base + row0 + k : base - row0 - k) = static_cast<T>(x[k][0]);
        }
    }
}

template <class T, int V, int K, int Dir, bool Sigmoid, bool Vjp, bool Packed>
__global__ void __launch_bounds__(kThreads) hawk_recurrence_tile(const RecArgs<T> a, const int phase) {
    typedef Acc<T> A;
    __shared__ A lds_p[kThreads * V], lds_h[kThreads * V];
    const int tid = threadIdx.x, lane = tid & 63;
    const int ncol = 1 << a.lcol, nt = 1 << a.lt;
    const int chunk = blockIdx.x % a.chunks;
    const int here = Dir == 0 ? tid & (ncol - 1) : tid >> a.lt;
    const int tl = Dir == 0 ? tid >> a.lcol : tid & (nt - 1);
    const int64_t col = static_cast<int64_t>(blockIdx.x / a.chunks) * ncol + here;
    const bool live = col < a.cols;
    const int64_t s = live ? col / a.groups : 0;
    int64_t c0 = live ? (col % a.groups) * V : 0;
    int skip = 0;
    if (c0 + V > a.chans) {              // the row's last channels: a full vector that ends with them
        skip = static_cast<int>(c0 + V - a.chans);
        c0 = a.chans - V;
    }
    const int row0 = chunk * (nt * K) + tl * K;
    const int left = a.steps - row0;
    const int rows = !live || left < 0 ? 0 : left < K ? left : K;
    const int64_t first_state = s * a.chans + c0;    // dense planes: this thread's states

    // load everything the tile needs
    const int at = row0 < a.steps ? row0 : a.steps - 1;
    A gate[K][V], in[K][V], x[K][V], prior[K][V];
    tile_load<T, V, K, Dir>(a.gate, a.gate.data + s * a.gate.seq + c0 * a.gate.chan, at, a.steps, gate);
    if constexpr (Vjp) {
        tile_load<T, V, K, Dir>(a.bar_h, a.bar_h.data + s * a.bar_h.seq + c0 * a.bar_h.chan, at, a.steps, in);
        if (phase != kAggregate) {
            if constexpr (Sigmoid)
                tile_load<T, V, K, Dir>(a.x, a.x.data + s * a.x.seq + c0 * a.x.chan, at, a.steps, x);
            // h a step earlier in the primal's direction, a step later in the scan's
            tile_load<T, V, K, Dir>(a.h, a.h.data + s * a.h.seq + c0 * a.h.chan,
                                    at + 1 < a.steps ? at + 1 : a.steps - 1, a.steps, prior);
        }
    } else {
        tile_load<T, V, K, Dir>(a.x, a.x.data + s * a.x.seq + c0 * a.x.chan, at, a.steps, in);
    }

    // packed rows: which of this thread's begin a sequence in the scan's
    // direction, which end one, and the sequence each is in
    unsigned begins = 0, ends = 0;
    int64_t seq_at = 0;
    if constexpr (Packed) {
        if (rows > 0) {
            const int64_t row = a.rev ? a.steps - 1 - row0 : row0;
            seq_at = sequence_of(a.offsets, a.offsets64, a.seqs, row);
            int64_t q = seq_at, low = cut_at(a.offsets, a.offsets64, q), high = cut_at(a.offsets, a.offsets64, q + 1);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (k >= rows) break;
                const int64_t r = a.rev ? row - k : row + k;
                while (!a.rev && r >= high && q + 1 < a.seqs) {
                    ++q;
                    low = high;
                    high = cut_at(a.offsets, a.offsets64, q + 1);
                }
                while (a.rev && r < low && q > 0) {
                    --q;
                    high = low;
                    low = cut_at(a.offsets, a.offsets64, q);
                }
                begins |= static_cast<unsigned>(r == (a.rev ? high - 1 : low)) << k;
                ends |= static_cast<unsigned>(r == (a.rev ? low : high - 1)) << k;
            }
        }
    }
    // The sequence of the k-th row, walking on from the k-1st's: begins bit k
    // moves to the next sequence that is not empty.
    auto moved = [&](int k, int64_t q) -> int64_t {
        if (k == 0) return q;
        const int64_t r = a.rev ? a.steps - 1 - row0 - k : row0 + k;
        return sequence_of(a.offsets, a.offsets64, a.seqs, r);
    };

    // fold this thread's steps from a zero state
    A local[K][V], product[K][V], P[V], H[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { P[v] = A(1); H[v] = A(0); }
    int64_t q = seq_at;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if constexpr (Packed) {
            if (begins >> k & 1) {
                q = moved(k, q);
#pragma unroll
                for (int v = 0; v < V; ++v) { P[v] = A(0); H[v] = a.init ? a.init[q * a.chans + c0 + v] : A(0); }
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            A g = gate[k][v], rest = A(0), b;
            if constexpr (Sigmoid) sigmoid(gate[k][v], g, rest);
            if constexpr (Vjp) b = g == A(0) ? A(0) : g * in[k][v];
            else b = Sigmoid ? rest * in[k][v] : in[k][v];
            if (k >= rows) { g = A(1); b = A(0); }
            if constexpr (Vjp) {           // what the gradient needs: the state before the step
                local[k][v] = H[v];
                product[k][v] = P[v];
            }
            H[v] = g == A(0) ? b : fused(g, H[v], b);
            P[v] = chain(P[v], g);
            if constexpr (!Vjp) {
                local[k][v] = H[v];
                product[k][v] = P[v];
            }
        }
    }

    // join the tile's threads: within a wave, then across its waves
    const int wt = Dir == 0 ? (ncol < 64 ? 64 >> a.lcol : 1) : (nt < 64 ? nt : 64);
    const int spacing = Dir == 0 ? ncol : 1;
    const int in_wave = Dir == 0 ? (ncol < 64 ? lane >> a.lcol : 0) : tl & (wt - 1);
    const int wave_group = tl / wt, wave_groups = nt / wt > 0 ? nt / wt : 1;
    for (int d = 1; d < wt; d <<= 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const A p = __shfl_up(P[v], d * spacing), h = __shfl_up(H[v], d * spacing);
            if (in_wave >= d) {
                H[v] = H[v] + cutmul(P[v], h);
                P[v] = chain(P[v], p);
            }
        }
    }
    A before_p[V], before_h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        before_p[v] = A(1);
        before_h[v] = A(0);
        if (wt > 1) {
            const A p = __shfl_up(P[v], spacing), h = __shfl_up(H[v], spacing);
            if (in_wave > 0) { before_p[v] = p; before_h[v] = h; }
        }
    }
    if (wave_groups > 1) {
        if (in_wave == wt - 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                lds_p[(wave_group * V + v) * ncol + here] = P[v];
                lds_h[(wave_group * V + v) * ncol + here] = H[v];
            }
        }
        __syncthreads();
        A p[V], h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { p[v] = A(1); h[v] = A(0); }
        for (int w = 0; w < wave_group; ++w) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const A wp = lds_p[(w * V + v) * ncol + here], wh = lds_h[(w * V + v) * ncol + here];
                h[v] = wh + cutmul(wp, h[v]);
                p[v] = chain(wp, p[v]);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            H[v] = H[v] + cutmul(P[v], h[v]);
            P[v] = chain(P[v], p[v]);
            before_h[v] = before_h[v] + cutmul(before_p[v], h[v]);
            before_p[v] = chain(before_p[v], p[v]);
        }
    }

    const int64_t states = a.states;
    if (phase == kAggregate) {
        if (tl == nt - 1 && live) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (v < skip) continue;
                a.agg_p[chunk * states + first_state + v] = P[v];
                a.agg_h[chunk * states + first_state + v] = H[v];
            }
        }
        return;
    }

    // the state that enters this thread's steps
    A enter[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        A c = A(0);
        if (phase == kApply) c = a.carry[chunk * states + first_state + v];
        else if (!Packed && a.init) c = a.init[first_state + v];
        enter[v] = before_h[v] + cutmul(before_p[v], c);
    }
    if (rows > 0) {
        if constexpr (Vjp) {
            A bar_gate[K][V], bar_x[K][V];
            q = seq_at;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if constexpr (Packed) {
                    if (begins >> k & 1) q = moved(k, q);
                }
                const bool last = k < rows && (Packed ? (ends >> k & 1) : row0 + k == a.steps - 1);
                const int64_t state = Packed ? q * a.chans + c0 : first_state;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    A g = gate[k][v], rest = A(0);
                    if constexpr (Sigmoid) sigmoid(gate[k][v], g, rest);
                    const A G = in[k][v] + (local[k][v] + cutmul(product[k][v], enter[v]));
                    const A h = last ? (a.h0 ? a.h0[state + v] : A(0)) : prior[k][v];
                    if constexpr (Sigmoid) {
                        bar_gate[k][v] = G * (h - x[k][v]) * g * rest;
                        bar_x[k][v] = rest * G;
                    } else {
                        bar_gate[k][v] = G * h;
                        bar_x[k][v] = G;
                    }
                    if (last && a.fin && v >= skip) a.fin[state + v] = g == A(0) ? A(0) : g * G;
                }
            }
            if (a.bar_gate.data)
                tile_store<T, V, K, Dir>(a.bar_gate, a.bar_gate.data + s * a.bar_gate.seq + c0 * a.bar_gate.chan, row0,
                                         rows, skip, bar_gate);
            if (a.bar_x.data)
                tile_store<T, V, K, Dir>(a.bar_x, a.bar_x.data + s * a.bar_x.seq + c0 * a.bar_x.chan, row0, rows, skip,
                                         bar_x);
        } else {
            q = seq_at;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if constexpr (Packed) {
                    if (begins >> k & 1) q = moved(k, q);
                }
                const bool last = k < rows && (Packed ? (ends >> k & 1) : row0 + k == a.steps - 1);
                const int64_t state = Packed ? q * a.chans + c0 : first_state;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    local[k][v] = local[k][v] + cutmul(product[k][v], enter[v]);
                    if (last && a.fin && v >= skip) a.fin[state + v] = local[k][v];
                }
            }
            tile_store<T, V, K, Dir>(a.h, a.h.data + s * a.h.seq + c0 * a.h.chan, row0, rows, skip, local);
        }
    }
    if constexpr (Packed) {               // a sequence without rows: its state passes through
        if (chunk == 0 && a.fin && live) {
            for (int64_t e = tl; e < a.seqs; e += nt) {
                if (cut_at(a.offsets, a.offsets64, e) < cut_at(a.offsets, a.offsets64, e + 1)) continue;
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (v >= skip) a.fin[e * a.chans + c0 + v] = a.init ? a.init[e * a.chans + c0 + v] : A(0);
            }
        }
    }
}

// The state that enters each tile: one thread a (sequence, channel) folds the
// tiles' (P, H) in order.
template <class A>
__global__ void __launch_bounds__(256) hawk_recurrence_carry(const A* agg_p, const A* agg_h, A* carry, const A* init,
                                                             int64_t states, int chunks) {
    const int64_t j = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (j >= states) return;
    A state = init ? init[j] : A(0);
    for (int c = 0; c < chunks; ++c) {
        carry[c * states + j] = state;
        state = agg_h[c * states + j] + cutmul(agg_p[c * states + j], state);
    }
}

// No steps at all: every state passes through.
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
// along the steps.
struct Shape {
    int v, k, dir;
    int lcol, lt, chunks, threads;
    int groups;
    int64_t cols, blocks, states;
};

template <class T, bool Vjp> struct Tile {
    static constexpr int kVec = 16 / static_cast<int>(sizeof(T));
    // steps a thread: the derivative holds twice the forward's registers
    static constexpr int kSteps = Vjp ? 4 : 8;
    static constexpr int kAlong = Vjp ? 4 : (kVec > 4 ? kVec : 4);   // steps a thread where they are contiguous
};

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
    const int64_t packed_seqs = j.offsets ? 1 : j.seqs;
    if (along && (j.chans == 1 || !chan)) {
        s.dir = (j.reverse != 0) != Vjp ? -1 : 1;
        s.v = 1;
        s.k = Tile<T, Vjp>::kAlong;
        s.groups = static_cast<int>(j.chans);
        s.cols = packed_seqs * s.groups;
        s.lt = log2_up((j.steps + s.k - 1) / s.k);
        if ((1 << s.lt) > kThreads) s.lt = log2_up(kThreads);
        s.lcol = log2_up(kThreads) - s.lt;
    } else {
        s.dir = 0;
        s.v = chan && j.chans >= Tile<T, Vjp>::kVec ? Tile<T, Vjp>::kVec : 1;
        s.k = Tile<T, Vjp>::kSteps;
        s.groups = static_cast<int>((j.chans + s.v - 1) / s.v);
        s.cols = packed_seqs * s.groups;
        int across = log2_up(s.groups);
        if (across > 6) across = 6;
        s.lt = log2_up((j.steps + s.k - 1) / s.k);
        if (s.lt + across > log2_up(kThreads)) s.lt = log2_up(kThreads) - across;
        s.lcol = log2_up(kThreads) - s.lt;
    }
    if (s.lcol > log2_up(s.cols)) s.lcol = log2_up(s.cols);
    s.threads = 1 << (s.lcol + s.lt);
    if (s.threads < 64) {
        s.lcol = 6 - s.lt;
        s.threads = 64;
    }
    const int64_t rows = int64_t(s.k) << s.lt;
    s.chunks = static_cast<int>((j.steps + rows - 1) / rows);
    s.blocks = ((s.cols + (int64_t(1) << s.lcol) - 1) >> s.lcol) * s.chunks;
    s.states = packed_seqs * j.chans;
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

template <class T, bool Vjp>
size_t scratch_of(const hk_recurrence_job& j) {
    if (j.seqs <= 0 || j.steps <= 0 || j.chans <= 0) return 0;
    const Shape s = shape_of<T, Vjp>(j);
    return s.chunks > 1 ? 3 * sizeof(Acc<T>) * static_cast<size_t>(s.states) * s.chunks : 0;
}

int launched(const char* what) {
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? HK_OK : hawk_internal::set_hip_error(what, err);
}

template <class T, int V, int K, int Dir, bool Vjp>
void launch_tile(const hk_recurrence_job& j, const RecArgs<T>& a, const Shape& s, int phase, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(s.blocks)), block(s.threads);
    if constexpr (Dir == 0) {
        if (j.offsets) {
            if (j.sigmoid) hipLaunchKernelGGL((hawk_recurrence_tile<T, V, K, Dir, true, Vjp, true>), grid, block, 0, stream, a, phase);
            else hipLaunchKernelGGL((hawk_recurrence_tile<T, V, K, Dir, false, Vjp, true>), grid, block, 0, stream, a, phase);
            return;
        }
    }
    if (j.sigmoid) hipLaunchKernelGGL((hawk_recurrence_tile<T, V, K, Dir, true, Vjp, false>), grid, block, 0, stream, a, phase);
    else hipLaunchKernelGGL((hawk_recurrence_tile<T, V, K, Dir, false, Vjp, false>), grid, block, 0, stream, a, phase);
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
    if (s.blocks > INT32_MAX) return hawk_internal::set_error(HK_EVALUE, who + ": the planes exceed the grid limit");
    if (s.chunks > 1 && !scratch) return hawk_internal::set_error(HK_EVALUE, who + ": scratch is required");
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
    a.lt = s.lt;
    a.chunks = s.chunks;
    a.states = s.states;
    a.rev = flip;
    a.agg_p = static_cast<A*>(scratch);
    a.agg_h = a.agg_p + s.states * s.chunks;
    a.carry = a.agg_h + s.states * s.chunks;
    constexpr int VV = Tile<T, Vjp>::kVec, KC = Tile<T, Vjp>::kSteps, KT = Tile<T, Vjp>::kAlong;
    auto tiles = [&](int phase) {
        if (s.dir > 0) launch_tile<T, 1, KT, 1, Vjp>(j, a, s, phase, stream);
        else if (s.dir < 0) launch_tile<T, 1, KT, -1, Vjp>(j, a, s, phase, stream);
        else if (s.v > 1) launch_tile<T, VV, KC, 0, Vjp>(j, a, s, phase, stream);
        else launch_tile<T, 1, KC, 0, Vjp>(j, a, s, phase, stream);
        return launched("hawk_recurrence_tile launch");
    };
    if (s.chunks == 1) return tiles(kSingle);
    int rc = tiles(kAggregate);
    if (rc != HK_OK) return rc;
    hipLaunchKernelGGL(hawk_recurrence_carry<A>, dim3(static_cast<unsigned>((s.states + 255) / 256)), dim3(256), 0,
                       stream, a.agg_p, a.agg_h, a.carry, j.offsets ? nullptr : init, s.states, s.chunks);
    rc = launched("hawk_recurrence_carry launch");
    return rc != HK_OK ? rc : tiles(kApply);
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
