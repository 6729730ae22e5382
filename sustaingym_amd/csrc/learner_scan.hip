// learner_scan.hip — gfx950 kernels of lrn_scan / lrn_scan_backward / lrn_advantages (include/learner_ops.h).
//
// All three are h_u = a_u h_{u-1} + x_u along an order u of the steps; what differs is what x, a and the outputs are:
//   scan       u runs with the sequence, x and a are read
//   backward   u runs against it: x_u = g_h, a_u = the gate of the step before in this order (1 in front of the first, so
//              that g_final enters as the state), and beside h = grad_x comes grad_gate = h * (the state before the step)
//   advantages u runs against time: x_u = d_t, a_u = gamma lam (1 - end_t), and beside h comes h + V_t
//
// The state before a step is h itself for float32 and float64.  For 16-bit sequences h is rounded, and a gate's gradient made of it
// is off by half a step more than its own rounding; so the forward pass keeps every eighth state as it is (float32, half a byte an
// element), at the places where the backward pass' runs end, and the backward pass walks the seven in between again from x and the
// gates: the traffic of reading h.
//
// A run of steps acts on the state in front of it as h -> A h + H, and two runs in a row as (A2 A1, A2 H1 + H2).  So the steps
// are dealt out in runs of L to lanes that hold them in registers: each computes its (A, H) from a state of 0, the states in
// front of the runs come from the pairs of the runs before, and each lane walks its run again with the right state and writes.
// Every element is read once.  Where there are too few columns to fill the GPU, the sequence is also cut into parts: a first
// launch writes the parts' pairs to the workspace, a second one starts each part from the pairs before it (x and a are then
// read twice, the second time mostly from the last-level cache).
//
// Three layouts.  COLUMNS: lanes lie along adjacent channels (or sequences, where time is the slow index), wavefronts of a
// workgroup along time; pairs go through LDS.  RUNS: time is the fast index, so lanes lie along time, pairs go through a
// wavefront scan.  TILES: as COLUMNS, with 16 bytes to a lane's load.  State, pairs and products are float32 (float64 for
// float64 sequences) whatever the elements' type.
//
// Bound by memory where there are columns for everybody (averages over three sets of inputs in turn, which no cache holds):
// advantages of 288 x 65 536 move 397 MB in 85 us (4.7 TB/s of a large copy's 5.1), returns of 288 x 16 384 float64 81 MB in 18;
// a memory of 16 x 2048 x 1024 bfloat16 218 MB in 50 forward and 352 MB in 75 backward.  131 073 x 72 float32, in 256 parts:
// 19 + 30 us for 113 MB, 75 of them twice.  A thread to a column, as it was first, took 173, 153, 2075, 2648 and 44 000 us.
//
// A coefficient of exactly 0 cuts: nothing of the state in front enters, whatever it holds.  For float32 that is the
// multiplication in which 0 times anything is 0, one instruction instead of a comparison and a selection behind an fma.  That
// would also hide a gate that is not finite from a state of 0, so such a gate makes its own step's x NaN (`seen`).
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "lrn_common.h"

namespace lrn {
namespace {

struct View {
    const void* p;
    int64_t st, sb, sc;
};

// Order u: 0 .. steps-1.  The views' time strides and bases already point that way.
struct Seq {
    int64_t steps, cols;        // cols = batch * channels, column q = (q / channels, q % channels)
    int64_t channels;
    View x, gate, resets, before, h, second;
    double gate_const, scale;   // advantages: gamma lam, gamma
    View keep;                  // 16-bit SCAN with a gradient to come, its BACKWARD: every L-th state, [runs of BACKWARD][cols]
    const void* initial;
    const void* edge;           // backward: the initial state; advantages: V behind the last step (float32)
    void* final;
    int64_t part;               // steps of a part
    int64_t group;              // RUNS: lanes of a column, where a wavefront has all its steps
    int64_t tight, width;       // COLUMNS: tiles of a sequence where a tile may not reach over two (else 0), and their channels
    void* pairs;                // [parts][2][cols]
    bool sums;                  // BACKWARD of 16-bit sequences: the gate's gradient in float32
};

enum Kind { SCAN, BACKWARD, ADVANTAGES };
enum Phase { WHOLE, PAIRS, APPLY };

template <class T> struct State { using type = float; };
template <> struct State<double> { using type = double; };

extern "C" __device__ float product_with_zero(float, float) __asm("llvm.amdgcn.fmul.legacy");
__device__ __forceinline__ float times(float a, float b) { return product_with_zero(a, b); }
__device__ __forceinline__ double times(double a, double b) { return a == 0.0 ? 0.0 : a * b; }
// x, or NaN beside a coefficient that is not finite
__device__ __forceinline__ float seen(float a, float x) { return __builtin_fmaf(a, 0.0f, x); }
__device__ __forceinline__ double seen(double a, double x) { return __builtin_fma(a, 0.0, x); }
__device__ __forceinline__ float step(float a, float h, float x) { return times(a, h) + x; }
__device__ __forceinline__ double step(double a, double h, double x) { return a == 0.0 ? x : __builtin_fma(a, h, x); }

// (A, H) of a run
template <class W> struct Pair {
    W a, h;
    __device__ __forceinline__ void then(W a2, W x) { h = step(a2, h, x); a = times(a2, a); }
    // what came before it
    __device__ __forceinline__ void after(const Pair& first) { h = step(a, first.h, h); a = times(a, first.a); }
};

constexpr int L = LRN_KEEP;      // steps of a lane's run: 8

// One of the three, for one type of elements: whether there is a gate tensor (else a constant), whether there are resets, and
// whether the second output (SCAN: the kept states) is wanted.  Compiled in: a condition between loads keeps them from being in flight together.
template <Kind K_, class T_, bool GATE_, bool RESETS_, bool SECOND_, class P_ = T_>
struct Op {
    static constexpr Kind K = K_;
    static constexpr bool GATE = GATE_, RESETS = RESETS_, SECOND = SECOND_ && K_ != SCAN;
    static constexpr bool KEEP = SECOND_ && K_ == SCAN, AGAIN = SECOND_ && K_ == BACKWARD && sizeof(T_) == 2;    // writes S.keep; walks from it
    using T = T_;
    using W = typename State<T_>::type;
    using Out = std::conditional_t<K_ == ADVANTAGES, float, T_>;
    using Second = std::conditional_t<K_ == ADVANTAGES, float, P_>;     // (P_: the gate's gradient, float32 where it is going to be summed)
};

// One lane's run, L steps of V adjacent columns: as it comes from memory ...
template <class O, int V>
struct Raw {
    using T = typename O::T;
    using W = typename O::W;
    static constexpr int N = L * V;
    T x[N];
    T g[O::GATE ? N + (O::AGAIN ? V : 0) : 1];             // SCAN: gate of the step; BACKWARD: of the step before in this order
    T before[O::K == BACKWARD && O::SECOND ? N : 1];       // the state before the step; AGAIN: the x that came with it
    W kept[O::AGAIN ? V : 1];                              // the state before the run's last step, the first of the forward walk
    float v[O::K == ADVANTAGES ? N + V : 1];               // values of the steps u0 - 1 .. u0 + L - 1
    uint8_t r[O::RESETS ? N + V : 1];                      // flags of the steps u0 .., BACKWARD: u0 - 1 ..
};
// ... and as it acts
template <class O, int V>
struct Run {
    using W = typename O::W;
    W a[L * V], x[L * V];
    std::conditional_t<O::K == ADVANTAGES, float, W> extra[O::SECOND ? L * V : 1];    // BACKWARD: the state before; ADVANTAGES: V
    uint32_t anew = 0;                                     // BACKWARD: bits of the steps that have a reset
};

// A lane's V columns in every view: the part of the address that is the same for the wavefront, and the lane's own.
struct Place {
    const char *x, *gate, *before, *resets;
    char *h, *second, *keep;
    uint32_t ox, og, ob, orr, oh, oo, ok;      // bytes
    uint32_t next_flags;                       // from the first column's flags to the second's
};

// ---- COLUMNS: loads and stores ------------------------------------------------------------------------------------------

typedef const char __attribute__((address_space(1)))* Global;
template <class E, int V> struct Vec { typedef E type __attribute__((ext_vector_type(V), aligned(sizeof(E)))); };

template <class E, int V> __device__ __forceinline__ void get(Global base, uint32_t lane, E* to) {
    if constexpr (V == 1) to[0] = *(const E __attribute__((address_space(1)))*)(base + lane);
    else {
        typedef typename Vec<E, V>::type vec;
        const vec w = *(const vec __attribute__((address_space(1)))*)(base + lane);
#pragma unroll
        for (int k = 0; k < V; k++) to[k] = w[k];
    }
}
template <class E, int V> __device__ __forceinline__ void put(Global base, uint32_t lane, const E* from) {
    if constexpr (V == 1) *(E __attribute__((address_space(1)))*)(base + lane) = from[0];
    else {
        typedef typename Vec<E, V>::type vec;
        vec w;
#pragma unroll
        for (int k = 0; k < V; k++) w[k] = from[k];
        *(vec __attribute__((address_space(1)))*)(base + lane) = w;
    }
}

// One step further, by a scalar addition at its place: eight multiples of every stride kept ready would not fit the scalar
// registers, and come back from vector lanes at two instructions a piece.  (Behind the asm only the type says what memory it is.)
__device__ __forceinline__ void advance(Global& p, int64_t bytes) {
    p += bytes;
    asm("" : "+s"(p));
}

// How many of `count` steps from `from` lie in front of `to`, and in it.
__device__ __forceinline__ int in_front(int64_t from, int64_t to, int count) { return to <= from ? 0 : to - from < count ? (int)(to - from) : count; }

// The lane's part of an address, as the 32-bit half of a load that has its other half in scalar registers: known to be
// invariant it would be added to the base ahead of the loop, and every load would add 64 bits in vector registers.
__device__ __forceinline__ uint32_t kept_apart(uint32_t lane) {
    asm volatile("" : "+v"(lane));
    return lane;
}

// COUNT steps from `from`.  FULL: all of them are there, but with BEFORE the first may lie in front of step 0 and with BEHIND the
// last at `hi`: its neighbour is read in its place, and whoever uses it knows.  Not FULL: what lies outside [0, hi) is 0.
template <class E, int V, int COUNT, bool FULL, bool BEFORE = false, bool BEHIND = false>
__device__ __forceinline__ void get_steps(const char* base, int64_t st, uint32_t lane, int64_t from, int64_t hi, E* to) {
    const int64_t stride = st * (int64_t)sizeof(E);
    const bool short_front = FULL && BEFORE && from < 0, short_back = FULL && BEHIND && from + COUNT > hi;
    Global p = (Global)(base + (short_front ? 0 : from * stride));
    lane = kept_apart(lane);
    const int first = FULL ? 0 : in_front(from, 0, COUNT), last = FULL ? COUNT : in_front(from, hi, COUNT);
#pragma unroll
    for (int i = 0; i < COUNT; i++) {
        if constexpr (!FULL) {
#pragma unroll
            for (int k = 0; k < V; k++) to[i * V + k] = E(0);
        }
        if (FULL || (i >= first && i < last)) get<E, V>(p, lane, to + i * V);
        if (i + 1 < COUNT) advance(p, (i == 0 && short_front) || (i == COUNT - 2 && short_back) ? 0 : stride);
    }
}

// Steps u0 .. u0 + L - 1 as they are in memory.
template <class O, int V, bool FULL, bool APPLYING>
__device__ __forceinline__ void load(const Seq& S, const Place& P, int64_t u0, int64_t end, Raw<O, V>& d) {
    using T = typename O::T;
    constexpr int shift = O::K == BACKWARD ? 1 : 0;
    constexpr bool back = O::K == BACKWARD;
    get_steps<T, V, L, FULL>(P.x, S.x.st, P.ox, u0, end, d.x);
    if constexpr (O::GATE) get_steps<T, V, L + (O::AGAIN && APPLYING ? 1 : 0), FULL, back>(P.gate, S.gate.st, P.og, u0 - shift, end, d.g);
    if constexpr (O::RESETS) {
        constexpr int COUNT = L + (O::K == BACKWARD && O::SECOND ? 1 : 0);
        if constexpr (V == 1) get_steps<uint8_t, 1, COUNT, FULL, back>(P.resets, S.resets.st, P.orr, u0 - shift, end, d.r);
        else {
            // (two sequences' flags are adjacent or the same)
            uint8_t one[V][COUNT];
#pragma unroll
            for (int k = 0; k < V; k++) get_steps<uint8_t, 1, COUNT, FULL, back>(P.resets, S.resets.st, P.orr + k * P.next_flags, u0 - shift, end, one[k]);
#pragma unroll
            for (int i = 0; i < COUNT * V; i++) d.r[i] = one[i % V][i / V];
        }
    }
    if constexpr (O::K == ADVANTAGES) get_steps<float, V, L + 1, FULL, true>(P.before, S.before.st, P.ob, u0 - 1, end, d.v);
    if constexpr (O::AGAIN && APPLYING) {
        using W = typename O::W;
        get_steps<T, V, L, FULL>(P.before, S.before.st, P.ob, u0, end, d.before);
        if (u0 + L < S.steps) get<W, V>((Global)(P.keep + u0 / L * S.keep.st * (int64_t)sizeof(W)), kept_apart(P.ok), d.kept);
    } else if constexpr (O::K == BACKWARD && O::SECOND && APPLYING) get_steps<T, V, L, FULL, false, true>(P.before, S.before.st, P.ob, u0 + 1, S.steps, d.before);
}

// What the steps do.  Behind the end: a = 1, x = 0, so that a run that is cut short has the pair of what it holds.
template <class O, int V, bool FULL>
__device__ __forceinline__ void fold(const Seq& S, const Raw<O, V>& d, const typename O::W (&edge)[V], int64_t u0, int64_t end, Run<O, V>& f) {
    using W = typename O::W;
    const int count = FULL ? L : in_front(u0, end, L), final_step = in_front(u0 + 1, S.steps, L);
#pragma unroll
    for (int i = 0; i < L; i++) {
        const bool in = FULL || i < count;
#pragma unroll
        for (int k = 0; k < V; k++) {
            const int n = i * V + k;
            W x = (W)d.x[n], a = (W)S.gate_const;
            bool cut = false;
            if constexpr (O::RESETS) cut = d.r[n] != 0;
            if constexpr (O::GATE) a = (W)d.g[n];
            if constexpr (O::K == ADVANTAGES) {
                const W now = (W)d.v[n + V], next = i == 0 && u0 == 0 ? edge[k] : (W)d.v[n];
                x = cut ? x - now : x + (W)S.scale * next - now;
                f.extra[n] = d.v[n + V];
            }
            if (cut) a = W(0);
            if constexpr (O::K == BACKWARD) {
                if (i == 0 && u0 == 0) a = W(1);                        // g_final enters as it is
                if constexpr (O::SECOND && O::RESETS) f.anew |= (d.r[n + V] != 0 ? 1u : 0u) << n;
                if constexpr (O::SECOND && !O::AGAIN) {
                    W prev = (W)d.before[n];
                    if (FULL ? i == L - 1 && final_step < L : i == final_step) prev = edge[k];
                    f.extra[n] = prev;
                }
            }
            f.a[n] = in ? a : W(1);
            f.x[n] = in ? seen(a, x) : W(0);
        }
    }
    if constexpr (O::AGAIN) {
        // the forward walk's steps, from the state in front of them (a run that is cut short has the sequence's first steps)
#pragma unroll
        for (int k = 0; k < V; k++) {
            W h = u0 + L < S.steps ? d.kept[k] : edge[k];
#pragma unroll
            for (int i = L - 1; i >= 0; i--) {
                const int n = i * V + k;
                f.extra[n] = h;
                const W a = O::RESETS && (f.anew >> n & 1) ? W(0) : (W)d.g[n + V], next = step(a, h, seen(a, (W)d.before[n]));
                h = FULL || i < count ? next : h;
            }
        }
    }
}

template <class O, int V, bool FULL, bool APPLYING>
__device__ __forceinline__ void take(const Seq& S, const Place& P, const typename O::W (&edge)[V], int64_t u0, int64_t end, Run<O, V>& f) {
    Raw<O, V> raw;
    load<O, V, FULL, APPLYING>(S, P, u0, end, raw);
    fold<O, V, FULL>(S, raw, edge, u0, end, f);
}

template <class O, int V> __device__ __forceinline__ Pair<typename O::W> pair_of(const Run<O, V>& f, int k) {
    Pair<typename O::W> p{f.a[k], f.x[k]};
#pragma unroll
    for (int i = 1; i < L; i++) p.then(f.a[i * V + k], f.x[i * V + k]);
    return p;
}

// The second output of a step from the state behind it.
template <class O, int V> __device__ __forceinline__ typename O::Second second_of(const Run<O, V>& f, int n, typename O::W h) {
    using W = typename O::W;
    if constexpr (O::K == BACKWARD) return (typename O::Second)(O::RESETS && (f.anew >> n & 1) ? W(0) : h * f.extra[n]);
    else return (typename O::Second)(h + (W)f.extra[n]);
}

// Where the state before step `at` of SCAN is kept: BACKWARD's runs are counted from the last step.
template <class O> __device__ __forceinline__ int64_t keep_offset(const Seq& S, int64_t at) { return ((S.steps - at) / L - 1) * S.keep.st * (int64_t)sizeof(typename O::W); }

// Walks the run from the state in front of it and writes.
template <class O, int V, bool FULL>
__device__ __forceinline__ void walk(const Seq& S, const Place& P, const Run<O, V>& f, int64_t u0, int64_t end, typename O::W (&h)[V]) {
    using E = typename O::Out;
    using D = typename O::Second;
    Global ph = (Global)(P.h + u0 * S.h.st * (int64_t)sizeof(E)), po = (Global)(P.second + u0 * S.second.st * (int64_t)sizeof(D));
    const int last = FULL ? L : in_front(u0, end, L);
    const uint32_t oh = kept_apart(P.oh), oo = O::SECOND ? kept_apart(P.oo) : 0;
    const int keep = (int)(S.steps % L);                   // of every run, the step that begins one of BACKWARD's
    typename O::W kept[V];
#pragma unroll
    for (int i = 0; i < L; i++) {
        E out[V];
        D second[V];
#pragma unroll
        for (int k = 0; k < V; k++) {
            if (O::KEEP && i == keep) kept[k] = h[k];
            h[k] = step(f.a[i * V + k], h[k], f.x[i * V + k]);
            out[k] = (E)h[k];
            if constexpr (O::SECOND) second[k] = second_of<O, V>(f, i * V + k, h[k]);
        }
        if (FULL || i < last) {
            put<E, V>(ph, oh, out);
            if constexpr (O::SECOND) put<D, V>(po, oo, second);
        }
        advance(ph, S.h.st * (int64_t)sizeof(E));
        if constexpr (O::SECOND) advance(po, S.second.st * (int64_t)sizeof(D));
    }
    if constexpr (O::KEEP) {
        if (u0 < end && u0 + keep < S.steps) put<typename O::W, V>((Global)(P.keep + keep_offset<O>(S, u0 + keep)), kept_apart(P.ok), kept);
    }
}

template <class E> __device__ __forceinline__ const char* uniform_part(const View& v, int64_t b, int64_t c) { return v.p ? (const char*)v.p + (b * v.sb + c * v.sc) * (int64_t)sizeof(E) : nullptr; }
template <class E> __device__ __forceinline__ uint32_t lane_part(const View& v, int64_t b, int64_t c) { return (uint32_t)((b * v.sb + c * v.sc) * (int64_t)sizeof(E)); }

// Column q = (b, c) seen from the tile's first, (b0, c0).
template <class O> __device__ __forceinline__ Place place_of(const Seq& S, int64_t b0, int64_t c0, int64_t b, int64_t c) {
    using T = typename O::T;
    using E = typename O::Out;
    Place P;
    P.x = uniform_part<T>(S.x, b0, c0); P.ox = lane_part<T>(S.x, b - b0, c - c0);
    P.gate = uniform_part<T>(S.gate, b0, c0); P.og = lane_part<T>(S.gate, b - b0, c - c0);
    P.before = uniform_part<E>(S.before, b0, c0); P.ob = lane_part<E>(S.before, b - b0, c - c0);
    P.resets = uniform_part<uint8_t>(S.resets, b0, 0); P.orr = lane_part<uint8_t>(S.resets, b - b0, 0);
    P.h = (char*)uniform_part<E>(S.h, b0, c0); P.oh = lane_part<E>(S.h, b - b0, c - c0);
    P.second = (char*)uniform_part<typename O::Second>(S.second, b0, c0); P.oo = lane_part<typename O::Second>(S.second, b - b0, c - c0);
    P.keep = (char*)uniform_part<typename O::W>(S.keep, b0, c0); P.ok = lane_part<typename O::W>(S.keep, b - b0, c - c0);
    P.next_flags = S.channels == 1 ? (uint32_t)S.resets.sb : 0;
    return P;
}

// The pair of parts [from, to) of column q.
template <class W> __device__ __forceinline__ Pair<W> joined_parts(const Seq& S, int64_t from, int64_t to, int64_t q) {
    const W* pairs = (const W*)S.pairs + q;
    Pair<W> all{W(1), W(0)};
    for (int64_t i = from; i < to; i += 4) {
        Pair<W> p[4];
#pragma unroll
        for (int k = 0; k < 4; k++) p[k] = i + k < to ? Pair<W>{pairs[2 * (i + k) * S.cols], pairs[(2 * (i + k) + 1) * S.cols]} : Pair<W>{W(1), W(0)};
#pragma unroll
        for (int k = 0; k < 4; k++) all.then(p[k].a, p[k].h);
    }
    return all;
}

template <Kind K, class W> __device__ __forceinline__ W first_state(const Seq& S, int64_t q) {
    return K == ADVANTAGES || !S.initial ? W(0) : ((const W*)S.initial)[q];
}
template <Kind K, class W> __device__ __forceinline__ W edge_of(const Seq& S, int64_t q) {
    if constexpr (K == BACKWARD) return S.edge ? ((const W*)S.edge)[q] : W(0);
    else if constexpr (K == ADVANTAGES) return (W)((const float*)S.edge)[q];
    else return W(0);
}
// The state behind the last step to `final`; the backward pass goes through the last step's own coefficient.
template <Kind K, class T, class W> __device__ __forceinline__ void put_final(const Seq& S, int64_t b, int64_t c, int64_t q, W h) {
    if (!S.final) return;
    if (K == BACKWARD && S.steps > 0) {
        const bool cut = S.resets.p && ((const uint8_t*)S.resets.p)[(S.steps - 1) * S.resets.st + b * S.resets.sb];
        W own = (W)S.gate_const;
        if (S.gate.p) own = (W)((const T*)S.gate.p)[(S.steps - 1) * S.gate.st + b * S.gate.sb + c * S.gate.sc];
        if (cut) own = W(0);
        h = step(own, h, seen(own, W(0)));
    }
    ((W*)S.final)[q] = h;
}

// ---- COLUMNS: 64 V columns to a wavefront, WT wavefronts of a workgroup one behind the other in time -----------------------

template <class O, int V, int WT, Phase PH>
__global__ __launch_bounds__(WT == 1 ? 256 : 64 * WT) void columns_kernel(Seq S) {
    constexpr Kind K = O::K;
    using T = typename O::T;
    using W = typename O::W;
    constexpr int WC = WT == 1 ? 4 : 1;               // tiles of columns to a workgroup
    constexpr int64_t TURN = WT * L;
    __shared__ Pair<W> pairs_of[2][WT > 1 ? WT : 1][WT > 1 ? 64 * V : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wt = WT > 1 ? wave : 0;
    const int64_t tile = (int64_t)blockIdx.x * WC + (WT > 1 ? 0 : wave);
    int64_t b0, c0 = 0, b, c, q;
    bool there;
    if (V == 1 && S.tight) {                          // a tile has columns of one sequence
        b0 = b = tile / S.tight;
        c0 = (tile - b * S.tight) * S.width;
        c = c0 + lane;
        there = lane < S.width && c < S.channels && b < S.cols / S.channels;
        q = b * S.channels + c;
    } else {
        q = tile * 64 * V + lane * V;
        there = q < S.cols;
        b0 = tile * 64 * V / S.channels;
        b = q / S.channels;
        c = q - b * S.channels;
    }
    // (a lane without a column goes along to the barriers, reads the tile's first column and writes nothing)
    if (!there) { b = b0; c = V == 1 && S.tight ? c0 : tile * 64 * V - b0 * S.channels; q = b * S.channels + c; }
    if (q >= S.cols) return;                          // WT = 1: a whole wavefront behind the last tile
    const int64_t part = PH == WHOLE ? 0 : blockIdx.y;
    const int64_t begin = part * S.part, end = PH == WHOLE ? S.steps : min(begin + S.part, S.steps);
    const Place P = place_of<O>(S, b0, c0, b, c);
    W carry[V], edge[V];
    Pair<W> all[V];
#pragma unroll
    for (int k = 0; k < V; k++) {
        carry[k] = first_state<K, W>(S, q + k);
        edge[k] = edge_of<K, W>(S, q + k);
        all[k] = Pair<W>{W(1), W(0)};
    }
    if constexpr (PH == APPLY) {
        // what came before this part: a wavefront joins its share of the parts, the workgroup the wavefronts'
        const int64_t share = (part + WT - 1) / WT, from = min(wt * share, part), to = min(from + share, part);
#pragma unroll
        for (int k = 0; k < V; k++) {
            pairs_of[1][wt][lane * V + k] = joined_parts<W>(S, from, to, q + k);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < V; k++)
#pragma unroll
            for (int w = 0; w < WT; w++) {
                const Pair<W> p = pairs_of[1][w][lane * V + k];
                carry[k] = step(p.a, carry[k], p.h);
            }
    }
    int turn = 0;
    for (int64_t u = begin; u < end; u += TURN, turn ^= 1) {
        const int64_t u0 = u + wt * L;
        const bool full = u0 + L <= end;                  // (the same for the wavefront)
        Run<O, V> f;
        if (full) take<O, V, true, PH != PAIRS>(S, P, edge, u0, end, f);
        else take<O, V, false, PH != PAIRS>(S, P, edge, u0, end, f);
        W mine[V];
        if constexpr (WT > 1) {
#pragma unroll
            for (int k = 0; k < V; k++) pairs_of[turn][wt][lane * V + k] = pair_of<O, V>(f, k);
            __syncthreads();
#pragma unroll
            for (int k = 0; k < V; k++) {
                if constexpr (PH == PAIRS) {
                    if (wt == 0) {
#pragma unroll
                        for (int w = 0; w < WT; w++) {
                            const Pair<W> p = pairs_of[turn][w][lane * V + k];
                            all[k].then(p.a, p.h);
                        }
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < WT; w++) {
                        if (w == wt) mine[k] = carry[k];
                        const Pair<W> p = pairs_of[turn][w][lane * V + k];
                        carry[k] = step(p.a, carry[k], p.h);
                    }
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < V; k++) mine[k] = carry[k];
        }
        if constexpr (PH != PAIRS) {
            if (there) {
                if (full) walk<O, V, true>(S, P, f, u0, end, mine);
                else walk<O, V, false>(S, P, f, u0, end, mine);
            }
            if constexpr (WT == 1) {
#pragma unroll
                for (int k = 0; k < V; k++) carry[k] = mine[k];
            }
        }
    }
    if (!there || wt) return;
    if constexpr (PH == PAIRS) {
        W* pairs = (W*)S.pairs + 2 * part * S.cols + q;
#pragma unroll
        for (int k = 0; k < V; k++) { pairs[k] = all[k].a; pairs[S.cols + k] = all[k].h; }
    } else if (end == S.steps) {
#pragma unroll
        for (int k = 0; k < V; k++) put_final<K, T, W>(S, S.channels == 1 ? b + k : b, S.channels == 1 ? c : c + k, q + k, carry[k]);
    }
}

// ---- TILES: as COLUMNS, where 64 adjacent channels are there for every wavefront ------------------------------------------
//
// A wavefront's run of 64 columns is L rows of 64 adjacent elements: it is loaded and stored 16 bytes to a lane, which takes an
// eighth (float32: a quarter) of the instructions and registers, so that the next turn's elements can be on their way while this
// one's are worked on.  What a lane needs, a column, it gets through its wavefront's own piece of LDS.  A tile lies in one
// sequence, whose flags are the same for all its lanes: bits of a scalar.
//
// Training, from inputs that no cache holds: 16 x 2048 x 1024 bfloat16 48 us forward and 73 backward where one element to a lane at
// a time, in the kernel above, takes 59 and 83; 4 x 300 x 8192 13.6 and 19.1 where it takes 25 and 35.  (Two turns ahead, tried
// while no states were kept: 45 us forward instead of 47, 67 backward instead of 66.)

template <class T> struct Tile {
    static constexpr int N = 16 / sizeof(T), LANES = 64 / N, ROWS = N, LOADS = L / ROWS, BYTES = L * 64 * sizeof(T);
    typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(2)));
    uint4 v[LOADS];
    // rows from .. of [0, hi), 0 outside
    __device__ __forceinline__ void load(const char* base, int64_t stride, int64_t from, int64_t hi, int lane) {
#pragma unroll
        for (int l = 0; l < LOADS; l++) {
            const int64_t row = from + l * ROWS + lane / LANES;
            v[l] = uint4{0, 0, 0, 0};
            if (row >= 0 && row < hi) v[l] = __builtin_bit_cast(uint4, (vec)*(const vec __attribute__((address_space(1)))*)((Global)base + (row * stride + lane % LANES * 16)));
        }
    }
    __device__ __forceinline__ void store(char* base, int64_t stride, int64_t from, int64_t hi, int lane) const {
#pragma unroll
        for (int l = 0; l < LOADS; l++) {
            const int64_t row = from + l * ROWS + lane / LANES;
            if (row < hi) *(vec __attribute__((address_space(1)))*)((Global)base + (row * stride + lane % LANES * 16)) = __builtin_bit_cast(vec, v[l]);
        }
    }
    __device__ __forceinline__ void to_rows(char* at, int lane) const {
#pragma unroll
        for (int l = 0; l < LOADS; l++) ((uint4*)at)[l * 64 + lane] = v[l];
    }
    __device__ __forceinline__ void from_rows(const char* at, int lane) {
#pragma unroll
        for (int l = 0; l < LOADS; l++) v[l] = ((const uint4*)at)[l * 64 + lane];
    }
};
// What a wavefront's lanes wrote is there for its other lanes: LDS works in order, the compiler has to keep to it.
__device__ __forceinline__ void rows_written() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// A barrier for what went through LDS; loads from memory stay on their way.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

constexpr int kTileWaves = 8;    // (16 take 0.5 - 1 us longer to begin and gain nothing; 4 leave half the loads out: 61 us for what took 38)

template <class O>
__global__ __launch_bounds__(64 * kTileWaves) void tiles_kernel(Seq S) {
    constexpr Kind K = O::K;
    constexpr int WT = kTileWaves;
    using T = typename O::T;
    using W = typename O::W;
    constexpr int64_t TURN = WT * L;
    constexpr bool back = K == BACKWARD, BEFORE = back && O::SECOND;
    using D = typename O::Second;
    constexpr int FLAGS = L + (BEFORE ? 1 : 0), shift = back ? 1 : 0, BYTES = std::max(Tile<T>::BYTES, Tile<D>::BYTES);
    __shared__ Pair<W> pairs_of[2][WT][64];
    __shared__ __attribute__((aligned(16))) char rows_of[WT][BEFORE ? 3 : 2][BYTES];
    const int lane = threadIdx.x & 63, wt = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t q0 = (int64_t)blockIdx.x * 64, b = q0 / S.channels, c0 = q0 - b * S.channels, q = q0 + lane;
    const char *px = uniform_part<T>(S.x, b, c0), *pg = uniform_part<T>(S.gate, b, c0), *pb = uniform_part<T>(S.before, b, c0);
    const char* pr = uniform_part<uint8_t>(S.resets, b, 0);
    char *ph = (char*)uniform_part<T>(S.h, b, c0), *po = (char*)uniform_part<D>(S.second, b, c0), *pk = (char*)uniform_part<W>(S.keep, b, c0);
    const int64_t size = sizeof(T), sx = S.x.st * size, sg = S.gate.st * size, sb = S.before.st * size;
    char *rx = rows_of[wt][0], *rg = rows_of[wt][1], *rb = rows_of[wt][BEFORE ? 2 : 0];
    W carry = first_state<K, W>(S, q);
    const W edge[1] = {edge_of<K, W>(S, q)};
    Tile<T> x, g, before;
    uint8_t flag = 0;
    T own{};                                          // AGAIN: the gate of the run's last step, and the state before it
    W kept{};
    auto ask = [&](int64_t u0) {
        x.load(px, sx, u0, S.steps, lane);
        if constexpr (O::GATE) g.load(pg, sg, u0 - shift, S.steps, lane);
        if constexpr (BEFORE) before.load(pb, sb, u0 + (O::AGAIN ? 0 : 1), S.steps, lane);
        if constexpr (O::AGAIN) {
            if (u0 + L <= S.steps) own = ((const T __attribute__((address_space(1)))*)((Global)pg + (u0 + L - 1) * sg))[lane];
            if (u0 + L < S.steps) kept = ((const W __attribute__((address_space(1)))*)((Global)pk + u0 / L * S.keep.st * (int64_t)sizeof(W)))[lane];
        }
        if constexpr (O::RESETS) {
            const int64_t at = u0 - shift + lane;
            flag = 0;
            if (lane < FLAGS && at >= 0 && at < S.steps) flag = (uint8_t)pr[at * S.resets.st];
        }
    };
    ask(wt * L);
    const int keep = (int)(S.steps % L);
    int turn = 0;
    for (int64_t u = 0; u < S.steps; u += TURN, turn ^= 1) {
        const int64_t u0 = u + wt * L;
        x.to_rows(rx, lane);
        if constexpr (O::GATE) g.to_rows(rg, lane);
        if constexpr (BEFORE) before.to_rows(rb, lane);
        const uint64_t flags = O::RESETS ? __ballot(flag != 0) : 0;
        Raw<O, 1> raw;
        if constexpr (O::AGAIN) { raw.g[L] = own; raw.kept[0] = kept; }
        rows_written();
        if (u + TURN < S.steps) ask(u0 + TURN);
#pragma unroll
        for (int i = 0; i < L; i++) {
            raw.x[i] = ((const T*)rx)[i * 64 + lane];
            if constexpr (O::GATE) raw.g[i] = ((const T*)rg)[i * 64 + lane];
            if constexpr (BEFORE) raw.before[i] = ((const T*)rb)[i * 64 + lane];
        }
        if constexpr (O::RESETS) {
#pragma unroll
            for (int i = 0; i < FLAGS; i++) raw.r[i] = flags >> i & 1;
        }
        Run<O, 1> f;
        fold<O, 1, false>(S, raw, edge, u0, S.steps, f);
        const Pair<W> own = pair_of<O, 1>(f, 0);
        pairs_of[turn][wt][lane] = own;
        lds_barrier();
        W h = carry, own_kept{};
#pragma unroll
        for (int w = 0; w < WT; w++) {
            if (w == wt) h = carry;
            const Pair<W> p = pairs_of[turn][w][lane];
            carry = step(p.a, carry, p.h);
        }
#pragma unroll
        for (int i = 0; i < L; i++) {
            if (O::KEEP && i == keep) own_kept = h;
            h = step(f.a[i], h, f.x[i]);
            ((T*)rx)[i * 64 + lane] = (T)h;
            if constexpr (O::SECOND) ((D*)rg)[i * 64 + lane] = second_of<O, 1>(f, i, h);
        }
        rows_written();
        Tile<T> out;
        out.from_rows(rx, lane);
        out.store(ph, S.h.st * size, u0, S.steps, lane);
        if constexpr (O::SECOND) {
            Tile<D> beside;
            beside.from_rows(rg, lane);
            beside.store(po, S.second.st * (int64_t)sizeof(D), u0, S.steps, lane);
        }
        if constexpr (O::KEEP) {
            if (u0 + keep < S.steps) ((W __attribute__((address_space(1)))*)((Global)pk + keep_offset<O>(S, u0 + keep)))[lane] = own_kept;
        }
        rows_written();
    }
    if (wt == 0) put_final<K, T, W>(S, b, c0 + lane, q, carry);
}

// ---- RUNS: 64 runs of one column to a wavefront, WT wavefronts to a column; or, of short ones, several columns ------------

// COUNT steps from `from`, 16 bytes at a time (at any alignment); DIR: whether they rise or fall in memory.  Not FULL: one by
// one, what lies outside [0, hi) is 0.
template <class E, int DIR, int COUNT, bool FULL>
__device__ __forceinline__ void get_run(const char* base, int64_t from, int64_t hi, E* to) {
    constexpr int VN = (int)(16 / sizeof(E)) < COUNT ? (int)(16 / sizeof(E)) : COUNT;
    const E* p = (const E*)base + (DIR > 0 ? from : -(from + COUNT - 1));
    if constexpr (FULL) {
#pragma unroll
        for (int j = 0; j < COUNT; j += VN) {
            const typename Vec<E, VN>::type w = *reinterpret_cast<const typename Vec<E, VN>::type*>(p + j);
#pragma unroll
            for (int k = 0; k < VN; k++) to[DIR > 0 ? j + k : COUNT - 1 - j - k] = w[k];
        }
    } else {
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            to[i] = E(0);
            if (from + i >= 0 && from + i < hi) to[i] = p[DIR > 0 ? i : COUNT - 1 - i];
        }
    }
}
template <class E, int DIR, bool FULL>
__device__ __forceinline__ void put_run(char* base, int64_t from, int64_t hi, const E* v) {
    constexpr int VN = (int)(16 / sizeof(E)) < L ? (int)(16 / sizeof(E)) : L;
    E* p = (E*)base + (DIR > 0 ? from : -(from + L - 1));
    if constexpr (FULL) {
#pragma unroll
        for (int j = 0; j < L; j += VN) {
            typename Vec<E, VN>::type w;
#pragma unroll
            for (int k = 0; k < VN; k++) w[k] = v[DIR > 0 ? j + k : L - 1 - j - k];
            *reinterpret_cast<typename Vec<E, VN>::type*>(p + j) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < L; i++)
            if (from + i < hi) p[DIR > 0 ? i : L - 1 - i] = v[i];
    }
}

// The run's own COUNT steps, with the one before them (BEFORE) or behind them (else); 0 where there is none.
template <class E, int DIR, bool FULL, bool BEFORE, int COUNT>
__device__ __forceinline__ void get_shifted(const char* base, int64_t u0, int64_t end, int64_t hi, E* to) {
    if constexpr (FULL) {
        E own[L];
        get_run<E, DIR, L, true>(base, u0, end, own);
        get_run<E, DIR, 1, false>(base, BEFORE ? u0 - 1 : u0 + L, hi, BEFORE ? to : to + L - 1);
#pragma unroll
        for (int i = 1; i < (BEFORE ? COUNT : L); i++) to[BEFORE ? i : i - 1] = own[BEFORE ? i - 1 : i];
    } else get_run<E, DIR, COUNT, false>(base, BEFORE ? u0 - 1 : u0 + 1, hi, to);
}

template <class O, int DIR, bool FULL, bool APPLYING>
__device__ __forceinline__ void load_run(const Seq& S, const Place& P, int64_t u0, int64_t end, Raw<O, 1>& d) {
    using T = typename O::T;
    get_run<T, DIR, L, FULL>(P.x, u0, end, d.x);
    if constexpr (O::K == BACKWARD) {
        if constexpr (O::GATE) get_shifted<T, DIR, FULL, true, L + (O::AGAIN && APPLYING ? 1 : 0)>(P.gate, u0, end, end, d.g);
        if constexpr (O::RESETS) get_shifted<uint8_t, DIR, FULL, true, L + (O::SECOND ? 1 : 0)>(P.resets, u0, end, end, d.r);
        if constexpr (O::AGAIN && APPLYING) {
            get_run<T, DIR, L, FULL>(P.before, u0, end, d.before);
            if (u0 + L < S.steps) d.kept[0] = ((const typename O::W*)P.keep)[u0 / L * S.keep.st];
        } else if constexpr (O::SECOND && APPLYING) get_shifted<T, DIR, FULL, false, L>(P.before, u0, end, S.steps, d.before);
    } else {
        if constexpr (O::GATE) get_run<T, DIR, L, FULL>(P.gate, u0, end, d.g);
        if constexpr (O::RESETS) get_run<uint8_t, DIR, L, FULL>(P.resets, u0, end, d.r);
        if constexpr (O::K == ADVANTAGES) get_shifted<float, DIR, FULL, true, L + 1>(P.before, u0, end, end, d.v);
    }
}

template <class O, int DIR, bool FULL, bool APPLYING>
__device__ __forceinline__ void take_run(const Seq& S, const Place& P, const typename O::W (&edge)[1], int64_t u0, int64_t end, Run<O, 1>& f) {
    Raw<O, 1> raw;
    load_run<O, DIR, FULL, APPLYING>(S, P, u0, end, raw);
    fold<O, 1, FULL>(S, raw, edge, u0, end, f);
}

template <class O, int DIR, bool FULL>
__device__ __forceinline__ void walk_run(const Seq& S, const Place& P, const Run<O, 1>& f, int64_t u0, int64_t end, typename O::W h) {
    using E = typename O::Out;
    using D = typename O::Second;
    E out[L];
    D second[O::SECOND ? L : 1];
    const int keep = (int)(S.steps % L);
    typename O::W kept{};
#pragma unroll
    for (int i = 0; i < L; i++) {
        if (O::KEEP && i == keep) kept = h;
        h = step(f.a[i], h, f.x[i]);
        out[i] = (E)h;
        if constexpr (O::SECOND) second[i] = second_of<O, 1>(f, i, h);
    }
    put_run<E, DIR, FULL>(P.h, u0, end, out);
    if constexpr (O::SECOND) put_run<D, DIR, FULL>(P.second, u0, end, second);
    if constexpr (O::KEEP) {
        if (u0 + keep < S.steps) *(typename O::W*)(P.keep + keep_offset<O>(S, u0 + keep)) = kept;
    }
}

template <class W> __device__ __forceinline__ Pair<W> up(const Pair<W>& p, int by) { return Pair<W>{__shfl_up(p.a, by), __shfl_up(p.h, by)}; }
template <class W> __device__ __forceinline__ void wave_scan(Pair<W>& p, int lane, int group) {
#pragma unroll
    for (int by = 1; by < 64; by <<= 1) {
        if (by >= group) break;
        const Pair<W> o = up(p, by);
        if (lane >= by) p.after(o);
    }
}

template <class O, int DIR, int WT, Phase PH>
__global__ __launch_bounds__(WT == 1 ? 256 : 64 * WT) void runs_kernel(Seq S) {
    constexpr Kind K = O::K;
    using T = typename O::T;
    using W = typename O::W;
    constexpr int64_t TURN = WT * 64 * L;
    __shared__ W pa[2][WT], ph[2][WT];
    const int group = WT > 1 ? 64 : (int)S.group;     // lanes of a column
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wt = WT > 1 ? wave : 0;
    const int lane = WT > 1 ? threadIdx.x & 63 : threadIdx.x & (group - 1), last = (threadIdx.x & 63) | (group - 1);
    const int64_t q = WT > 1 ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * 256 + threadIdx.x) / group;
    if (q >= S.cols) return;                          // WT > 1: a whole workgroup, else whole groups of lanes and no barrier
    const int64_t part = PH == WHOLE ? 0 : blockIdx.y;
    const int64_t begin = part * S.part, end = PH == WHOLE ? S.steps : min(begin + S.part, S.steps);
    const Place P = place_of<O>(S, q, 0, q, 0);       // (one channel: the column is the sequence)
    W carry = first_state<K, W>(S, q);
    const W edge[1] = {edge_of<K, W>(S, q)};
    Pair<W> all{W(1), W(0)};
    const int64_t mine = (int64_t)(wt * 64 + lane) * L, turn_steps = WT > 1 ? TURN : group * L;
    if constexpr (PH == APPLY) {
        const int64_t share = (part + WT * 64 - 1) / (WT * 64), from = min((wt * 64 + lane) * share, part), to = min(from + share, part);
        Pair<W> p = joined_parts<W>(S, from, to, q);
        wave_scan(p, lane, 64);
        if (lane == 63) { pa[1][wt] = p.a; ph[1][wt] = p.h; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WT; w++) carry = step(pa[1][w], carry, ph[1][w]);
    }
    int turn = 0;
    for (int64_t u = begin; u < end; u += turn_steps, turn ^= 1) {
        const int64_t u0 = u + mine;
        Run<O, 1> f;
        if (u0 + L <= end) take_run<O, DIR, true, PH != PAIRS>(S, P, edge, u0, end, f);
        else if (u0 < end) take_run<O, DIR, false, PH != PAIRS>(S, P, edge, u0, end, f);
        else {
#pragma unroll
            for (int i = 0; i < L; i++) { f.a[i] = W(1); f.x[i] = W(0); if constexpr (O::SECOND) f.extra[i] = 0; }
        }
        Pair<W> p = pair_of<O, 1>(f, 0);
        wave_scan(p, lane, group);
        Pair<W> front = up(p, 1);                     // of the lanes before this one
        if (lane == 0) front = Pair<W>{W(1), W(0)};
        Pair<W> whole{__shfl(p.a, last), __shfl(p.h, last)};
        if constexpr (WT > 1) {
            if (lane == 0) { pa[turn][wt] = whole.a; ph[turn][wt] = whole.h; }
            __syncthreads();
            Pair<W> before{W(1), W(0)}, total{W(1), W(0)};
#pragma unroll
            for (int w = 0; w < WT; w++) {
                if (w == wt) before = total;
                total.then(pa[turn][w], ph[turn][w]);
            }
            front.after(before);
            whole = total;
        }
        if constexpr (PH == PAIRS) {
            all.then(whole.a, whole.h);
        } else {
            const W h = step(front.a, carry, front.h);
            carry = step(whole.a, carry, whole.h);
            if (u0 + L <= end) walk_run<O, DIR, true>(S, P, f, u0, end, h);
            else if (u0 < end) walk_run<O, DIR, false>(S, P, f, u0, end, h);
        }
    }
    if (wt || lane) return;
    if constexpr (PH == PAIRS) {
        W* pairs = (W*)S.pairs + 2 * part * S.cols + q;
        pairs[0] = all.a;
        pairs[S.cols] = all.h;
    } else if (end == S.steps) put_final<K, T, W>(S, q, 0, q, carry);
}

// ---- host side ---------------------------------------------------------------------------------------------------------

View ordered(const lrn_view* v, int64_t steps, int64_t bytes, bool against) {
    if (!v || !v->data) return View{nullptr, 0, 0, 0};
    View r{v->data, v->st, v->sb, v->sc};
    if (against && steps > 0) {
        r.p = (const char*)v->data + (steps - 1) * v->st * bytes;
        r.st = -v->st;
    }
    return r;
}

int checked(const lrn_seq* q, const char* who) {
    if (!q) return fail(-1, "%s: null sequence", who);
    if (q->steps < 0 || q->batch < 0 || q->channels < 0) return fail(-1, "%s: %lld steps, batch %lld, %lld channels", who, (long long)q->steps, (long long)q->batch, (long long)q->channels);
    if (q->dtype < LRN_F32 || q->dtype > LRN_F64) return fail(-1, "%s: dtype %d", who, q->dtype);
    return 0;
}

int check_views(const char* who, std::initializer_list<const lrn_view*> views) {
    for (const lrn_view* v : views)
        if (v && v->data && (v->sb < 0 || v->sc < 0)) return fail(-1, "%s: batch and channel strides may not be negative", who);
    return 0;
}

int64_t bytes_of(int dtype) { return dtype == LRN_F64 ? 8 : dtype == LRN_F32 ? 4 : 2; }

// How the steps are dealt out.  It goes by the sequence's sizes alone, so that the workspace can be asked for beforehand.
struct Deal {
    int wt;                     // wavefronts along time
    int64_t part, parts;
};

// COLUMNS: one wavefront where a column's steps are a run or the columns alone fill the GPU (2048 wavefronts of 64 columns),
// else 4 or 16 behind one another; parts where even 16 leave compute units without a workgroup, of 256 steps at least.
Deal deal_columns(int64_t steps, int64_t cols) {
    const int64_t tiles = cdiv(cols, 64);
    Deal d{1, steps, 1};
    if (steps > L && tiles < 2048) d.wt = steps > 4 * L && tiles < 1024 ? 16 : 4;
    if (d.wt == 16 && tiles <= 128 && steps >= 512) {
        d.part = std::max<int64_t>(256, cdiv(cdiv(steps, cdiv(512, tiles)), 128) * 128);
        d.parts = cdiv(steps, d.part);
    }
    return d;
}
// RUNS: a wavefront's turn is 512 steps
Deal deal_runs(int64_t steps, int64_t cols) {
    Deal d{1, steps, 1};
    if (steps > 64 * L && cols < 2048) d.wt = steps > 256 * L && cols < 512 ? 16 : 4;
    if (d.wt == 16 && cols <= 128 && steps >= 4096 * L) {
        d.part = std::max<int64_t>(1024 * L, cdiv(cdiv(steps, cdiv(256, cols)), 1024 * L) * 1024 * L);
        d.parts = cdiv(steps, d.part);
    }
    return d;
}

int64_t pair_bytes(const lrn_seq* q) {
    const int64_t cols = q->batch * q->channels;
    if (cols == 0) return 0;
    int64_t parts = deal_columns(q->steps, cols).parts;
    if (q->channels == 1) parts = std::max(parts, deal_runs(q->steps, cols).parts);
    return parts > 1 ? parts * 2 * cols * (q->dtype == LRN_F64 ? 8 : 4) : 0;
}

// 16 wavefronts of a workgroup have 128 registers each, which float64 states and elements do not fit: 8 there.
template <class O> constexpr int kMany = std::is_same<typename O::T, double>::value ? 8 : 16;

// A lane's part of an address has 32 bits: how far the columns of one tile lie apart in a view.
bool near(const View& v, const Seq& S, int64_t size, int tile) {
    constexpr int64_t far = (int64_t)1 << 40;
    const int64_t over = std::min(S.cols / S.channels - 1, tile / S.channels + 1);
    return !v.p || (v.sb <= far && v.sc <= far / S.channels && over * v.sb * size + S.channels * v.sc * size < ((int64_t)1 << 32));
}
template <class O> bool near(const Seq& S, int tile) {
    constexpr int64_t n = sizeof(typename O::T);
    return near(S.keep, S, sizeof(typename O::W), tile) && near(S.x, S, n, tile) && near(S.gate, S, n, tile) && near(S.before, S, n, tile) && near(S.resets, S, 1, tile) &&
           near(S.h, S, n, tile) && near(S.second, S, sizeof(typename O::Second), tile);
}

template <class O, int V, int WT> void launch_columns(Seq& S, const Deal& d, hipStream_t stream) {
    const bool flat = V > 1 || near<O>(S, 64);
    if (!flat) {
        // Channels that lie so far apart that 64 of them pass 32 bits (time is the fast index of a long trajectory): fewer to a tile.
        S.width = 64;
        for (const View* v : {&S.x, &S.gate, &S.before, &S.h, &S.second, &S.keep})
            while (S.width > 1 && v->p && v->sc >= ((int64_t)1 << 32) / (S.width * (int64_t)sizeof(typename O::W))) S.width /= 2;
        S.tight = cdiv(S.channels, S.width);
    }
    const int64_t tiles = cdiv(flat ? cdiv(S.cols, 64 * V) : S.cols / S.channels * S.tight, WT == 1 ? 4 : 1);
    const int threads = WT == 1 ? 256 : 64 * WT;
    if (d.parts > 1) {
        if constexpr (WT == kMany<O>) {
            columns_kernel<O, V, WT, PAIRS><<<dim3((unsigned)tiles, (unsigned)d.parts), threads, 0, stream>>>(S);
            columns_kernel<O, V, WT, APPLY><<<dim3((unsigned)tiles, (unsigned)d.parts), threads, 0, stream>>>(S);
        }
    } else if constexpr (V == 1 || WT != kMany<O>) columns_kernel<O, V, WT, WHOLE><<<(unsigned)tiles, threads, 0, stream>>>(S);
}
template <class O, int DIR, int WT> void launch_runs(Seq& S, const Deal& d, hipStream_t stream) {
    // As many lanes to a column as it has runs, so that short sequences share a wavefront (1 048 576 of 16 float32: 23 us, 5.9 TB/s
    // out of the last-level cache; a wavefront to each took 297, by columns 90).
    S.group = 1;
    while (S.group < 64 && S.group * L < S.steps) S.group *= 2;
    const int64_t blocks = WT == 1 ? cdiv(S.cols * S.group, 256) : S.cols;
    const int threads = WT == 1 ? 256 : 64 * WT;
    if (d.parts > 1) {
        if constexpr (WT == kMany<O>) {
            runs_kernel<O, DIR, WT, PAIRS><<<dim3((unsigned)blocks, (unsigned)d.parts), threads, 0, stream>>>(S);
            runs_kernel<O, DIR, WT, APPLY><<<dim3((unsigned)blocks, (unsigned)d.parts), threads, 0, stream>>>(S);
        }
    } else runs_kernel<O, DIR, WT, WHOLE><<<(unsigned)blocks, threads, 0, stream>>>(S);
}
template <class O, int DIR> void launch_runs(Seq& S, const Deal& d, hipStream_t stream) {
    if (d.wt == 1) launch_runs<O, DIR, 1>(S, d, stream);
    else if (d.wt == 4) launch_runs<O, DIR, 4>(S, d, stream);
    else launch_runs<O, DIR, kMany<O>>(S, d, stream);
}

bool dense(const View& v, int64_t channels) { return !v.p || (channels == 1 ? v.sb : v.sc) == 1; }

template <class O> int launch(Seq S, void* workspace, hipStream_t stream, const char* who) {
    // time is the fast index of everything there is (a view that is the same at all steps, say, is read by columns)
    const int64_t st = S.h.st;
    bool runs = S.channels == 1 && S.steps > 1 && (st == 1 || st == -1);
    for (const View* v : {&S.x, &S.gate, &S.resets, &S.before, &S.h, &S.second}) runs = runs && (!v->p || v->st == st);
    for (const View* v : {&S.x, &S.h}) runs = runs && (S.cols == 1 || v->sb != 1);
    runs = runs && S.cols < ((int64_t)1 << 26) - 4;   // (a grid has fewer than 2^32 lanes)
    const Deal d = runs ? deal_runs(S.steps, S.cols) : deal_columns(S.steps, S.cols);
    if (d.parts > 65535 || S.cols > ((int64_t)1 << 31)) return fail(-1, "%s: %lld steps of %lld columns are too many for one call", who, (long long)S.steps, (long long)S.cols);
    S.part = d.part;
    S.pairs = workspace;
    if (runs) {
        if (st == 1) launch_runs<O, 1>(S, d, stream);
        else launch_runs<O, -1>(S, d, stream);
    } else {
        // Two columns to a lane, wider rows and half the instructions: in sequences in parts where it takes fewer tiles (131 073
        // steps of 72 float32: 45 us instead of 55; float64 gains nothing), and for advantages where four wavefronts stand behind
        // one another for more than a turn: 21 bytes a step keep the memory busy with half the wavefronts, and rows that start
        // off a cache line are fetched by fewer of them (288 steps of 65 534 sequences, float64 rewards: 102 us instead of 117;
        // 65 536: 86 instead of 90; 2000 steps 655 instead of 838 and 540 instead of 549).  Elsewhere one column is level or
        // ahead: 32 steps of 65 536 10.9 instead of 12.0, 288 of 131 072 float32 118 instead of 129, 262 144 level; in parts 2048
        // x 2000 float64 31 instead of 41.
        const bool even = S.cols % 2 == 0 && (S.channels == 1 || S.channels % 2 == 0) && dense(S.x, S.channels) && dense(S.gate, S.channels) &&
                          dense(S.before, S.channels) && dense(S.h, S.channels) && dense(S.second, S.channels) && dense(S.keep, S.channels) && near<O>(S, 128);
        if constexpr (O::K == ADVANTAGES) {
            if (even && d.wt == 4 && S.steps > 4 * L) return launch_columns<O, 2, 4>(S, d, stream), 0;
        } else if constexpr (sizeof(typename O::T) <= 4) {
            if (even && d.parts > 1 && S.cols > 64) return launch_columns<O, 2, kMany<O>>(S, d, stream), 0;
        }
        // Tiles where wavefronts stand behind one another, in one part, and all eight have steps where there are tiles enough
        // (64 x 500 x 1024 bfloat16: 67.7 us backward instead of 75.6, 32 x 500 x 1024 33 instead of 49).  Where a wavefront has
        // all steps the memory is busy without: 256 x 300 x 1024 bfloat16 113 us forward on both sides, 172 backward, with them
        // 177; at half of that batch they would be ahead (59 instead of 63, 84 instead of 106).
        if constexpr (O::K != ADVANTAGES && sizeof(typename O::T) <= 4) {
            bool tiles = (d.wt == 16 || (d.wt == 4 && S.steps > kTileWaves * L)) && d.parts == 1 && S.channels % 64 == 0;
            for (const View* v : {&S.x, &S.gate, &S.before, &S.h, &S.second, &S.keep}) tiles = tiles && (!v->p || v->sc == 1);
            if (tiles) return tiles_kernel<O><<<(unsigned)(S.cols / 64), 64 * kTileWaves, 0, stream>>>(S), 0;
        }
        if (d.wt == 1) launch_columns<O, 1, 1>(S, d, stream);
        else if (d.wt == 4) launch_columns<O, 1, 4>(S, d, stream);
        else launch_columns<O, 1, kMany<O>>(S, d, stream);
    }
    return 0;
}

template <Kind K, class T> int run(const Seq& S, void* workspace, hipStream_t stream, const char* who) {
    int rc;
    if constexpr (K == ADVANTAGES) rc = launch<Op<K, T, false, true, true>>(S, workspace, stream, who);
    else {
        const bool resets = S.resets.p;
        if (S.keep.p && K == SCAN) {
            if constexpr (sizeof(T) == 2) rc = resets ? launch<Op<K, T, true, true, true>>(S, workspace, stream, who) : launch<Op<K, T, true, false, true>>(S, workspace, stream, who);
            else rc = fail(-1, "%s: 16-bit sequences only", who);
        } else if (sizeof(T) == 2 && K == BACKWARD && S.second.p && S.sums) {
            using P = std::conditional_t<sizeof(T) == 2 && K == BACKWARD, float, T>;
            if (resets) rc = launch<Op<K, T, true, true, K == BACKWARD, P>>(S, workspace, stream, who);
            else rc = launch<Op<K, T, true, false, K == BACKWARD, P>>(S, workspace, stream, who);
        } else if (K == BACKWARD && S.second.p) {
            if (resets) rc = launch<Op<K, T, true, true, K == BACKWARD>>(S, workspace, stream, who);
            else rc = launch<Op<K, T, true, false, K == BACKWARD>>(S, workspace, stream, who);
        } else if (S.gate.p) {
            if (resets) rc = launch<Op<K, T, true, true, false>>(S, workspace, stream, who);
            else rc = launch<Op<K, T, true, false, false>>(S, workspace, stream, who);
        } else {
            if (resets) rc = launch<Op<K, T, false, true, false>>(S, workspace, stream, who);
            else rc = launch<Op<K, T, false, false, false>>(S, workspace, stream, who);
        }
    }
    if (rc) return rc;
    LRN_LAUNCHED(who);
    return 0;
}

template <Kind K> int run(const Seq& S, int dtype, void* workspace, hipStream_t stream, const char* who) {
    if (dtype == LRN_F32) return run<K, float>(S, workspace, stream, who);
    if (dtype == LRN_F64) return run<K, double>(S, workspace, stream, who);
    if constexpr (K != ADVANTAGES) {
        if (dtype == LRN_BF16) return run<K, bf16>(S, workspace, stream, who);
        return run<K, f16>(S, workspace, stream, who);
    }
    return 0;
}

int check_workspace(const lrn_seq* q, const void* workspace, int64_t bytes, const char* who) {
    const int64_t need = pair_bytes(q);
    if (need && (!workspace || bytes < need)) return fail(-1, "%s: a workspace of %lld bytes is needed, got %lld", who, (long long)need, (long long)bytes);
    return 0;
}

int scan(const char* who, int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* x, const lrn_view* gate, double gate_const,
         const lrn_view* resets, const void* initial, const lrn_view* h_out, const lrn_view* kept_out, void* final_out, void* workspace,
         int64_t workspace_bytes) {
    if (int rc = checked(seq, who)) return rc;
    if (seq->batch * seq->channels == 0) return 0;
    if (seq->steps && (!x || !x->data || !h_out || !h_out->data)) return fail(-1, "%s: null x or h", who);
    if (int rc = check_views(who, {x, gate, resets, h_out, kept_out})) return rc;
    if (int rc = check_workspace(seq, workspace, workspace_bytes, who)) return rc;
    LRN_ON_DEVICE(device);
    const bool rev = seq->reverse != 0;
    const int64_t n = bytes_of(seq->dtype);
    Seq S{};
    S.steps = seq->steps; S.cols = seq->batch * seq->channels; S.channels = seq->channels;
    S.x = ordered(x, seq->steps, n, rev); S.gate = ordered(gate, seq->steps, n, rev);
    S.resets = ordered(resets, seq->steps, 1, rev); S.h = ordered(h_out, seq->steps, n, rev);
    S.keep = ordered(seq->steps ? kept_out : nullptr, 0, 4, false);
    S.gate_const = gate_const; S.initial = initial; S.final = final_out;
    return run<SCAN>(S, seq->dtype, workspace, (hipStream_t)hip_stream, who);
}

// `states`: h, or x beside `kept`
int backward(const char* who, int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* gate, double gate_const, const lrn_view* resets,
             const void* initial, const lrn_view* states, const lrn_view* kept, const lrn_view* g_h, const void* g_final, const lrn_view* grad_x_out,
             const lrn_view* grad_gate_out, bool sums, void* grad_initial_out, void* workspace, int64_t workspace_bytes) {
    if (int rc = checked(seq, who)) return rc;
    if (seq->batch * seq->channels == 0) return 0;
    if (seq->steps && (!g_h || !g_h->data || !grad_x_out || !grad_x_out->data)) return fail(-1, "%s: null g_h or grad_x", who);
    const bool want_gate = seq->steps && grad_gate_out && grad_gate_out->data;
    if (want_gate && (!states || !states->data || !gate || !gate->data)) return fail(-1, "%s: null %s or gate", who, kept ? "x" : "h");
    if (int rc = check_views(who, {gate, resets, states, kept, g_h, grad_x_out, grad_gate_out})) return rc;
    if (int rc = check_workspace(seq, workspace, workspace_bytes, who)) return rc;
    LRN_ON_DEVICE(device);
    const bool rev = seq->reverse == 0;
    const int64_t n = bytes_of(seq->dtype);
    Seq S{};
    S.steps = seq->steps; S.cols = seq->batch * seq->channels; S.channels = seq->channels;
    S.x = ordered(g_h, seq->steps, n, rev); S.gate = ordered(gate, seq->steps, n, rev);
    S.resets = ordered(resets, seq->steps, 1, rev); S.before = ordered(want_gate ? states : nullptr, seq->steps, n, rev);
    S.keep = ordered(want_gate ? kept : nullptr, 0, 4, false);
    S.h = ordered(grad_x_out, seq->steps, n, rev); S.second = ordered(want_gate ? grad_gate_out : nullptr, seq->steps, sums ? 4 : n, rev);
    S.sums = sums; S.gate_const = gate_const; S.initial = g_final; S.edge = initial; S.final = grad_initial_out;
    return run<BACKWARD>(S, seq->dtype, workspace, (hipStream_t)hip_stream, who);
}

int keeping(const lrn_seq* seq, const lrn_view* gate, const lrn_view* kept, const char* who) {
    if (int rc = checked(seq, who)) return rc;
    if (seq->dtype != LRN_BF16 && seq->dtype != LRN_F16) return fail(-1, "%s: dtype %d: 16-bit sequences only (h holds the states of the others)", who, seq->dtype);
    if (seq->steps && seq->batch * seq->channels && (!gate || !gate->data || !kept || !kept->data)) return fail(-1, "%s: null gate or kept states", who);
    return 0;
}

int64_t workspace_of(const lrn_seq* q) { return q && checked(q, "workspace") == 0 ? pair_bytes(q) : 0; }

}  // namespace
}  // namespace lrn

using namespace lrn;

extern "C" {

int64_t lrn_scan_workspace(const lrn_seq* seq) { return workspace_of(seq); }

int lrn_scan(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* x, const lrn_view* gate,
             double gate_const, const lrn_view* resets, const void* initial, const lrn_view* h_out, void* final_out, void* workspace,
             int64_t workspace_bytes) {
    return scan("lrn_scan", device, hip_stream, seq, x, gate, gate_const, resets, initial, h_out, nullptr, final_out, workspace, workspace_bytes);
}

int lrn_scan_keep(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* x, const lrn_view* gate,
                  const lrn_view* resets, const void* initial, const lrn_view* h_out, const lrn_view* kept_out, void* final_out,
                  void* workspace, int64_t workspace_bytes) {
    if (int rc = keeping(seq, gate, kept_out, "lrn_scan_keep")) return rc;
    return scan("lrn_scan_keep", device, hip_stream, seq, x, gate, 0.0, resets, initial, h_out, kept_out, final_out, workspace, workspace_bytes);
}

int lrn_scan_backward(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* gate, double gate_const,
                      const lrn_view* resets, const void* initial, const lrn_view* h, const lrn_view* g_h,
                      const void* g_final, const lrn_view* grad_x_out, const lrn_view* grad_gate_out,
                      void* grad_initial_out, void* workspace, int64_t workspace_bytes) {
    if (seq && (seq->dtype == LRN_BF16 || seq->dtype == LRN_F16) && grad_gate_out && grad_gate_out->data)
        return fail(-1, "lrn_scan_backward: h holds rounded states: lrn_scan_keep_backward has the gate's gradient of 16-bit sequences");
    return backward("lrn_scan_backward", device, hip_stream, seq, gate, gate_const, resets, initial, h, nullptr, g_h, g_final, grad_x_out, grad_gate_out,
                    false, grad_initial_out, workspace, workspace_bytes);
}

int lrn_scan_keep_backward(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* x, const lrn_view* gate,
                           const lrn_view* resets, const void* initial, const lrn_view* kept, const lrn_view* g_h,
                           const void* g_final, const lrn_view* grad_x_out, const lrn_view* grad_gate_out, int32_t grad_gate_dtype,
                           void* grad_initial_out, void* workspace, int64_t workspace_bytes) {
    if (int rc = keeping(seq, gate, kept, "lrn_scan_keep_backward")) return rc;
    if (seq->steps && (!grad_gate_out || !grad_gate_out->data)) return fail(-1, "lrn_scan_keep_backward: null grad_gate");
    if (grad_gate_dtype != LRN_F32 && grad_gate_dtype != seq->dtype) return fail(-1, "lrn_scan_keep_backward: grad_gate of dtype %d", grad_gate_dtype);
    return backward("lrn_scan_keep_backward", device, hip_stream, seq, gate, 0.0, resets, initial, x, kept, g_h, g_final, grad_x_out, grad_gate_out,
                    grad_gate_dtype == LRN_F32, grad_initial_out, workspace, workspace_bytes);
}

int64_t lrn_advantages_workspace(const lrn_seq* seq) { return workspace_of(seq); }

int lrn_advantages(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* rewards, const lrn_view* values,
                   const lrn_view* ends, const float* last_values, double gamma, double lam, const lrn_view* advantage_out,
                   const lrn_view* target_out, void* workspace, int64_t workspace_bytes) {
    if (int rc = checked(seq, "lrn_advantages")) return rc;
    if (seq->channels != 1) return fail(-1, "lrn_advantages: %lld channels", (long long)seq->channels);
    if (seq->dtype != LRN_F32 && seq->dtype != LRN_F64) return fail(-1, "lrn_advantages: dtype %d", seq->dtype);
    if (seq->batch == 0 || seq->steps == 0) return 0;
    if (!rewards || !rewards->data || !values || !values->data || !ends || !ends->data || !last_values || !advantage_out ||
        !advantage_out->data || !target_out || !target_out->data)
        return fail(-1, "lrn_advantages: null argument");
    if (int rc = check_views("lrn_advantages", {rewards, values, ends, advantage_out, target_out})) return rc;
    if (int rc = check_workspace(seq, workspace, workspace_bytes, "lrn_advantages")) return rc;
    LRN_ON_DEVICE(device);
    Seq S{};
    S.steps = seq->steps; S.cols = seq->batch; S.channels = 1;
    S.x = ordered(rewards, seq->steps, bytes_of(seq->dtype), true); S.before = ordered(values, seq->steps, 4, true);
    S.resets = ordered(ends, seq->steps, 1, true);
    S.h = ordered(advantage_out, seq->steps, 4, true); S.second = ordered(target_out, seq->steps, 4, true);
    S.gate_const = gamma * lam; S.scale = gamma; S.edge = last_values;
    return run<ADVANTAGES>(S, seq->dtype, workspace, (hipStream_t)hip_stream, "lrn_advantages");
}

}  // extern "C"
