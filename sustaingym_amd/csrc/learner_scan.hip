// learner_scan.hip — gfx950 kernels of lrn_scan / lrn_scan_backward / lrn_advantages (include/learner_ops.h).
//
// All three are h_u = a_u h_{u-1} + x_u along an order u of the steps; what differs is what x, a and the outputs are:
//   scan       u runs with the sequence, x and a are read
//   backward   u runs against it: x_u = g_h, a_u = the gate of the step before in this order (1 in front of the first, so
//              that g_final enters as the state), and beside h = grad_x comes grad_gate = h * (the state before the step)
//   advantages u runs against time: x_u = d_t, a_u = gamma lam (1 - end_t), and beside h comes h + V_t
//
// A run of steps acts on the state in front of it as h -> A h + H, and two runs in a row as (A2 A1, A2 H1 + H2).  So the steps
// are dealt out in runs of L to lanes that hold them in registers: each computes its (A, H) from a state of 0, the states in
// front of the runs come from the pairs of the runs before, and each lane walks its run again with the right state and writes.
// Every element is read once.  Where there are too few columns to fill the GPU, the sequence is also cut into parts: a first
// launch writes the parts' pairs to the workspace, a second one starts each part from the pairs before it (x and a are then
// read twice, the second time mostly from the last-level cache).
//
// Two layouts.  COLUMNS: lanes lie along adjacent channels (or sequences, where time is the slow index), wavefronts of a
// workgroup along time; pairs go through LDS.  RUNS: time is the fast index, so lanes lie along time, pairs go through a
// wavefront scan.  State, pairs and products are float32 (float64 for float64 sequences) whatever the elements' type.
//
// A coefficient of exactly 0 cuts: nothing of the state in front enters, whatever it holds.
#include <algorithm>

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
    View x, gate, resets, before, h, gate_out;
    double gate_const, scale;   // advantages: gamma lam, gamma
    const void* initial;
    const void* edge;           // backward: the initial state; advantages: V behind the last step (float32)
    void* final;
    int64_t part;               // steps of a part
    void* pairs;                // [parts][2][cols]
};

enum Kind { SCAN, BACKWARD, ADVANTAGES };
enum Phase { WHOLE, PAIRS, APPLY };

template <class T> struct State { using type = float; };
template <> struct State<double> { using type = double; };

template <class W> __device__ __forceinline__ W step(W a, W h, W x) { return a == W(0) ? x : a * h + x; }

// (A, H) of a run
template <class W> struct Pair {
    W a, h;
    __device__ __forceinline__ void then(W a2, W x) { h = step(a2, h, x); a = a2 == W(0) ? W(0) : a2 * a; }
    // what came before it
    __device__ __forceinline__ void after(const Pair& first) { h = step(a, first.h, h); a = a == W(0) ? W(0) : a * first.a; }
};

constexpr int L = 8;             // steps of a lane's run

// The elements of one lane's run: L steps of V adjacent columns.
template <Kind K, class T, int V>
struct Run {
    using W = typename State<T>::type;
    static constexpr int N = L * V;
    T x[N];
    T g[N];                      // SCAN: gate of the step; BACKWARD: of the step before in this order
    T before[K == BACKWARD ? N : 1];
    float v[K == ADVANTAGES ? N + V : 1];     // values of the steps u0 - 1 .. u0 + L - 1
    uint8_t r[N + V];            // SCAN, ADVANTAGES: flags of u0 ..; BACKWARD: of u0 - 1 ..

    // the coefficient and the addend of step i
    __device__ __forceinline__ W coefficient(const Seq& S, int i, int k) const {
        const bool cut = r[i * V + k] != 0;
        if constexpr (K == ADVANTAGES) return cut ? W(0) : (W)S.gate_const;
        else return cut ? W(0) : (W)g[i * V + k];
    }
    __device__ __forceinline__ W addend(const Seq& S, int i, int k) const {
        const W e = (W)x[i * V + k];
        if constexpr (K == ADVANTAGES) {
            const W now = (W)v[(i + 1) * V + k], next = (W)v[i * V + k];
            return r[i * V + k] ? e - now : e + (W)S.scale * next - now;
        } else return e;
    }
};

// ---- loads and stores --------------------------------------------------------------------------------------------------

template <class E, int V> struct Vec { typedef E type __attribute__((ext_vector_type(V), aligned(sizeof(E)))); };

// V adjacent columns at one step
template <class E, int V> __device__ __forceinline__ void get(const E* p, E* to) {
    if constexpr (V == 1) to[0] = p[0];
    else {
        const typename Vec<E, V>::type w = *reinterpret_cast<const typename Vec<E, V>::type*>(p);
#pragma unroll
        for (int k = 0; k < V; k++) to[k] = w[k];
    }
}
template <class E, int V> __device__ __forceinline__ void put(E* p, const E* from) {
    if constexpr (V == 1) p[0] = from[0];
    else {
        typename Vec<E, V>::type w;
#pragma unroll
        for (int k = 0; k < V; k++) w[k] = from[k];
        *reinterpret_cast<typename Vec<E, V>::type*>(p) = w;
    }
}

// COLUMNS: E[from .. from + count) of the V columns at p, `fill` outside [lo, hi)
template <class E, int V, int COUNT>
__device__ __forceinline__ void get_steps(const void* base, int64_t st, int64_t from, int64_t lo, int64_t hi, E fill, E* to) {
    const E* p = (const E*)base + from * st;
    if (from >= lo && from + COUNT <= hi) {
#pragma unroll
        for (int i = 0; i < COUNT; i++) get<E, V>(p + i * st, to + i * V);
    } else {
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
#pragma unroll
            for (int k = 0; k < V; k++) to[i * V + k] = fill;
            if (from + i >= lo && from + i < hi) get<E, V>(p + i * st, to + i * V);
        }
    }
}

// RUNS: the same of one column whose steps are adjacent (either way round): 16 bytes at a time
template <class E, int COUNT>
__device__ __forceinline__ void get_run(const void* base, int64_t st, int64_t from, int64_t lo, int64_t hi, E fill, E* to) {
    constexpr int VN = 16 / sizeof(E) < COUNT ? 16 / sizeof(E) : COUNT;
    if (COUNT % VN == 0 && from >= lo && from + COUNT <= hi && (st == 1 || st == -1)) {
        const E* p = (const E*)base + (st == 1 ? from : -(from + COUNT - 1));
#pragma unroll
        for (int j = 0; j < COUNT; j += VN) {
            const typename Vec<E, VN>::type w = *reinterpret_cast<const typename Vec<E, VN>::type*>(p + j);
#pragma unroll
            for (int k = 0; k < VN; k++) to[j + k] = w[k];
        }
        if (st == -1) {
#pragma unroll
            for (int j = 0; j < COUNT / 2; j++) { const E t = to[j]; to[j] = to[COUNT - 1 - j]; to[COUNT - 1 - j] = t; }
        }
    } else get_steps<E, 1, COUNT>(base, st, from, lo, hi, fill, to);
}
template <class E>
__device__ __forceinline__ void put_run(void* base, int64_t st, int64_t from, int64_t hi, const E* v) {
    constexpr int VN = 16 / sizeof(E) < L ? 16 / sizeof(E) : L;
    if (from + L <= hi && (st == 1 || st == -1)) {
        E* p = (E*)base + (st == 1 ? from : -(from + L - 1));
#pragma unroll
        for (int j = 0; j < L; j += VN) {
            typename Vec<E, VN>::type w;
#pragma unroll
            for (int k = 0; k < VN; k++) w[k] = st == 1 ? v[j + k] : v[L - 1 - j - k];
            *reinterpret_cast<typename Vec<E, VN>::type*>(p + j) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < L; i++)
            if (from + i < hi) ((E*)base)[(from + i) * st] = v[i];
    }
}

// A lane's V columns: where they start in every view.
struct Base {
    const void *x, *gate, *before;
    const uint8_t* resets;
    int64_t second;                    // flags of the second column
    void *h, *gate_out;
};
template <class E> __device__ __forceinline__ const void* column(const View& v, int64_t b, int64_t c) { return v.p ? (const void*)((const E*)v.p + b * v.sb + c * v.sc) : nullptr; }

template <Kind K, class T> __device__ __forceinline__ Base base_of(const Seq& S, int64_t q) {
    int64_t b, c;
    if ((uint64_t)S.cols <= 0xffffffffu) { b = (uint32_t)q / (uint32_t)S.channels; c = (uint32_t)q - (uint32_t)b * (uint32_t)S.channels; }
    else { b = q / S.channels; c = q - b * S.channels; }
    using O = std::conditional_t<K == ADVANTAGES, float, T>;
    return Base{column<T>(S.x, b, c), column<T>(S.gate, b, c), column<O>(S.before, b, c), (const uint8_t*)column<uint8_t>(S.resets, b, 0),
                S.channels == 1 ? S.resets.sb : 0, (void*)column<O>(S.h, b, c), (void*)column<O>(S.gate_out, b, c)};
}

template <Kind K, class T, int V, bool RUNS, bool APPLYING>
__device__ __forceinline__ void load(const Seq& S, const Base& B, int64_t q, int64_t u0, int64_t end, Run<K, T, V>& d) {
    constexpr int N = L * V;
    auto steps = [&](auto fill, auto count, const void* base, int64_t st, int64_t from, int64_t lo, int64_t hi, auto* to) {
        using E = decltype(fill);
        if constexpr (RUNS) get_run<E, decltype(count)::value>(base, st, from, lo, hi, fill, to);
        else get_steps<E, V, decltype(count)::value>(base, st, from, lo, hi, fill, to);
    };
    constexpr auto run = std::integral_constant<int, L>{};
    constexpr int64_t shift = K == BACKWARD ? 1 : 0;
    if (K == BACKWARD && !B.x) {
#pragma unroll
        for (int i = 0; i < N; i++) d.x[i] = T(0);
    } else steps(T(0), run, B.x, S.x.st, u0, 0, end, d.x);
    if constexpr (K != ADVANTAGES) {
        if (B.gate) {
            // behind the end: a coefficient of 1, so that a run that is cut short has the pair of what it holds
            steps(T(1), run, B.gate, S.gate.st, u0 - shift, 0, end - shift, d.g);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) d.g[i] = (T)S.gate_const;
        }
    }
    // flags, a byte each
    constexpr int COUNT = K == BACKWARD ? L + 1 : L;
    if (B.resets) {
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            const int64_t u = u0 - shift + i;
            const bool in = u >= 0 && u < end;
#pragma unroll
            for (int k = 0; k < V; k++) d.r[i * V + k] = in ? B.resets[u * S.resets.st + k * B.second] : 0;
        }
    } else {
#pragma unroll
        for (int i = 0; i < COUNT * V; i++) d.r[i] = 0;
    }
    if constexpr (K == ADVANTAGES) {
        steps(0.0f, run, B.before, S.before.st, u0, 0, end, d.v + V);
#pragma unroll
        for (int k = 0; k < V; k++) {
            const int64_t at = RUNS ? 0 : k;
            d.v[k] = u0 == 0 ? ((const float*)S.edge)[q + k] : u0 <= end ? ((const float*)B.before)[(u0 - 1) * S.before.st + at] : 0.0f;
        }
    }
    if constexpr (K == BACKWARD && APPLYING) {
        // (the state before the step that is last in this order is the initial one, which is not in h: see walk)
        if (B.gate_out) steps(T(0), run, B.before, S.before.st, u0 + 1, 0, S.steps, d.before);
        else {
#pragma unroll
            for (int i = 0; i < N; i++) d.before[i] = T(0);
        }
    }
}

// What lies outside the sequence: no coefficient in front of the first step of the backward pass but 1, and a constant gate
// does not act behind the end.
template <Kind K, class T, int V>
__device__ __forceinline__ typename State<T>::type coefficient(const Seq& S, const Run<K, T, V>& d, int64_t u, int64_t end, int i, int k) {
    using W = typename State<T>::type;
    if (u + i >= end) return W(1);
    if constexpr (K == BACKWARD)
        if (u + i == 0) return W(1);
    if constexpr (K != ADVANTAGES)
        if (!S.gate.p) return d.r[i * V + k] ? W(0) : (W)S.gate_const;
    return d.coefficient(S, i, k);
}

template <Kind K, class T, int V>
__device__ __forceinline__ Pair<typename State<T>::type> pair_of(const Seq& S, const Run<K, T, V>& d, int64_t u0, int64_t end, int k) {
    using W = typename State<T>::type;
    Pair<W> p{W(1), W(0)};
#pragma unroll
    for (int i = 0; i < L; i++) p.then(coefficient<K, T, V>(S, d, u0, end, i, k), u0 + i < end ? d.addend(S, i, k) : W(0));
    return p;
}

// Walks the run from the state in front of it and writes.
template <Kind K, class T, int V, bool RUNS>
__device__ __forceinline__ void walk(const Seq& S, const Base& B, int64_t q, const Run<K, T, V>& d, int64_t u0, int64_t end, typename State<T>::type (&h)[V]) {
    using W = typename State<T>::type;
    using O = std::conditional_t<K == ADVANTAGES, float, T>;
    O out[L * V], second[K == SCAN ? 1 : L * V];
#pragma unroll
    for (int i = 0; i < L; i++) {
#pragma unroll
        for (int k = 0; k < V; k++) {
            const bool in = u0 + i < end;
            const W a = coefficient<K, T, V>(S, d, u0, end, i, k);
            h[k] = step(a, h[k], in ? d.addend(S, i, k) : W(0));
            out[i * V + k] = (O)h[k];
            if constexpr (K == BACKWARD) {
                W prev = (W)d.before[i * V + k];
                if (u0 + i + 1 == S.steps) prev = S.edge ? ((const W*)S.edge)[q + k] : W(0);
                second[i * V + k] = (O)(d.r[(i + 1) * V + k] ? W(0) : h[k] * prev);
            }
            if constexpr (K == ADVANTAGES) second[i * V + k] = (O)(h[k] + (W)d.v[(i + 1) * V + k]);
            if (S.final && u0 + i + 1 == S.steps) {
                W f = h[k];
                if constexpr (K == BACKWARD) {         // through the coefficient of the step itself
                    const W own = d.r[(i + 1) * V + k] ? W(0) : B.gate ? (W)((const T*)B.gate)[(S.steps - 1) * S.gate.st + k] : (W)S.gate_const;
                    f = own == W(0) ? W(0) : own * h[k];
                }
                ((W*)S.final)[q + k] = f;
            }
        }
    }
    auto write = [&](void* base, int64_t st, const O* v) {
        if (!base) return;
        if constexpr (RUNS) put_run<O>(base, st, u0, end, v);
        else {
            O* p = (O*)base + u0 * st;
#pragma unroll
            for (int i = 0; i < L; i++)
                if (u0 + i < end) put<O, V>(p + i * st, v + i * V);
        }
    };
    write(B.h, S.h.st, out);
    if constexpr (K != SCAN) write(B.gate_out, S.gate_out.st, second);
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

// ---- COLUMNS: 64 V columns to a wavefront, WT wavefronts of a workgroup one behind the other in time -----------------------

template <Kind K, class T, int V, int WT, Phase P>
__global__ __launch_bounds__(WT == 1 ? 256 : 64 * WT) void columns_kernel(Seq S) {
    using W = typename State<T>::type;
    constexpr int WC = WT == 1 ? 4 : 1;               // tiles of columns to a workgroup
    __shared__ W pa[2][WT > 1 ? WT : 1][WT > 1 ? 64 * V : 1], ph[2][WT > 1 ? WT : 1][WT > 1 ? 64 * V : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wt = WT > 1 ? wave : 0;
    int64_t q = ((int64_t)blockIdx.x * WC + (WT > 1 ? 0 : wave)) * 64 * V + lane * V;
    const bool there = q < S.cols;
    if (!there) q = 0;                                // (goes along to the barriers, reads column 0, writes nothing)
    const int64_t part = P == WHOLE ? 0 : blockIdx.y;
    const int64_t begin = part * S.part, end = P == WHOLE ? S.steps : min(begin + S.part, S.steps);
    const Base B = base_of<K, T>(S, q);
    W carry[V];
    Pair<W> all[V];
#pragma unroll
    for (int k = 0; k < V; k++) {
        carry[k] = first_state<K, W>(S, q + k);
        all[k] = Pair<W>{W(1), W(0)};
    }
    if constexpr (P == APPLY) {
        // what came before this part: a wavefront joins its share of the parts, the workgroup the wavefronts'
        const int64_t share = (part + WT - 1) / WT, from = min(wt * share, part), to = min(from + share, part);
#pragma unroll
        for (int k = 0; k < V; k++) {
            const Pair<W> p = joined_parts<W>(S, from, to, q + k);
            pa[1][wt][lane * V + k] = p.a;
            ph[1][wt][lane * V + k] = p.h;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < V; k++)
#pragma unroll
            for (int w = 0; w < WT; w++) carry[k] = step(pa[1][w][lane * V + k], carry[k], ph[1][w][lane * V + k]);
    }
    if (P != PAIRS && S.steps == 0 && S.final && there && wt == 0) {
#pragma unroll
        for (int k = 0; k < V; k++) ((W*)S.final)[q + k] = carry[k];
    }
    Run<K, T, V> next;
    load<K, T, V, false, P != PAIRS>(S, B, q, begin + wt * L, end, next);
    int turn = 0;
    for (int64_t u = begin; u < end; u += WT * L, turn ^= 1) {
        const int64_t u0 = u + wt * L;
        const Run<K, T, V> d = next;
        if (u + WT * L < end) load<K, T, V, false, P != PAIRS>(S, B, q, u0 + WT * L, end, next);
        W mine[V];
        if constexpr (WT > 1) {
            Pair<W> p[V];
#pragma unroll
            for (int k = 0; k < V; k++) {
                p[k] = pair_of<K, T, V>(S, d, u0, end, k);
                pa[turn][wt][lane * V + k] = p[k].a;
                ph[turn][wt][lane * V + k] = p[k].h;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < V; k++) {
                if constexpr (P == PAIRS) {
                    if (wt == 0) {
#pragma unroll
                        for (int w = 0; w < WT; w++) {
                            Pair<W> o{pa[turn][w][lane * V + k], ph[turn][w][lane * V + k]};
                            o.after(all[k]);
                            all[k] = o;
                        }
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < WT; w++) {
                        if (w == wt) mine[k] = carry[k];
                        carry[k] = step(pa[turn][w][lane * V + k], carry[k], ph[turn][w][lane * V + k]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < V; k++) {
                if constexpr (P == PAIRS) {
                    Pair<W> o = pair_of<K, T, V>(S, d, u0, end, k);
                    o.after(all[k]);
                    all[k] = o;
                } else mine[k] = carry[k];
            }
        }
        if constexpr (P != PAIRS) {
            if (there && u0 < end) walk<K, T, V, false>(S, B, q, d, u0, end, mine);
            if constexpr (WT == 1) {
#pragma unroll
                for (int k = 0; k < V; k++) carry[k] = mine[k];
            }
        }
    }
    if (P == PAIRS && there && wt == 0) {
        W* pairs = (W*)S.pairs + 2 * part * S.cols + q;
#pragma unroll
        for (int k = 0; k < V; k++) { pairs[k] = all[k].a; pairs[S.cols + k] = all[k].h; }
    }
}

// ---- RUNS: 64 runs of one column to a wavefront, WT wavefronts to a column -----------------------------------------------

template <class W> __device__ __forceinline__ Pair<W> up(const Pair<W>& p, int by) { return Pair<W>{__shfl_up(p.a, by), __shfl_up(p.h, by)}; }

template <Kind K, class T, int WT, Phase P>
__global__ __launch_bounds__(WT == 1 ? 256 : 64 * WT) void runs_kernel(Seq S) {
    using W = typename State<T>::type;
    __shared__ W pa[2][WT], ph[2][WT];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wt = WT > 1 ? wave : 0;
    const int64_t q = WT > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    if (q >= S.cols) return;                          // WT > 1: a whole workgroup, else a whole wavefront and no barrier
    const int64_t part = P == WHOLE ? 0 : blockIdx.y;
    const int64_t begin = part * S.part, end = P == WHOLE ? S.steps : min(begin + S.part, S.steps);
    const Base B = base_of<K, T>(S, q);
    W carry = first_state<K, W>(S, q);
    if constexpr (P == APPLY) {
        const int64_t share = (part + WT * 64 - 1) / (WT * 64), from = min((wt * 64 + lane) * share, part), to = min(from + share, part);
        Pair<W> p = joined_parts<W>(S, from, to, q);
#pragma unroll
        for (int by = 1; by < 64; by <<= 1) {
            const Pair<W> o = up(p, by);
            if (lane >= by) p.after(o);
        }
        if (lane == 63) { pa[1][wt] = p.a; ph[1][wt] = p.h; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WT; w++) carry = step(pa[1][w], carry, ph[1][w]);
    }
    if (P != PAIRS && S.steps == 0 && S.final && wt == 0 && lane == 0) ((W*)S.final)[q] = carry;
    Pair<W> all{W(1), W(0)};
    const int64_t mine = (int64_t)(wt * 64 + lane) * L;
    Run<K, T, 1> next;
    load<K, T, 1, true, P != PAIRS>(S, B, q, begin + mine, end, next);
    int turn = 0;
    for (int64_t u = begin; u < end; u += WT * 64 * L, turn ^= 1) {
        const int64_t u0 = u + mine;
        const Run<K, T, 1> d = next;
        if (u + WT * 64 * L < end) load<K, T, 1, true, P != PAIRS>(S, B, q, u0 + WT * 64 * L, end, next);
        Pair<W> p = pair_of<K, T, 1>(S, d, u0, end, 0);
#pragma unroll
        for (int by = 1; by < 64; by <<= 1) {
            const Pair<W> o = up(p, by);
            if (lane >= by) p.after(o);
        }
        Pair<W> front = up(p, 1);                     // of the lanes before this one
        if (lane == 0) front = Pair<W>{W(1), W(0)};
        Pair<W> whole{__shfl(p.a, 63), __shfl(p.h, 63)};
        if constexpr (WT > 1) {
            if (lane == 0) { pa[turn][wt] = whole.a; ph[turn][wt] = whole.h; }
            __syncthreads();
            Pair<W> before{W(1), W(0)}, total{W(1), W(0)};
#pragma unroll
            for (int w = 0; w < WT; w++) {
                if (w == wt) before = total;
                Pair<W> o{pa[turn][w], ph[turn][w]};
                o.after(total);
                total = o;
            }
            front.after(before);
            whole = total;
        }
        if constexpr (P == PAIRS) {
            whole.after(all);
            all = whole;
        } else {
            W h[1] = {step(front.a, carry, front.h)};
            carry = step(whole.a, carry, whole.h);
            if (u0 < end) walk<K, T, 1, true>(S, B, q, d, u0, end, h);
        }
    }
    if (P == PAIRS && wt == 0 && lane == 0) {
        W* pairs = (W*)S.pairs + 2 * part * S.cols + q;
        pairs[0] = all.a;
        pairs[S.cols] = all.h;
    }
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

template <Kind K, class T, int V, int WT> void launch_columns(Seq& S, const Deal& d, hipStream_t stream) {
    const int64_t tiles = cdiv(cdiv(S.cols, 64 * V), WT == 1 ? 4 : 1);
    const int threads = WT == 1 ? 256 : 64 * WT;
    if (d.parts > 1) {
        if constexpr (WT == 16) {
            columns_kernel<K, T, V, WT, PAIRS><<<dim3((unsigned)tiles, (unsigned)d.parts), threads, 0, stream>>>(S);
            columns_kernel<K, T, V, WT, APPLY><<<dim3((unsigned)tiles, (unsigned)d.parts), threads, 0, stream>>>(S);
        }
    } else columns_kernel<K, T, V, WT, WHOLE><<<(unsigned)tiles, threads, 0, stream>>>(S);
}
template <Kind K, class T, int WT> void launch_runs(Seq& S, const Deal& d, hipStream_t stream) {
    const int64_t blocks = WT == 1 ? cdiv(S.cols, 4) : S.cols;
    const int threads = WT == 1 ? 256 : 64 * WT;
    if (d.parts > 1) {
        if constexpr (WT == 16) {
            runs_kernel<K, T, WT, PAIRS><<<dim3((unsigned)blocks, (unsigned)d.parts), threads, 0, stream>>>(S);
            runs_kernel<K, T, WT, APPLY><<<dim3((unsigned)blocks, (unsigned)d.parts), threads, 0, stream>>>(S);
        }
    } else runs_kernel<K, T, WT, WHOLE><<<(unsigned)blocks, threads, 0, stream>>>(S);
}

bool dense(const View& v, int64_t channels) { return !v.p || (channels == 1 ? v.sb : v.sc) == 1; }

template <Kind K, class T> int launch(Seq S, void* workspace, int64_t bytes, hipStream_t stream, const char* who) {
    // time is the fast index of what is read
    const View& main = S.x.p ? S.x : S.h;
    const bool runs = S.channels == 1 && S.steps > 1 && (main.st == 1 || main.st == -1) && (main.sb != 1 || S.cols == 1);
    const Deal d = runs ? deal_runs(S.steps, S.cols) : deal_columns(S.steps, S.cols);
    if (d.parts > 65535 || S.cols > ((int64_t)1 << 32)) return fail(-1, "%s: %lld steps of %lld columns are too many for one call", who, (long long)S.steps, (long long)S.cols);
    S.part = d.part;
    S.pairs = workspace;
    if (runs) {
        if (d.wt == 1) launch_runs<K, T, 1>(S, d, stream);
        else if (d.wt == 4) launch_runs<K, T, 4>(S, d, stream);
        else launch_runs<K, T, 16>(S, d, stream);
    } else {
        // Two columns to a lane (wider rows, half the instructions) where there are enough for the GPU all the same.
        const bool two = S.cols >= 65536 && S.cols % 2 == 0 && (S.channels == 1 || S.channels % 2 == 0) && dense(S.x, S.channels) &&
                         dense(S.gate, S.channels) && dense(S.before, S.channels) && dense(S.h, S.channels) && dense(S.gate_out, S.channels);
        if (two) {
            if (d.wt == 1) launch_columns<K, T, 2, 1>(S, d, stream);
            else launch_columns<K, T, 2, 4>(S, Deal{4, S.steps, 1}, stream);
        } else if (d.wt == 1) launch_columns<K, T, 1, 1>(S, d, stream);
        else if (d.wt == 4) launch_columns<K, T, 1, 4>(S, d, stream);
        else launch_columns<K, T, 1, 16>(S, d, stream);
    }
    LRN_LAUNCHED(who);
    return 0;
}

template <Kind K> int run(const Seq& S, int dtype, void* workspace, int64_t bytes, hipStream_t stream, const char* who) {
    if (dtype == LRN_F32) return launch<K, float>(S, workspace, bytes, stream, who);
    if (dtype == LRN_F64) return launch<K, double>(S, workspace, bytes, stream, who);
    if constexpr (K != ADVANTAGES) {
        if (dtype == LRN_BF16) return launch<K, bf16>(S, workspace, bytes, stream, who);
        return launch<K, f16>(S, workspace, bytes, stream, who);
    }
    return 0;
}

int check_workspace(const lrn_seq* q, const void* workspace, int64_t bytes, const char* who) {
    const int64_t need = pair_bytes(q);
    if (need && (!workspace || bytes < need)) return fail(-1, "%s: a workspace of %lld bytes is needed, got %lld", who, (long long)need, (long long)bytes);
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
    if (int rc = checked(seq, "lrn_scan")) return rc;
    if (seq->batch * seq->channels == 0) return 0;
    if (seq->steps && (!x || !x->data || !h_out || !h_out->data)) return fail(-1, "lrn_scan: null x or h");
    if (int rc = check_workspace(seq, workspace, workspace_bytes, "lrn_scan")) return rc;
    LRN_ON_DEVICE(device);
    const bool rev = seq->reverse != 0;
    const int64_t n = bytes_of(seq->dtype);
    Seq S{};
    S.steps = seq->steps; S.cols = seq->batch * seq->channels; S.channels = seq->channels;
    S.x = ordered(x, seq->steps, n, rev); S.gate = ordered(gate, seq->steps, n, rev);
    S.resets = ordered(resets, seq->steps, 1, rev); S.h = ordered(h_out, seq->steps, n, rev);
    S.gate_const = gate_const; S.initial = initial; S.final = final_out;
    return run<SCAN>(S, seq->dtype, workspace, workspace_bytes, (hipStream_t)hip_stream, "lrn_scan");
}

int lrn_scan_backward(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* gate, double gate_const,
                      const lrn_view* resets, const void* initial, const lrn_view* h, const lrn_view* g_h,
                      const void* g_final, const lrn_view* grad_x_out, const lrn_view* grad_gate_out,
                      void* grad_initial_out, void* workspace, int64_t workspace_bytes) {
    if (int rc = checked(seq, "lrn_scan_backward")) return rc;
    if (seq->batch * seq->channels == 0) return 0;
    if (grad_gate_out && grad_gate_out->data && seq->steps && (!h || !h->data)) return fail(-1, "lrn_scan_backward: null h");
    if (int rc = check_workspace(seq, workspace, workspace_bytes, "lrn_scan_backward")) return rc;
    LRN_ON_DEVICE(device);
    const bool rev = seq->reverse == 0;
    const int64_t n = bytes_of(seq->dtype);
    Seq S{};
    S.steps = seq->steps; S.cols = seq->batch * seq->channels; S.channels = seq->channels;
    S.x = ordered(g_h, seq->steps, n, rev); S.gate = ordered(gate, seq->steps, n, rev);
    S.resets = ordered(resets, seq->steps, 1, rev); S.before = ordered(h, seq->steps, n, rev);
    S.h = ordered(grad_x_out, seq->steps, n, rev); S.gate_out = ordered(grad_gate_out, seq->steps, n, rev);
    S.gate_const = gate_const; S.initial = g_final; S.edge = initial; S.final = grad_initial_out;
    return run<BACKWARD>(S, seq->dtype, workspace, workspace_bytes, (hipStream_t)hip_stream, "lrn_scan_backward");
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
    if (int rc = check_workspace(seq, workspace, workspace_bytes, "lrn_advantages")) return rc;
    LRN_ON_DEVICE(device);
    Seq S{};
    S.steps = seq->steps; S.cols = seq->batch; S.channels = 1;
    S.x = ordered(rewards, seq->steps, bytes_of(seq->dtype), true); S.before = ordered(values, seq->steps, 4, true);
    S.resets = ordered(ends, seq->steps, 1, true);
    S.h = ordered(advantage_out, seq->steps, 4, true); S.gate_out = ordered(target_out, seq->steps, 4, true);
    S.gate_const = gamma * lam; S.scale = gamma; S.edge = last_values;
    return run<ADVANTAGES>(S, seq->dtype, workspace, workspace_bytes, (hipStream_t)hip_stream, "lrn_advantages");
}

}  // extern "C"
