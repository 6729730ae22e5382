// learner_rows.hip — gfx950 kernels of lrn_choose / lrn_score / lrn_score_backward (include/learner_ops.h).
//
// One pass over a row with the running maximum m, s = sum exp(z - m) and t = sum exp(z - m) (z - m): when the maximum moves
// from m to m', c = exp(m - m') rescales s' = c s and t' = c (t + s (m - m')).  log s and t / s are all that the log
// probability and the entropy need.  Sums are float32 whatever the logits' type.
#include <algorithm>
#include <type_traits>

#include "lrn_common.h"
#include "lrn_grid.h"

namespace lrn {

char* error_text() {
    static thread_local char text[512] = "";
    return text;
}

namespace {

__device__ __forceinline__ int64_t block_number() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

struct Rows {
    const void* logits;
    const uint8_t* mask;
    int64_t rows, inner;
    int64_t so, si, mo, mi;
    int32_t levels, mask_level;
    int64_t limit, mask_limit;   // elements from the first of any row to behind the last of any
    bool dense, mask_dense;      // row r starts at r * levels
};

struct Sums {
    float m, s, t;
    __device__ __forceinline__ void clear() { m = kNegInf; s = 0.0f; t = 0.0f; }
    // A part without an allowed logit has s = 0 and says nothing; NaN stays NaN.
    __device__ __forceinline__ void join(const Sums& o) {
        if (o.s == 0.0f) return;
        if (s == 0.0f) { *this = o; return; }
        const float top = fmaxf(m, o.m), da = m - top, db = o.m - top;
        const float ca = fast_exp(da), cb = fast_exp(db);
        t = (ca > 0.0f ? ca * (t + s * da) : 0.0f) + (cb > 0.0f ? cb * (o.t + o.s * db) : 0.0f);
        s = ca * s + cb * o.s;
        m = top;
    }
};

struct Best {
    float v;
    int j;
    __device__ __forceinline__ void clear() { v = kNegInf; j = 0x7fffffff; }
    __device__ __forceinline__ void add(float x, int i) { if (x > v || (x == v && i < j)) { v = x; j = i; } }
};

// A level's place in the choice.  Noise of -inf (the logarithm of a logarithm of a uniform 0) and NaN puts an allowed level last,
// not out: the only one left is chosen all the same.
__device__ __forceinline__ float choice_key(float z, float noise) { return fmaxf(z + noise, -3.4028234e38f); }

__device__ __forceinline__ float lane_of(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// The 64 best of what a wavefront has seen, lane i the i-th (falling, the lowest index first among equals).  Candidates go in
// one at a time: k (1 + log(n / k)) of n values do.  What an insertion costs is latency, so nothing in it goes through LDS: the
// candidate and the bound are scalars (v_readlane), the entries behind it move up by one lane with a whole-wavefront shift
// (exchanges through LDS instead: 45 us for what takes 32, both without the floor).
struct TopList {
    float v;
    int j;
    float floor;                 // `top` values of at least this are known to come
    float bound;                 // what a candidate has to be ahead of: the top-th entry, or the floor until there is one
    int bound_j;
    __device__ __forceinline__ void clear(float at_least = kNegInf) { v = kNegInf; bound = floor = at_least; j = bound_j = 0x7fffffff; }
    // every lane offers one candidate (-inf: none)
    __device__ __forceinline__ void offer(float x, int i, int top, int lane) {
        for (;;) {
            const unsigned long long some = __ballot(x > bound || (x == bound && x > kNegInf && i < bound_j));
            if (!some) return;
            const int src = __ffsll((long long)some) - 1;
            const float cv = lane_of(x, src);
            const int cj = lane_of(i, src);
            const int at = __popcll(__ballot(v > cv || (v == cv && j < cj)));
            const float pv = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x138, 0xf, 0xf, true));
            const int pj = __builtin_amdgcn_update_dpp(0, j, 0x138, 0xf, 0xf, true);
            v = lane > at ? pv : lane == at ? cv : v;
            j = lane > at ? pj : lane == at ? cj : j;
            const float last = lane_of(v, top - 1);
            if (last >= floor) { bound = last; bound_j = lane_of(j, top - 1); }
            if (lane == src) x = kNegInf;
        }
    }
};

// The `count`-th largest of 256 values (four a lane) by halving the ordered bit patterns.
__device__ __forceinline__ float nth_of_256(const float (&v)[4], int count) {
    uint32_t key[4], at = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v[k]);
        key[k] = u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
    }
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
        const uint32_t t = at | bit;
        int n = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) n += __popcll(__ballot(key[k] >= t));
        if (n >= count) at = t;
    }
    return __builtin_bit_cast(float, at & 0x80000000u ? at ^ 0x80000000u : ~at);
}

// row r = (o, i)
__device__ __forceinline__ void split(const Rows& R, int64_t r, int64_t& o, int64_t& i) {
    if ((uint64_t)R.rows <= 0xffffffffu) { o = (uint32_t)r / (uint32_t)R.inner; i = (uint32_t)r - (uint32_t)o * (uint32_t)R.inner; }
    else { o = r / R.inner; i = r - o * R.inner; }
}
__device__ __forceinline__ int64_t row_base(const Rows& R, int64_t r) { int64_t o, i; split(R, r, o, i); return o * R.so + i * R.si; }
__device__ __forceinline__ const uint8_t* row_mask(const Rows& R, int64_t r) {
    if (!R.mask) return nullptr;
    int64_t o, i;
    split(R, r, o, i);
    return R.mask + o * R.mo + i * R.mi;
}

// +inf among the allowed logits: no distribution
__device__ __forceinline__ void finish(Sums& a) { if (a.m == -kNegInf) a.s = __builtin_nanf(""); }
__device__ __forceinline__ float entropy_of(const Sums& a, float logs) { return a.s != 0.0f ? logs - a.t * fast_inverse(a.s) : 0.0f; }

struct ChooseOut { const float* noise; int64_t no, ni, limit; bool dense; int64_t* level; float* logprob; float* entropy; };

// Where row r starts in the logits, the mask and the noise.
__device__ __forceinline__ void offsets(const Rows& R, int64_t r, int64_t& off, int64_t& moff, const ChooseOut* O = nullptr, int64_t* noff = nullptr) {
    off = moff = r * R.levels;
    if (O) *noff = off;
    if (R.dense && (!R.mask || R.mask_dense) && (!O || O->dense)) return;
    int64_t o, i;
    split(R, r, o, i);
    off = o * R.so + i * R.si;
    moff = o * R.mo + i * R.mi;
    if (O) *noff = o * O->no + i * O->ni;
}

struct ScoreOut { const int64_t* level; float* logprob; float* entropy; float* stat; int top; float* top_logprob; int64_t* top_level; };

struct BackIn { const int64_t* level; const float* stat; const float* entropy; const float* g_lp; const float* g_h; int g_lp_stride, g_h_stride; };

// ---- rows of up to 1024 levels: G lanes to a row, E adjacent levels to a lane --------------------------------------------
//
// A lane takes its levels with one or two vector loads (at any alignment; what they read beyond the row belongs to the next
// one and is dropped, and only where there is no next one do single loads take over), so no index is computed per level and
// rows at any stride go the same way.  Rows of up to eight levels have their length compiled in.  The maximum comes first and
// every weight is computed once; the group's sums go through DPP.  The backward pass computes the row's maximum and sums again
// from the logits that it has to read anyway: cheaper than 12 bytes a row of saved statistics.  Its results meet in LDS, from
// where they leave as one run of 16-byte stores.
//
// Bound by memory where rows are short and float32 (65 536 x 54 x 5: 127 MB in 28 us = 4.5 TB/s of a large copy's 5.1, backward
// 198 MB in 33); of two bytes a level, by trips to memory behind one another (logits, mask, then the level's own: 110 MB in 31.5
// with a mask, backward 145 MB in 31.8); longer rows of two bytes a level by the issue of some 25 instructions a level (16 000 x
// 1000 bfloat16: 13.6 us forward, 19.8 backward).  An earlier form that brought all rows through LDS, with a division of every
// element's index, took 16 and 30 for the last.

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int CTRL> __device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true); }

// f(v) for the partner lanes: neighbours, pairs, quads and half rows of 16 by DPP (each step's partner holds the other half's
// result, mirrored where the hardware has no exchange), 16 and 32 lanes apart by a lane exchange.
template <int G, class F> __device__ __forceinline__ void over_group(F&& f) {
    if constexpr (G >= 2) f([](auto v) { return dpp<0xB1>(v); });
    if constexpr (G >= 4) f([](auto v) { return dpp<0x4E>(v); });
    if constexpr (G >= 8) f([](auto v) { return dpp<0x141>(v); });
    if constexpr (G >= 16) f([](auto v) { return dpp<0x140>(v); });
    if constexpr (G >= 32) f([](auto v) { return __shfl_xor(v, 16); });
    if constexpr (G >= 64) f([](auto v) { return __shfl_xor(v, 32); });
}

template <class V, int N> __device__ __forceinline__ void take(const V* p, V (&to)[N]) { __builtin_memcpy(to, p, sizeof(to)); }

// A workgroup's rows of up to eight 16-bit logits, and their mask, through LDS: at 2 to 16 bytes a row a lane's own loads are
// many, small and askew, the run of them is a few 16-byte loads (65 536 x 54 rows of five bfloat16 with a mask, 110 MB: 30.6 us
// instead of 32.6).
template <class T, int G, int E> constexpr bool kStaged = G == 1 && sizeof(T) == 2;
template <class T, int E> struct Stage {
    __attribute__((aligned(16))) T z[256 * E];
    __attribute__((aligned(16))) uint8_t mask[256 * E];
};
template <class T, int G, int E> using StageOf = std::conditional_t<kStaged<T, G, E>, Stage<T, E>, char>;

__device__ __forceinline__ void copy_run(const void* from, void* to, int bytes) {
    typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(1)));
    for (int at = threadIdx.x * 16; at < bytes; at += 256 * 16) {
        if (at + 16 <= bytes) *reinterpret_cast<uint4*>((char*)to + at) = __builtin_bit_cast(uint4, (vec)*reinterpret_cast<const vec*>((const char*)from + at));
        else
            for (int k = at; k < bytes; k++) ((char*)to)[k] = ((const char*)from)[k];
    }
}
template <class T, int G, int E> __device__ __forceinline__ void stage(const Rows& R, int64_t r0, int here, StageOf<T, G, E>& S) {
    if constexpr (kStaged<T, G, E>) {
        const int n = here * E;
        if (R.dense) copy_run((const T*)R.logits + r0 * E, S.z, n * 2);
        if (R.mask && R.mask_dense) copy_run(R.mask + r0 * E, S.mask, n);
        __syncthreads();
    }
}

// Lane g's levels g E .. of row r: -inf where masked or behind the row.
template <class T, int G, int E>
__device__ __forceinline__ void load_levels(const Rows& R, const StageOf<T, G, E>& S, int64_t off, int64_t moff, int g, float (&z)[E]) {
    const int j0 = g * E, valid = R.levels - j0;
    T v[E];
    uint8_t b[E];
    const T* src = (const T*)R.logits + off + j0;
    bool here = false, mask_here = false;
    if constexpr (kStaged<T, G, E>) {
        here = R.dense;
        mask_here = R.mask && R.mask_dense;
        if (here) {
#pragma unroll
            for (int k = 0; k < E; k++) v[k] = S.z[threadIdx.x * E + k];
        }
        if (mask_here) {
#pragma unroll
            for (int k = 0; k < E; k++) b[k] = S.mask[threadIdx.x * E + k];
        }
    }
    if (!here && valid > 0) {
        if (off + j0 + E <= R.limit) take(src, v);
        else {
#pragma unroll
            for (int k = 0; k < E; k++)
                if (k < valid) v[k] = src[k];
        }
    }
    if (R.mask) {
        const uint8_t* mk = R.mask + moff;
        if (mask_here) {
        } else if (!R.mask_level) {
            const uint8_t on = mk[0];
#pragma unroll
            for (int k = 0; k < E; k++) b[k] = on;
        } else if (valid > 0) {
            if (moff + j0 + E <= R.mask_limit) take(mk + j0, b);
            else {
#pragma unroll
                for (int k = 0; k < E; k++)
                    if (k < valid) b[k] = mk[j0 + k];
            }
        }
#pragma unroll
        for (int k = 0; k < E; k++) z[k] = k < valid && b[k] ? to_f32(v[k]) : kNegInf;
    } else {
#pragma unroll
        for (int k = 0; k < E; k++) z[k] = k < valid ? to_f32(v[k]) : kNegInf;
    }
}

// The row's maximum and sums, and the weights of the lane's own levels.
template <int G, int E>
__device__ __forceinline__ Sums group_sums(const float (&z)[E], float (&e)[E]) {
    Sums a;
    a.m = z[0];
#pragma unroll
    for (int k = 1; k < E; k++) a.m = fmaxf(a.m, z[k]);
    over_group<G>([&](auto from) { a.m = fmaxf(a.m, from(a.m)); });
    const float m = a.m == kNegInf ? 0.0f : a.m;       // nothing allowed: all weights 0 (or NaN)
    a.s = a.t = 0.0f;
#pragma unroll
    for (int k = 0; k < E; k++) {
        const float d = z[k] - m;
        e[k] = fast_exp(d);
        a.s += e[k];
        a.t += e[k] * fmaxf(d, -3.0e38f);              // a masked level: 0 times a number
    }
    over_group<G>([&](auto from) { a.s += from(a.s); a.t += from(a.t); });
    finish(a);
    return a;
}

template <class T, int G, int E>
__global__ __launch_bounds__(256) void group_choose_kernel(Rows R, ChooseOut O) {
    const int g = threadIdx.x % G;
    const int64_t r0 = block_number() * (256 / G), r = r0 + threadIdx.x / G;
    const int here = rows_here(R.rows, r0, 256 / G);
    if (!here) return;                          // a whole workgroup behind the last row, before any barrier
    __shared__ StageOf<T, G, E> S;
    stage<T, G, E>(R, r0, here, S);
    if (r >= R.rows) return;                    // whole groups: no lane of a group leaves alone
    int64_t off, moff, noff;
    offsets(R, r, off, moff, &O, &noff);
    float z[E], e[E], w[E];
    load_levels<T, G, E>(R, S, off, moff, g, z);
    Best b;
    b.clear();
    if (O.noise) {
        const float* ns = O.noise + noff + g * E;
        if (noff + g * E + E <= O.limit) take(ns, w);
        else {
#pragma unroll
            for (int k = 0; k < E; k++) w[k] = g * E + k < R.levels ? ns[k] : 0.0f;
        }
    } else {
#pragma unroll
        for (int k = 0; k < E; k++) w[k] = 0.0f;
    }
    const Sums a = group_sums<G, E>(z, e);
    float chosen = 0.0f;
#pragma unroll
    for (int k = 0; k < E; k++) {
        const float key = O.noise ? choice_key(z[k], w[k]) : z[k];
        if (z[k] > kNegInf && key > b.v) { b.v = key; b.j = g * E + k; chosen = z[k]; }
    }
    over_group<G>([&](auto from) {
        const float v = from(b.v), c = from(chosen);
        const int j = from(b.j);
        if (v > b.v || (v == b.v && j < b.j)) { b.v = v; b.j = j; chosen = c; }
    });
    if (g == 0) {
        const bool some = a.s != 0.0f, found = b.j < R.levels;
        const float logs = fast_log(a.s);
        O.level[r] = some && found ? b.j : 0;
        O.logprob[r] = !some ? 0.0f : found ? chosen - a.m - logs : __builtin_nanf("");
        O.entropy[r] = entropy_of(a, logs);
    }
}

// A level in the order of alternatives: by logit, the lowest index first among equals.  16-bit logits and their index fit one
// word whose unsigned order is that order; 0: none.
template <class T> struct Key {
    uint32_t k;
    __device__ __forceinline__ void set(float z, int j) {
        const T t = (T)(z + 0.0f);                                       // (-0 is 0)
        const uint32_t u = __builtin_bit_cast(uint16_t, t);
        k = z > kNegInf ? ((u & 0x8000 ? ~u & 0xffff : u | 0x8000) << 16) | (0xffffu - j) : 0u;
    }
    __device__ __forceinline__ bool some() const { return k != 0; }
    __device__ __forceinline__ float value() const {
        const uint32_t u = k >> 16;
        return to_f32(__builtin_bit_cast(T, (uint16_t)(u & 0x8000 ? u & 0x7fff : ~u)));
    }
    __device__ __forceinline__ int level() const { return 0xffff - (int)(k & 0xffff); }
    __device__ __forceinline__ void order(Key& o) { const uint32_t hi = max(k, o.k), lo = min(k, o.k); k = hi; o.k = lo; }
    template <int G> __device__ __forceinline__ Key best() const {
        uint32_t b = k;
        over_group<G>([&](auto from) { b = max(b, (uint32_t)from((int)b)); });
        return Key{b};
    }
    __device__ __forceinline__ bool is(const Key& o) const { return k == o.k; }
};
template <> struct Key<float> {
    float v;
    int j;
    __device__ __forceinline__ void set(float z, int i) { v = z > kNegInf ? z : kNegInf; j = z > kNegInf ? i : 0x7fffffff; }
    __device__ __forceinline__ bool some() const { return v > kNegInf; }
    __device__ __forceinline__ float value() const { return v; }
    __device__ __forceinline__ int level() const { return j; }
    __device__ __forceinline__ void order(Key& o) {
        const bool swap = o.v > v || (o.v == v && o.j < j);
        const Key t = *this;
        if (swap) { *this = o; o = t; }
    }
    template <int G> __device__ __forceinline__ Key best() const {
        float b = v;
        over_group<G>([&](auto from) { b = fmaxf(b, from(b)); });
        int i = v == b ? j : 0x7fffffff;
        over_group<G>([&](auto from) { i = min(i, from(i)); });
        return Key{b, i};
    }
    __device__ __forceinline__ bool is(const Key& o) const { return j == o.j; }
};

// A merge-exchange network for N values (Batcher 1968; Knuth volume 3, 5.2.2 M).
template <int N> struct Network {
    int a[64], b[64], n;
    constexpr Network() : a(), b(), n(0) {
        int t = 0;
        while ((1 << t) < N) t++;
        for (int p = t ? 1 << (t - 1) : 0; p > 0; p >>= 1) {
            int q = 1 << (t - 1), r = 0, d = p;
            for (;;) {
                for (int i = 0; i + d < N; i++)
                    if ((i & p) == r) { a[n] = i; b[n++] = i + d; }
                if (q == p) break;
                d = q - p;
                q >>= 1;
                r = p;
            }
        }
    }
};

template <class T, int G, int E>
__global__ __launch_bounds__(256) void group_score_kernel(Rows R, ScoreOut O) {
    const int g = threadIdx.x % G;
    const int64_t r0 = block_number() * (256 / G), r = r0 + threadIdx.x / G;
    const int here = rows_here(R.rows, r0, 256 / G);
    if (!here) return;
    __shared__ StageOf<T, G, E> S;
    stage<T, G, E>(R, r0, here, S);
    if (r >= R.rows) return;
    int64_t off, moff;
    offsets(R, r, off, moff);
    const int K = R.levels;
    const int64_t l = O.level[r];
    float z[E], e[E], zl = kNegInf;
    load_levels<T, G, E>(R, S, off, moff, g, z);
    if (g == 0 && l >= 0 && l < K && !(R.mask && !R.mask[moff + l * R.mask_level])) zl = to_f32(((const T*)R.logits)[off + l]);
    const Sums a = group_sums<G, E>(z, e);
    const float logs = fast_log(a.s);
    if (g == 0) {
        O.logprob[r] = l >= K ? __builtin_nanf("") : l < 0 || a.s == 0.0f ? 0.0f : zl - a.m - logs;
        O.entropy[r] = entropy_of(a, logs);
        if (O.stat) { O.stat[2 * r] = a.m; O.stat[2 * r + 1] = a.s; }
    }
    if (!O.top) return;
    // Every lane puts its levels in order; the best of the lanes' first ones is the next alternative, O.top times.  Lane n % G
    // keeps the n-th, so that G of them leave together.
    Key<T> key[E];
#pragma unroll
    for (int k = 0; k < E; k++) key[k].set(z[k], g * E + k);
    constexpr Network<E> net;
#pragma unroll
    for (int c = 0; c < net.n; c++) key[net.a[c]].order(key[net.b[c]]);
    Key<T> kept = key[0];
    for (int n = 0; n < O.top; n++) {
        const Key<T> best = key[0].template best<G>();
        if (n % G == g) kept = best;
        if (key[0].is(best)) {
#pragma unroll
            for (int k = 0; k + 1 < E; k++) key[k] = key[k + 1];
            key[E - 1].set(kNegInf, 0);
        }
        if (n % G == G - 1 || n == O.top - 1) {
            const int at = n - n % G + g;
            if (at <= n) {
                O.top_logprob[r * O.top + at] = kept.some() ? kept.value() - a.m - logs : a.s == a.s ? kNegInf : a.s;
                O.top_level[r * O.top + at] = kept.some() ? kept.level() : -1;
            }
        }
    }
}

template <class T, int G, int E>
__global__ __launch_bounds__(256) void group_backward_kernel(Rows R, BackIn I, T* grad) {
    __shared__ __attribute__((aligned(16))) T out[256 * E];
    const int row = threadIdx.x / G, g = threadIdx.x % G, K = R.levels;
    const int64_t r0 = block_number() * (256 / G), r = r0 + row;
    const int here = rows_here(R.rows, r0, 256 / G);
    if (!here) return;
    __shared__ StageOf<T, G, E> S;
    stage<T, G, E>(R, r0, here, S);
    if (r < R.rows) {
        int64_t off, moff;
        offsets(R, r, off, moff);
        const int64_t l = I.level[r];
        const float gl = l >= K ? __builtin_nanf("") : I.g_lp && l >= 0 ? I.g_lp[r * I.g_lp_stride] : 0.0f;
        const float gh = I.g_h ? I.g_h[r * I.g_h_stride] : 0.0f;
        float z[E], e[E];
        load_levels<T, G, E>(R, S, off, moff, g, z);
        const Sums a = group_sums<G, E>(z, e);
        const float logs = fast_log(a.s), inv = fast_inverse(a.s), lift = entropy_of(a, logs) - logs, m = a.m;
        const int mine = l >= 0 && l < K ? (int)l - g * E : -1;
        T* to = out + row * K + g * E;
#pragma unroll
        for (int k = 0; k < E; k++) {
            // p (g_lp + g_h (log p + H)), log p = z - m - log s; a weight of 0 has p log p = 0
            float d = -(e[k] * inv) * (gl + gh * (e[k] > 0.0f ? z[k] - m + lift : 0.0f));
            if (k == mine) d += gl;
            if (z[k] == kNegInf) d = 0.0f;
            if (g * E + k < K) to[k] = (T)d;
        }
    }
    __syncthreads();
    constexpr int N = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    const int n = here * K;
    T* to = grad + r0 * K;
    for (int e0 = threadIdx.x * N; e0 < n; e0 += 256 * N) {
        if (e0 + N <= n) *reinterpret_cast<vec*>(to + e0) = *reinterpret_cast<const vec*>(out + e0);
        else {
#pragma unroll
            for (int k = 0; k < N; k++)
                if (e0 + k < n) to[e0 + k] = out[e0 + k];
        }
    }
}

// Up to eight levels: the row itself; then eight levels to a lane (a full set of wavefronts has the registers), or twelve where
// that takes half the lanes (33 levels: four lanes with 48 places and not eight with 64), sixteen where a row would not fit a
// wavefront otherwise.
constexpr int kGroupLevels = LRN_SHORT_ROW;
#define BY_LEVELS(K, call)                                                          \
    switch (K) {                                                                    \
        case 1: { constexpr int G = 1, E = 1; call; break; }                        \
        case 2: { constexpr int G = 1, E = 2; call; break; }                        \
        case 3: { constexpr int G = 1, E = 3; call; break; }                        \
        case 4: { constexpr int G = 1, E = 4; call; break; }                        \
        case 5: { constexpr int G = 1, E = 5; call; break; }                        \
        case 6: { constexpr int G = 1, E = 6; call; break; }                        \
        case 7: { constexpr int G = 1, E = 7; call; break; }                        \
        case 8: { constexpr int G = 1, E = 8; call; break; }                        \
        default:                                                                    \
            if ((K) <= 16) { constexpr int G = 2, E = 8; call; }                    \
            else if ((K) <= 24) { constexpr int G = 2, E = 12; call; }              \
            else if ((K) <= 32) { constexpr int G = 4, E = 8; call; }               \
            else if ((K) <= 48) { constexpr int G = 4, E = 12; call; }              \
            else if ((K) <= 64) { constexpr int G = 8, E = 8; call; }               \
            else if ((K) <= 96) { constexpr int G = 8, E = 12; call; }              \
            else if ((K) <= 128) { constexpr int G = 16, E = 8; call; }             \
            else if ((K) <= 192) { constexpr int G = 16, E = 12; call; }            \
            else if ((K) <= 256) { constexpr int G = 32, E = 8; call; }             \
            else if ((K) <= 384) { constexpr int G = 32, E = 12; call; }            \
            else if ((K) <= 512) { constexpr int G = 64, E = 8; call; }             \
            else if ((K) <= 768) { constexpr int G = 64, E = 12; call; }            \
            else { constexpr int G = 64, E = 16; call; }                            \
    }

// Alternatives by the dozen: lanes with eight levels sort and shift less (540 000 rows of 24 float32 with twenty: 60 us instead of
// 70; with three, rows of 33 in twelves are ahead).
int lanes_for(int K, int top) {
    if (top <= 4 || K <= 8) return K;
    int p = 16;
    while (p < K) p *= 2;
    return p;
}

int group_rows(int K) { int n = 256; BY_LEVELS(K, (n = 256 / G, (void)E)); return n; }

// ---- longer rows: a workgroup to a row, or to a part of one -----------------------------------------------------------
//
// Every lane walks 16-byte pieces of the row (at any alignment: the hardware takes a vector load at its element's) with a
// running maximum and sums of its own, rescaled when a piece raises the maximum; the lanes join at the end.  Where there are
// too few rows to fill the GPU a row is cut into up to 64 parts, whose sums, best level and best alternatives go through the
// workspace to a second launch, a wavefront to a row.
//
// 1024 x 32768 bfloat16: 67 MB in 18 us (3.7 TB/s), bound by instructions as much as by memory: twelve a level, four of them the
// exponential's issue.  A row in parts is bound by latency: 8 x 131 071 float32 with 20 alternatives 15 + 11 us for 4 MB (a
// wavefront to a row, as it was first, took 1070).

template <class T> struct Piece {
    static constexpr int N = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
struct Mask8 { typedef uint8_t vec __attribute__((ext_vector_type(8), aligned(1))); };
struct Mask4 { typedef uint8_t vec __attribute__((ext_vector_type(4), aligned(1))); };

// The levels e0 .. of a row into z (-inf where masked or behind `end`).
template <class T, int N = Piece<T>::N>
__device__ __forceinline__ void load_piece(const T* src, const uint8_t* mk, int mask_level, int e0, int end, float (&z)[N]) {
    if (e0 + N <= end) {
        const typename Piece<T>::vec v = *reinterpret_cast<const typename Piece<T>::vec*>(src + e0);
#pragma unroll
        for (int k = 0; k < N; k++) z[k] = to_f32(v[k]);
        if (mk && mask_level) {
            using M = std::conditional_t<N == 8, Mask8, Mask4>;
            const typename M::vec b = *reinterpret_cast<const typename M::vec*>(mk + e0);
#pragma unroll
            for (int k = 0; k < N; k++) z[k] = b[k] ? z[k] : kNegInf;
        } else if (mk) {
            const bool on = mk[0];
#pragma unroll
            for (int k = 0; k < N; k++) z[k] = on ? z[k] : kNegInf;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) z[k] = e0 + k < end && !(mk && !mk[(e0 + k) * (int64_t)mask_level]) ? to_f32(src[e0 + k]) : kNegInf;
    }
}

// f(z, e0) for every piece of a lane; kAhead pieces are asked for before the first is used.
constexpr int kAhead = 4;
template <class T, bool MASK, bool NOISE, class F>
__device__ __forceinline__ void over_pieces(const T* src, const uint8_t* mk, int mask_level, const float* ns, int begin, int end, F&& f) {
    constexpr int N = Piece<T>::N, STEP = 256 * N;
    using V = typename Piece<T>::vec;
    using M = typename std::conditional_t<N == 8, Mask8, Mask4>::vec;
    int base = begin;
    for (; base + kAhead * STEP <= end; base += kAhead * STEP) {
        const int e0 = base + (int)threadIdx.x * N;
        V v[kAhead];
        M b[kAhead];
        float w[NOISE ? kAhead : 1][N];
#pragma unroll
        for (int u = 0; u < kAhead; u++) v[u] = *reinterpret_cast<const V*>(src + e0 + u * STEP);
        if (NOISE && ns) {
#pragma unroll
            for (int u = 0; u < kAhead; u++) take(ns + e0 + u * STEP, w[NOISE ? u : 0]);
        }
        if (MASK && mask_level) {
#pragma unroll
            for (int u = 0; u < kAhead; u++) b[u] = *reinterpret_cast<const M*>(mk + e0 + u * STEP);
        } else if (MASK) {
            const uint8_t on = mk[0];
#pragma unroll
            for (int u = 0; u < kAhead; u++) b[u] = on;
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            float z[N];
#pragma unroll
            for (int k = 0; k < N; k++) z[k] = !MASK || b[u][k] ? to_f32(v[u][k]) : kNegInf;
            f(z, w[NOISE ? u : 0], e0 + u * STEP);
        }
    }
    for (; base < end; base += STEP) {
        const int e0 = base + (int)threadIdx.x * N;
        float z[N];
        float w[N];
        load_piece<T>(src, mk, mask_level, e0, end, z);
        if (NOISE && ns) {
#pragma unroll
            for (int k = 0; k < N; k++) w[k] = e0 + k < end ? ns[e0 + k] : 0.0f;
        }
        f(z, w, e0);
    }
}

template <int N> __device__ __forceinline__ void add_piece(Sums& a, const float (&z)[N]) {
    float top = z[0];
#pragma unroll
    for (int k = 1; k < N; k++) top = fmaxf(top, z[k]);
    if (top > a.m) {
        const float d = a.m - top, c = fast_exp(d);              // a.m = -inf: c = 0, and s = t = 0
        a.t = c > 0.0f ? c * (a.t + a.s * d) : 0.0f;
        a.s = c * a.s;
        a.m = top;
    }
    if (a.m == kNegInf) {                                        // nothing allowed so far, or NaN
#pragma unroll
        for (int k = 0; k < N; k++)
            if (z[k] != z[k]) a.s = z[k];
        return;
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
        const float d = z[k] - a.m, e = fast_exp(d);
        a.s += e;
        a.t += e * fmaxf(d, -3.0e38f);                           // a masked level: 0 times a number
    }
}

__device__ __forceinline__ void wave_join(Sums& a) {
    over_group<64>([&](auto from) { a.join(Sums{from(a.m), from(a.s), from(a.t)}); });
}

struct Part { float m, s, t, v; int j; };

struct Cut {
    int parts, length;           // levels of a part
    Part* part;                  // [rows][parts], parts > 1
    float* top_v;                // [rows][parts][top]
    int* top_j;
};

// The row's outputs, from its joined sums; called by one whole wavefront.
template <class T> __device__ __forceinline__ void put_choice(const Rows& R, const ChooseOut& O, int64_t r, const Sums& a, const Best& b, int lane) {
    if (lane) return;
    const bool some = a.s != 0.0f, found = b.j < R.levels;
    const float logs = fast_log(a.s);
    O.level[r] = some && found ? b.j : 0;
    O.logprob[r] = !some ? 0.0f : found ? to_f32(((const T*)R.logits + row_base(R, r))[b.j]) - a.m - logs : __builtin_nanf("");
    O.entropy[r] = entropy_of(a, logs);
}
// (asked for early: two dependent loads)
struct Given { int64_t l; float z; };
template <class T> __device__ __forceinline__ Given given_level(const Rows& R, const ScoreOut& O, int64_t r) {
    Given x{O.level[r], kNegInf};
    if (x.l >= 0 && x.l < R.levels) {
        const uint8_t* mk = row_mask(R, r);
        if (!mk || mk[x.l * R.mask_level]) x.z = to_f32(((const T*)R.logits + row_base(R, r))[x.l]);
    }
    return x;
}
template <class T> __device__ __forceinline__ void put_score(const Rows& R, const ScoreOut& O, int64_t r, const Given& x, const Sums& a, const TopList& list, int lane) {
    const float logs = fast_log(a.s);
    if (lane == 0) {
        O.logprob[r] = x.l >= R.levels ? __builtin_nanf("") : x.l < 0 || a.s == 0.0f ? 0.0f : x.z - a.m - logs;
        O.entropy[r] = entropy_of(a, logs);
        if (O.stat) { O.stat[2 * r] = a.m; O.stat[2 * r + 1] = a.s; }
    }
    if (lane < O.top) {
        const bool some = list.v > kNegInf;
        O.top_logprob[r * O.top + lane] = some ? list.v - a.m - logs : a.s == a.s ? kNegInf : a.s;
        O.top_level[r * O.top + lane] = some ? list.j : -1;
    }
}

template <class T, bool CHOOSE, bool MASK>
__global__ __launch_bounds__(256) void wide_kernel(Rows R, ChooseOut C, ScoreOut O, Cut cut) {
    constexpr int N = Piece<T>::N;
    __shared__ Part waves[4];
    __shared__ float maxima[256];
    __shared__ float list_v[3 * LRN_MAX_TOP];
    __shared__ int list_j[3 * LRN_MAX_TOP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t number = block_number(), r = cut.parts > 1 ? number / cut.parts : number;
    const int p = (int)(number - r * cut.parts);
    if (r >= R.rows) return;
    const int begin = p * cut.length, end = min(begin + cut.length, R.levels);
    int64_t o, i;
    split(R, r, o, i);
    const T* src = (const T*)R.logits + o * R.so + i * R.si;
    const uint8_t* mk = MASK ? R.mask + o * R.mo + i * R.mi : nullptr;
    const float* ns = CHOOSE && C.noise ? C.noise + o * C.no + i * C.ni : nullptr;
    Sums a;
    a.clear();
    Best b;
    b.clear();
    TopList list;
    list.clear();
    const int top = CHOOSE ? 0 : O.top;
    Given given{};
    if (!CHOOSE && cut.parts == 1 && tid == 0) given = given_level<T>(R, O, r);
    over_pieces<T, MASK, CHOOSE>(src, mk, R.mask_level, ns, begin, end, [&](const float (&z)[N], const float (&w)[N], int e0) {
        add_piece(a, z);
        if constexpr (CHOOSE) {
#pragma unroll
            for (int k = 0; k < N; k++) {                        // (a lane's levels rise)
                const float key = ns ? choice_key(z[k], w[k]) : z[k];
                if (z[k] > kNegInf && key > b.v) { b.v = key; b.j = e0 + k; }
            }
        }
    });
    if (top) {
        // The top-th largest of the 256 lanes' maxima is at most the row's: a second walk (the part is in the caches) has
        // little more than `top` candidates left to put in order.
        maxima[tid] = a.m;
        __syncthreads();
        list.clear(nth_of_256({maxima[lane], maxima[lane + 64], maxima[lane + 128], maxima[lane + 192]}, top));
        over_pieces<T, MASK, false>(src, mk, R.mask_level, nullptr, begin, end, [&](const float (&z)[N], const float (&)[N], int e0) {      // (whole wavefronts)
            float best = z[0];
#pragma unroll
            for (int k = 1; k < N; k++) best = fmaxf(best, z[k]);
            if (__ballot(best >= list.bound && best > kNegInf)) {
#pragma unroll
                for (int k = 0; k < N; k++) list.offer(z[k], e0 + k, top, lane);
            }
        });
    }
    wave_join(a);
    if constexpr (CHOOSE) over_group<64>([&](auto from) { b.add(from(b.v), from(b.j)); });
    if (lane == 0) waves[wave] = Part{a.m, a.s, a.t, b.v, b.j};
    if (top && wave && lane < top) { list_v[(wave - 1) * LRN_MAX_TOP + lane] = list.v; list_j[(wave - 1) * LRN_MAX_TOP + lane] = list.j; }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < 4; w++) {
        a.join(Sums{waves[w].m, waves[w].s, waves[w].t});
        if constexpr (CHOOSE) b.add(waves[w].v, waves[w].j);
        else if (top) list.offer(lane < top ? list_v[(w - 1) * LRN_MAX_TOP + lane] : kNegInf, lane < top ? list_j[(w - 1) * LRN_MAX_TOP + lane] : 0, top, lane);
    }
    if (cut.parts == 1) {
        finish(a);
        if constexpr (CHOOSE) put_choice<T>(R, C, r, a, b, lane);
        else put_score<T>(R, O, r, given, a, list, lane);
    } else {
        if (lane == 0) cut.part[number] = Part{a.m, a.s, a.t, b.v, b.j};
        if (lane < top) { cut.top_v[number * top + lane] = list.v; cut.top_j[number * top + lane] = list.j; }
    }
}

template <class T, bool CHOOSE>
__global__ __launch_bounds__(64) void join_kernel(Rows R, ChooseOut C, ScoreOut O, Cut cut) {
    const int lane = threadIdx.x;
    const int64_t r = block_number();
    if (r >= R.rows) return;
    Given given{};
    if (!CHOOSE && lane == 0) given = given_level<T>(R, O, r);
    Part mine{kNegInf, 0.0f, 0.0f, kNegInf, 0x7fffffff};
    if (lane < cut.parts) mine = cut.part[r * cut.parts + lane];
    Sums a{mine.m, mine.s, mine.t};
    Best b{mine.v, mine.j};
    TopList list;
    list.clear();
    if constexpr (CHOOSE) {
        wave_join(a);
        finish(a);
        over_group<64>([&](auto from) { b.add(from(b.v), from(b.j)); });
        put_choice<T>(R, C, r, a, b, lane);
    } else {
        // The parts' best first, then their second best, ...: 64 candidates hold one of each part, and where none of them
        // gets in, nothing that follows does.
        const int top = O.top, n = cut.parts * top;
        auto fetch = [&](int k, float& v, int& j) {
            const int64_t from = r * n + (k % cut.parts) * top + k / cut.parts;
            v = k < n ? cut.top_v[from] : kNegInf;
            j = k < n ? cut.top_j[from] : 0x7fffffff;
        };
        float v, next_v;
        int j, next_j;
        fetch(lane, next_v, next_j);
        wave_join(a);
        finish(a);
        for (int k0 = 0; k0 < n; k0 += 64) {
            v = next_v;
            j = next_j;
            if (!__ballot(v > list.bound || (v == list.bound && v > kNegInf && j < list.bound_j))) break;
            fetch(k0 + 64 + lane, next_v, next_j);
            list.offer(v, j, top, lane);
        }
        put_score<T>(R, O, r, given, a, list, lane);
    }
}

// One piece of 16 bytes after the other, with the row's statistics: bound by memory (1024 x 32768 bfloat16: 134 MB in 25.6 us,
// 5.2 TB/s; the forward pass has just left the logits in the last-level cache).
constexpr int kBackPieces = 4;       // pieces a lane
template <class T>
__global__ __launch_bounds__(256) void wide_backward_kernel(Rows R, BackIn I, T* grad, int parts) {
    constexpr int N = Piece<T>::N;
    const int64_t number = block_number(), r = number / parts;
    if (r >= R.rows) return;
    const int begin = (int)(number - r * parts) * (256 * N * kBackPieces), end = min(begin + 256 * N * kBackPieces, R.levels);
    int64_t o, i;
    split(R, r, o, i);
    const T* src = (const T*)R.logits + o * R.so + i * R.si;
    const uint8_t* mk = R.mask ? R.mask + o * R.mo + i * R.mi : nullptr;
    T* out = grad + r * R.levels;
    const float m = I.stat[2 * r], s = I.stat[2 * r + 1], H = I.entropy[r];
    const int64_t l = I.level[r];
    float g = I.g_lp && l >= 0 ? I.g_lp[r * I.g_lp_stride] : 0.0f;
    const float gh = I.g_h ? I.g_h[r * I.g_h_stride] : 0.0f, inv = s != 0.0f ? fast_inverse(s) : 0.0f;
    const float lift = s != 0.0f ? H - fast_log(s) : 0.0f;           // log p + H = z - m + lift
    if (l >= R.levels) g = __builtin_nanf("");
#pragma unroll
    for (int n = 0; n < kBackPieces; n++) {
        const int e0 = begin + (n * 256 + (int)threadIdx.x) * N;
        if (e0 >= end) return;
        float z[N];
        load_piece<T>(src, mk, R.mask_level, e0, end, z);
        typename Piece<T>::vec v;
#pragma unroll
        for (int k = 0; k < N; k++) {
            const float w = z[k] - m, e = fast_exp(w), p = e * inv;
            float d = -p * (g + gh * (e > 0.0f ? w + lift : 0.0f));
            if (e0 + k == l) d += g;
            v[k] = (T)(z[k] == kNegInf ? 0.0f : d);
        }
        if (e0 + N <= end) *reinterpret_cast<typename Piece<T>::vec*>(out + e0) = v;
        else {
#pragma unroll
            for (int k = 0; k < N; k++)
                if (e0 + k < end) out[e0 + k] = v[k];
        }
    }
}

// Parts of a row: enough workgroups for four a compute unit, parts of 4096 levels at least (a part's fixed cost, its joins, is
// about that of 2000 levels), at most one for each lane of the joining wavefront.
Cut cut_of(const Rows& R, int top, void* workspace) {
    Cut c{};
    int64_t parts = std::min<int64_t>({cdiv(1024, R.rows), cdiv(R.levels, 4096), 64});
    c.length = (int)(cdiv(cdiv(R.levels, parts), 2048) * 2048);
    c.parts = (int)cdiv(R.levels, c.length);
    if (c.parts > 1) {
        c.part = (Part*)workspace;
        c.top_v = (float*)(c.part + R.rows * c.parts);
        c.top_j = (int*)(c.top_v + R.rows * c.parts * top);
    }
    return c;
}
int64_t cut_bytes(const Rows& R, int top) {
    if (R.levels <= kGroupLevels || R.rows <= 0) return 0;
    const Cut c = cut_of(R, top, nullptr);
    return c.parts > 1 ? R.rows * c.parts * (int64_t)(sizeof(Part) + 8 * top) : 0;
}

bool dense(const lrn_rows& in, int64_t so, int64_t si) { return (in.inner <= 1 || si == in.levels) && (in.outer <= 1 || so == in.levels * in.inner); }
int64_t extent(const lrn_rows& in, int64_t so, int64_t si, int64_t levels) {
    return (in.outer > 0 ? in.outer - 1 : 0) * so + (in.inner > 0 ? in.inner - 1 : 0) * si + levels;
}

int checked(const lrn_rows* in, Rows* out) {
    if (!in) return fail(-1, "rows: null");
    if (in->outer < 0 || in->inner < 0 || in->levels < 1 || in->levels > 0x3fffffff)
        return fail(-1, "rows: outer %lld, inner %lld, levels %lld", (long long)in->outer, (long long)in->inner, (long long)in->levels);
    if (in->dtype != LRN_F32 && in->dtype != LRN_BF16 && in->dtype != LRN_F16) return fail(-1, "rows: dtype %d", in->dtype);
    if (in->mask_level != 0 && in->mask_level != 1) return fail(-1, "rows: mask_level %d", in->mask_level);
    out->rows = in->outer * in->inner;
    if (out->rows && !in->logits) return fail(-1, "rows: null logits");
    out->logits = in->logits;
    out->mask = in->mask;
    out->inner = in->inner ? in->inner : 1;
    out->so = in->stride_outer; out->si = in->stride_inner;
    out->mo = in->mask_outer; out->mi = in->mask_inner;
    out->levels = (int32_t)in->levels;
    out->mask_level = in->mask_level;
    if (in->stride_outer < 0 || in->stride_inner < 0 || in->mask_outer < 0 || in->mask_inner < 0) return fail(-1, "rows: negative strides");
    out->dense = dense(*in, out->so, out->si);
    out->mask_dense = out->mask_level == 1 && dense(*in, out->mo, out->mi);
    out->limit = extent(*in, out->so, out->si, in->levels);
    out->mask_limit = extent(*in, out->mo, out->mi, out->mask_level ? in->levels : 1);
    return 0;
}

int64_t size_of(int dtype) { return dtype == LRN_F32 ? 4 : 2; }
int grid_of(int64_t blocks, dim3* grid) {
    if (blocks >= (int64_t)1 << 36) return fail(-1, "rows: too many for one call");
    const RowGrid g = row_grid(blocks);
    *grid = dim3((unsigned)g.x, (unsigned)g.y);
    return 0;
}

int check_workspace(int64_t need, const void* workspace, int64_t bytes, const char* who) {
    if (need && (!workspace || bytes < need)) return fail(-1, "%s: a workspace of %lld bytes is needed, got %lld", who, (long long)need, (long long)bytes);
    return 0;
}

template <class T, bool CHOOSE> int launch_wide(const Rows& R, const ChooseOut& C, const ScoreOut& O, int top, void* workspace, hipStream_t stream, const char* who) {
    const Cut cut = cut_of(R, top, workspace);
    dim3 grid, rows;
    if (int rc = grid_of(R.rows * cut.parts, &grid)) return rc;
    if (int rc = grid_of(R.rows, &rows)) return rc;
    if (R.mask) wide_kernel<T, CHOOSE, true><<<grid, 256, 0, stream>>>(R, C, O, cut);
    else wide_kernel<T, CHOOSE, false><<<grid, 256, 0, stream>>>(R, C, O, cut);
    if (cut.parts > 1) join_kernel<T, CHOOSE><<<rows, 64, 0, stream>>>(R, C, O, cut);
    LRN_LAUNCHED(who);
    return 0;
}

}  // namespace
}  // namespace lrn

using namespace lrn;

#define BY_TYPE(dtype, call)                                   \
    switch (dtype) {                                           \
        case LRN_F32: { using T = float; call; break; }        \
        case LRN_BF16: { using T = bf16; call; break; }        \
        default: { using T = f16; call; break; }               \
    }

extern "C" {

const char* lrn_last_error(void) { return error_text(); }

int64_t lrn_choose_workspace(const lrn_rows* rows) {
    Rows R;
    return rows && checked(rows, &R) == 0 ? cut_bytes(R, 0) : 0;
}

int lrn_choose(int32_t device, void* hip_stream, const lrn_rows* rows, const float* noise, int64_t noise_outer,
               int64_t noise_inner, int64_t* level_out, float* logprob_out, float* entropy_out, void* workspace, int64_t workspace_bytes) {
    Rows R;
    if (int rc = checked(rows, &R)) return rc;
    if (!R.rows) return 0;
    if (!level_out || !logprob_out || !entropy_out) return fail(-1, "lrn_choose: null output");
    if (noise_outer < 0 || noise_inner < 0) return fail(-1, "lrn_choose: negative noise strides");
    if (int rc = check_workspace(cut_bytes(R, 0), workspace, workspace_bytes, "lrn_choose")) return rc;
    LRN_ON_DEVICE(device);
    const ChooseOut O{noise, noise_outer, noise_inner, extent(*rows, noise_outer, noise_inner, R.levels),
                      !noise || dense(*rows, noise_outer, noise_inner), level_out, logprob_out, entropy_out};
    if (R.levels <= kGroupLevels) {
        dim3 grid;
        if (int rc = grid_of(cdiv(R.rows, group_rows(R.levels)), &grid)) return rc;
        hipStream_t stream = (hipStream_t)hip_stream;
        BY_TYPE(rows->dtype, BY_LEVELS(R.levels, (group_choose_kernel<T, G, E><<<grid, 256, 0, stream>>>(R, O))));
        LRN_LAUNCHED("lrn_choose");
        return 0;
    }
    BY_TYPE(rows->dtype, return (launch_wide<T, true>(R, O, ScoreOut{}, 0, workspace, (hipStream_t)hip_stream, "lrn_choose")));
}

int64_t lrn_score_workspace(const lrn_rows* rows, int32_t top) {
    Rows R;
    return rows && top >= 0 && top <= LRN_MAX_TOP && checked(rows, &R) == 0 ? cut_bytes(R, top) : 0;
}

int lrn_score(int32_t device, void* hip_stream, const lrn_rows* rows, const int64_t* level, float* logprob_out,
              float* entropy_out, float* stat_out, int32_t top, float* top_logprob_out, int64_t* top_level_out, void* workspace,
              int64_t workspace_bytes) {
    Rows R;
    if (int rc = checked(rows, &R)) return rc;
    if (top < 0 || top > LRN_MAX_TOP || top > R.levels) return fail(-1, "lrn_score: top %d of %d levels (at most %d)", top, R.levels, LRN_MAX_TOP);
    if (!R.rows) return 0;
    if (!level || !logprob_out || !entropy_out || (top && (!top_logprob_out || !top_level_out))) return fail(-1, "lrn_score: null argument");
    if (int rc = check_workspace(cut_bytes(R, top), workspace, workspace_bytes, "lrn_score")) return rc;
    LRN_ON_DEVICE(device);
    const ScoreOut O{level, logprob_out, entropy_out, stat_out, top, top_logprob_out, top_level_out};
    if (R.levels <= kGroupLevels) {
        dim3 grid;
        const int lanes = lanes_for(R.levels, top);
        if (int rc = grid_of(cdiv(R.rows, group_rows(lanes)), &grid)) return rc;
        hipStream_t stream = (hipStream_t)hip_stream;
        BY_TYPE(rows->dtype, BY_LEVELS(lanes, (group_score_kernel<T, G, E><<<grid, 256, 0, stream>>>(R, O))));
        LRN_LAUNCHED("lrn_score");
        return 0;
    }
    BY_TYPE(rows->dtype, return (launch_wide<T, false>(R, ChooseOut{}, O, top, workspace, (hipStream_t)hip_stream, "lrn_score")));
}

int lrn_score_backward(int32_t device, void* hip_stream, const lrn_rows* rows, const int64_t* level, const float* stat,
                       const float* entropy, const float* g_logprob, int32_t g_logprob_stride, const float* g_entropy,
                       int32_t g_entropy_stride, void* grad_out) {
    Rows R;
    if (int rc = checked(rows, &R)) return rc;
    if (!R.rows) return 0;
    const bool again = R.levels <= kGroupLevels;
    if (!level || !grad_out || (!again && (!stat || !entropy))) return fail(-1, "lrn_score_backward: null argument");
    if ((g_logprob_stride & ~1) || (g_entropy_stride & ~1)) return fail(-1, "lrn_score_backward: gradient strides are 0 or 1");
    LRN_ON_DEVICE(device);
    const BackIn I{level, stat, entropy, g_logprob, g_entropy, g_logprob_stride, g_entropy_stride};
    if (again) {
        dim3 grid;
        if (int rc = grid_of(cdiv(R.rows, group_rows(R.levels)), &grid)) return rc;
        hipStream_t stream = (hipStream_t)hip_stream;
        BY_TYPE(rows->dtype, BY_LEVELS(R.levels, (group_backward_kernel<T, G, E><<<grid, 256, 0, stream>>>(R, I, (T*)grad_out))));
        LRN_LAUNCHED("lrn_score_backward");
        return 0;
    }
    const int64_t parts = cdiv(R.levels, 256 * kBackPieces * 16 / size_of(rows->dtype));
    dim3 grid;
    if (int rc = grid_of(R.rows * parts, &grid)) return rc;
    BY_TYPE(rows->dtype, (wide_backward_kernel<T><<<grid, 256, 0, (hipStream_t)hip_stream>>>(R, I, (T*)grad_out, (int)parts)));
    LRN_LAUNCHED("lrn_score_backward");
    return 0;
}

}  // extern "C"
