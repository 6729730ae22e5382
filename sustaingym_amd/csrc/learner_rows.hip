// learner_rows.hip — gfx950 kernels of lrn_choose / lrn_score / lrn_score_backward (include/learner_ops.h).
//
// One pass over a row with the running maximum m, s = sum exp(z - m) and t = sum exp(z - m) (z - m): when the maximum moves
// from m to m', c = exp(m - m') rescales s' = c s and t' = c (t + s (m - m')).  log s and t / s are all that the log
// probability and the entropy need.  Sums are float32 whatever the logits' type.
#include <algorithm>
#include <type_traits>

#include "lrn_common.h"

namespace lrn {

char* error_text() {
    static thread_local char text[512] = "";
    return text;
}

namespace {

struct Rows {
    const void* logits;
    const uint8_t* mask;
    int64_t rows, inner;
    int64_t so, si, mo, mi;
    int32_t levels, mask_level;
    uint32_t per_level;          // ceil(2^32 / levels): e / levels = e per_level >> 32 for e < 2^16, levels <= 1024
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

__device__ __forceinline__ float lane_of(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// The 64 best of what a wavefront has seen, lane i the i-th (falling, the lowest index first among equals).  Candidates go in
// one at a time: k (1 + log(n / k)) of n values do.  What an insertion costs is latency, so nothing in it goes through LDS: the
// candidate and the bound are scalars (v_readlane), the entries behind it move up by one lane with a whole-wavefront shift.
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
__device__ __forceinline__ float entropy_of(const Sums& a, float logs) { return a.s != 0.0f ? logs - a.t / a.s : 0.0f; }

struct ChooseOut { const float* noise; int64_t no, ni; int64_t* level; float* logprob; float* entropy; };
struct ScoreOut { const int64_t* level; float* logprob; float* entropy; float* stat; int top; float* top_logprob; int64_t* top_level; };

struct BackIn { const int64_t* level; const float* stat; const float* entropy; const float* g_lp; const float* g_h; int g_lp_stride, g_h_stride; };

// ---- rows of up to 1024 levels: G lanes to a row -----------------------------------------------------------------------
//
// A workgroup takes 256 / G rows.  Their logits are one run of memory (FLAT): 16-byte loads by all lanes bring it, whatever
// the rows' length, and the rows are picked out of LDS, where they sit an odd number of words apart (no two lanes of a
// half-wavefront on one bank).  A lane holds E levels of its row in registers, so that the maximum comes first and every
// weight is computed once; the group's sums go through DPP.  The backward pass computes the row's maximum and sums again from
// the logits that it has to read anyway: cheaper than 12 bytes a row of saved statistics.  Rows at other strides, broadcast
// masks and unaligned starts are read a row at a time by the row's own lanes (not FLAT).

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

// What a group knows of its row: the levels g, g + G, ... are z[0], z[1], ... of lane g (-inf behind the row and where masked).
template <int G, int E>
__device__ __forceinline__ Sums group_sums(const float (&z)[E], float (&e)[E]) {
    Sums a;
    a.m = z[0];
#pragma unroll
    for (int k = 1; k < E; k++) a.m = fmaxf(a.m, z[k]);
    over_group<G>([&](auto from) { a.m = fmaxf(a.m, from(a.m)); });
    a.s = a.t = 0.0f;
#pragma unroll
    for (int k = 0; k < E; k++) {
        const float d = z[k] - a.m;
        e[k] = z[k] == kNegInf ? 0.0f : fast_exp(d);
        a.s += e[k];
        a.t += e[k] > 0.0f ? e[k] * d : 0.0f;
    }
    over_group<G>([&](auto from) { a.s += from(a.s); a.t += from(a.t); });
    finish(a);
    return a;
}

template <int G, int E> constexpr int kTile = 256 / G * (G * E + 1);

// The tile's logits (and noise) into LDS as float32; masked ones as -inf.
template <class T, int G, int E, bool FLAT, bool NOISE>
__device__ __forceinline__ void load_tile(const Rows& R, const ChooseOut* C, int64_t r0, int rows, float* z, float* nz) {
    const int K = R.levels, pitch = K | 1, tid = threadIdx.x;
    if constexpr (FLAT) {
        constexpr int VE = 16 / sizeof(T);
        const int n = rows * K;
        const T* src = (const T*)R.logits + r0 * K;
        const uint8_t* mk = R.mask ? R.mask + r0 * K : nullptr;
        const float* ns = NOISE && C->noise ? C->noise + r0 * K : nullptr;
        for (int e0 = tid * VE; e0 < n; e0 += 256 * VE) {
            int row = __umulhi((uint32_t)e0, R.per_level), col = e0 - row * K;
            T v[VE];
            uint8_t b[VE];
            float w[VE];
            const bool whole = e0 + VE <= n;
            if (whole) {
                *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(src + e0);
                if (mk) {
                    if constexpr (VE == 8) *reinterpret_cast<uint2*>(b) = *reinterpret_cast<const uint2*>(mk + e0);
                    else *reinterpret_cast<uint32_t*>(b) = *reinterpret_cast<const uint32_t*>(mk + e0);
                }
                if (NOISE && ns) {
#pragma unroll
                    for (int k = 0; k < VE; k += 4) *reinterpret_cast<float4*>(w + k) = *reinterpret_cast<const float4*>(ns + e0 + k);
                }
            } else {
#pragma unroll
                for (int k = 0; k < VE; k++)
                    if (e0 + k < n) { v[k] = src[e0 + k]; if (mk) b[k] = mk[e0 + k]; if (NOISE && ns) w[k] = ns[e0 + k]; }
            }
#pragma unroll
            for (int k = 0; k < VE; k++) {
                if (whole || e0 + k < n) {
                    z[row * pitch + col] = mk && !b[k] ? kNegInf : to_f32(v[k]);
                    if (NOISE && ns) nz[row * pitch + col] = w[k];
                }
                if (++col == K) { col = 0; row++; }
            }
        }
    } else {
        const int row = tid / G, g = tid % G;
        if (row < rows) {
            int64_t o, i;
            split(R, r0 + row, o, i);
            const T* src = (const T*)R.logits + o * R.so + i * R.si;
            const uint8_t* mk = R.mask ? R.mask + o * R.mo + i * R.mi : nullptr;
            const float* ns = NOISE && C->noise ? C->noise + o * C->no + i * C->ni : nullptr;
#pragma unroll
            for (int k = 0; k < E; k++) {
                const int j = g + G * k;
                if (j < K) {
                    z[row * pitch + j] = mk && !mk[j * R.mask_level] ? kNegInf : to_f32(src[j]);
                    if (NOISE && ns) nz[row * pitch + j] = ns[j];
                }
            }
        }
    }
    __syncthreads();
}

template <class T, int G, int E, bool FLAT>
__global__ __launch_bounds__(256) void group_choose_kernel(Rows R, ChooseOut O) {
    __shared__ float zs[kTile<G, E>], ns[kTile<G, E>];
    const int64_t r0 = (int64_t)blockIdx.x * (256 / G);
    const int rows = (int)min((int64_t)(256 / G), R.rows - r0), K = R.levels;
    load_tile<T, G, E, FLAT, true>(R, &O, r0, rows, zs, ns);
    const int row = threadIdx.x / G, g = threadIdx.x % G;
    if (row >= rows) return;                    // whole groups: no lane of a group leaves alone
    const float* mine = zs + row * (K | 1);
    const float* noise = ns + row * (K | 1);
    float z[E], e[E];
    Best b;
    b.clear();
#pragma unroll
    for (int k = 0; k < E; k++) {
        const int j = g + G * k;
        z[k] = j < K ? mine[j] : kNegInf;
        if (z[k] != kNegInf) b.add(O.noise ? z[k] + noise[j] : z[k], j);
    }
    const Sums a = group_sums<G, E>(z, e);
    over_group<G>([&](auto from) { b.add(from(b.v), from(b.j)); });
    if (g == 0) {
        const bool some = a.s != 0.0f, found = b.j < K;
        const float logs = logf(a.s);
        O.level[r0 + row] = some && found ? b.j : 0;
        O.logprob[r0 + row] = !some ? 0.0f : found ? mine[b.j] - a.m - logs : __builtin_nanf("");
        O.entropy[r0 + row] = entropy_of(a, logs);
    }
}

template <class T, int G, int E, bool FLAT>
__global__ __launch_bounds__(256) void group_score_kernel(Rows R, ScoreOut O) {
    __shared__ float zs[kTile<G, E>];
    const int64_t r0 = (int64_t)blockIdx.x * (256 / G);
    const int rows = (int)min((int64_t)(256 / G), R.rows - r0), K = R.levels;
    load_tile<T, G, E, FLAT, false>(R, nullptr, r0, rows, zs, nullptr);
    const int row = threadIdx.x / G, g = threadIdx.x % G;
    if (row >= rows) return;
    const int64_t r = r0 + row;
    const float* mine = zs + row * (K | 1);
    const int64_t l = g == 0 ? O.level[r] : 0;
    float z[E], e[E];
#pragma unroll
    for (int k = 0; k < E; k++) z[k] = g + G * k < K ? mine[g + G * k] : kNegInf;
    const Sums a = group_sums<G, E>(z, e);
    const float logs = logf(a.s);
    if (g == 0) {
        O.logprob[r] = l >= K ? __builtin_nanf("") : l < 0 || a.s == 0.0f ? 0.0f : mine[l] - a.m - logs;
        O.entropy[r] = entropy_of(a, logs);
        if (O.stat) { O.stat[2 * r] = a.m; O.stat[2 * r + 1] = a.s; }
    }
    for (int n = 0; n < O.top; n++) {           // the best of what is left, O.top times
        Best b;
        b.clear();
#pragma unroll
        for (int k = 0; k < E; k++)
            if (z[k] > kNegInf) b.add(z[k], g + G * k);
        over_group<G>([&](auto from) { b.add(from(b.v), from(b.j)); });
#pragma unroll
        for (int k = 0; k < E; k++)
            if (g + G * k == b.j) z[k] = kNegInf;
        if (g == 0) {
            const bool some = b.j < K;
            O.top_logprob[r * O.top + n] = some ? b.v - a.m - logs : a.s == a.s ? kNegInf : a.s;
            O.top_level[r * O.top + n] = some ? b.j : -1;
        }
    }
}

template <class T, int G, int E, bool FLAT>
__global__ __launch_bounds__(256) void group_backward_kernel(Rows R, BackIn I, T* grad, bool aligned) {
    __shared__ float zs[kTile<G, E>];
    const int64_t r0 = (int64_t)blockIdx.x * (256 / G);
    const int rows = (int)min((int64_t)(256 / G), R.rows - r0), K = R.levels, pitch = K | 1;
    load_tile<T, G, E, FLAT, false>(R, nullptr, r0, rows, zs, nullptr);
    const int row = threadIdx.x / G, g = threadIdx.x % G;
    if (row < rows) {
        const int64_t r = r0 + row;
        float* mine = zs + row * pitch;
        const int64_t l = I.level[r];
        const float gl = I.g_lp && l >= 0 ? I.g_lp[r * I.g_lp_stride] : 0.0f, gh = I.g_h ? I.g_h[r * I.g_h_stride] : 0.0f;
        float z[E], e[E];
#pragma unroll
        for (int k = 0; k < E; k++) z[k] = g + G * k < K ? mine[g + G * k] : kNegInf;
        const Sums a = group_sums<G, E>(z, e);
        const float logs = logf(a.s), inv = 1.0f / a.s, H = entropy_of(a, logs);
#pragma unroll
        for (int k = 0; k < E; k++) {
            const int j = g + G * k;
            const float p = e[k] * inv;
            float d = (j == l ? gl : 0.0f) - p * (gl + gh * (e[k] > 0.0f ? z[k] - a.m - logs + H : 0.0f));
            if (z[k] == kNegInf) d = 0.0f;
            if (l >= K) d = __builtin_nanf("");
            if (j < K) mine[j] = d;
        }
    }
    __syncthreads();
    constexpr int VE = 16 / sizeof(T);
    const int n = rows * K;
    T* out = grad + r0 * K;
    for (int e0 = threadIdx.x * VE; e0 < n; e0 += 256 * VE) {
        int at = __umulhi((uint32_t)e0, R.per_level), col = e0 - at * K;
        T v[VE];
#pragma unroll
        for (int k = 0; k < VE; k++) {
            v[k] = e0 + k < n ? (T)zs[at * pitch + col] : (T)0.0f;
            if (++col == K) { col = 0; at++; }
        }
        if (aligned && e0 + VE <= n) *reinterpret_cast<uint4*>(out + e0) = *reinterpret_cast<const uint4*>(v);
        else {
#pragma unroll
            for (int k = 0; k < VE; k++)
                if (e0 + k < n) out[e0 + k] = v[k];
        }
    }
}

// 8 levels to a lane fill the registers of a full set of wavefronts; up to 1024 levels a wavefront is one row.
constexpr int kGroupLevels = 1024;
#define BY_LEVELS(K, call)                                                          \
    do {                                                                            \
        if ((K) <= 4) { constexpr int G = 1, E = 4; call; }                         \
        else if ((K) <= 8) { constexpr int G = 1, E = 8; call; }                    \
        else if ((K) <= 16) { constexpr int G = 2, E = 8; call; }                   \
        else if ((K) <= 32) { constexpr int G = 4, E = 8; call; }                   \
        else if ((K) <= 64) { constexpr int G = 8, E = 8; call; }                   \
        else if ((K) <= 128) { constexpr int G = 16, E = 8; call; }                 \
        else if ((K) <= 256) { constexpr int G = 32, E = 8; call; }                 \
        else if ((K) <= 512) { constexpr int G = 64, E = 8; call; }                 \
        else { constexpr int G = 64, E = 16; call; }                                \
    } while (0)

int group_rows(int64_t K) { int g = 256; BY_LEVELS(K, (g = 256 / G, (void)E)); return g; }

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Whether the rows (and mask, noise) are one dense run whose tiles start on 16 bytes (the mask's on 8, float32: 4).
bool flat(const Rows& R, int64_t size, const float* noise, int64_t no, int64_t ni) {
    const int64_t K = R.levels, per = group_rows(K) * K;
    const bool one = R.rows == R.inner;
    auto dense = [&](int64_t o, int64_t i) { return (R.inner == 1 || i == K) && (one || o == K * R.inner); };
    if (!dense(R.so, R.si) || !aligned16(R.logits) || (per * size) % 16) return false;
    if (R.mask && (R.mask_level != 1 || !dense(R.mo, R.mi) || ((uintptr_t)R.mask & 7) || per % 8)) return false;
    return !noise || (dense(no, ni) && aligned16(noise) && per % 4 == 0);
}

// ---- longer rows: a workgroup to a row, or to a part of one -----------------------------------------------------------
//
// Every lane walks 16-byte pieces of the row (at any alignment: the hardware takes a vector load at its element's) with a
// running maximum and sums of its own, rescaled when a piece raises the maximum; the lanes join at the end.  Where there are
// too few rows to fill the GPU a row is cut into up to 64 parts, whose sums, best level and best alternatives go through the
// workspace to a second launch, a wavefront to a row.

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
template <class T, bool MASK, class F>
__device__ __forceinline__ void over_pieces(const T* src, const uint8_t* mk, int mask_level, int begin, int end, F&& f) {
    constexpr int N = Piece<T>::N, STEP = 256 * N;
    using V = typename Piece<T>::vec;
    using M = typename std::conditional_t<N == 8, Mask8, Mask4>::vec;
    int base = begin;
    for (; base + kAhead * STEP <= end; base += kAhead * STEP) {
        const int e0 = base + (int)threadIdx.x * N;
        V v[kAhead];
        M b[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; u++) v[u] = *reinterpret_cast<const V*>(src + e0 + u * STEP);
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
            f(z, e0 + u * STEP);
        }
    }
    for (; base < end; base += STEP) {
        const int e0 = base + (int)threadIdx.x * N;
        float z[N];
        load_piece<T>(src, mk, mask_level, e0, end, z);
        f(z, e0);
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
    const float logs = logf(a.s);
    O.level[r] = some && found ? b.j : 0;
    O.logprob[r] = !some ? 0.0f : found ? to_f32(((const T*)R.logits + row_base(R, r))[b.j]) - a.m - logs : __builtin_nanf("");
    O.entropy[r] = entropy_of(a, logs);
}
template <class T> __device__ __forceinline__ void put_score(const Rows& R, const ScoreOut& O, int64_t r, const Sums& a, const TopList& list, int lane) {
    const float logs = logf(a.s);
    if (lane == 0) {
        const int64_t l = O.level[r];
        float lp = 0.0f;
        if (l >= R.levels) lp = __builtin_nanf("");
        else if (l >= 0 && a.s != 0.0f) {
            const uint8_t* mk = row_mask(R, r);
            lp = (mk && !mk[l * R.mask_level] ? kNegInf : to_f32(((const T*)R.logits + row_base(R, r))[l])) - a.m - logs;
        }
        O.logprob[r] = lp;
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
    const int64_t r = cut.parts > 1 ? (int64_t)blockIdx.x / cut.parts : blockIdx.x;
    const int p = cut.parts > 1 ? (int)(blockIdx.x - r * cut.parts) : 0;
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
    over_pieces<T, MASK>(src, mk, R.mask_level, begin, end, [&](const float (&z)[N], int e0) {
        add_piece(a, z);
        if constexpr (CHOOSE) {
#pragma unroll
            for (int k = 0; k < N; k++)
                if (z[k] != kNegInf) b.add(ns ? z[k] + ns[e0 + k] : z[k], e0 + k);
        }
    });
    if (top) {
        // The top-th largest of the 256 lanes' maxima is at most the row's: a second walk (the part is in the caches) has
        // little more than `top` candidates left to put in order.
        maxima[tid] = a.m;
        __syncthreads();
        list.clear(nth_of_256({maxima[lane], maxima[lane + 64], maxima[lane + 128], maxima[lane + 192]}, top));
        over_pieces<T, MASK>(src, mk, R.mask_level, begin, end, [&](const float (&z)[N], int e0) {      // (whole wavefronts)
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
        else put_score<T>(R, O, r, a, list, lane);
    } else {
        if (lane == 0) cut.part[blockIdx.x] = Part{a.m, a.s, a.t, b.v, b.j};
        if (lane < top) { cut.top_v[(int64_t)blockIdx.x * top + lane] = list.v; cut.top_j[(int64_t)blockIdx.x * top + lane] = list.j; }
    }
}

template <class T, bool CHOOSE>
__global__ __launch_bounds__(64) void join_kernel(Rows R, ChooseOut C, ScoreOut O, Cut cut) {
    const int lane = threadIdx.x;
    const int64_t r = blockIdx.x;
    Part mine{kNegInf, 0.0f, 0.0f, kNegInf, 0x7fffffff};
    if (lane < cut.parts) mine = cut.part[r * cut.parts + lane];
    Sums a{mine.m, mine.s, mine.t};
    Best b{mine.v, mine.j};
    TopList list;
    list.clear();
    wave_join(a);
    finish(a);
    if constexpr (CHOOSE) {
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
        for (int k0 = 0; k0 < n; k0 += 64) {
            v = next_v;
            j = next_j;
            if (!__ballot(v > list.bound || (v == list.bound && v > kNegInf && j < list.bound_j))) break;
            fetch(k0 + 64 + lane, next_v, next_j);
            list.offer(v, j, top, lane);
        }
        put_score<T>(R, O, r, a, list, lane);
    }
}

// One piece of 16 bytes after the other, with the row's statistics: bound by memory.
constexpr int kBackPieces = 4;       // pieces a lane
template <class T>
__global__ __launch_bounds__(256) void wide_backward_kernel(Rows R, BackIn I, T* grad, int parts) {
    constexpr int N = Piece<T>::N;
    const int64_t r = blockIdx.x / (unsigned)parts;
    const int begin = (int)(blockIdx.x - r * parts) * (256 * N * kBackPieces), end = min(begin + 256 * N * kBackPieces, R.levels);
    int64_t o, i;
    split(R, r, o, i);
    const T* src = (const T*)R.logits + o * R.so + i * R.si;
    const uint8_t* mk = R.mask ? R.mask + o * R.mo + i * R.mi : nullptr;
    T* out = grad + r * R.levels;
    const float m = I.stat[2 * r], s = I.stat[2 * r + 1], H = I.entropy[r];
    const int64_t l = I.level[r];
    float g = I.g_lp && l >= 0 ? I.g_lp[r * I.g_lp_stride] : 0.0f;
    const float gh = I.g_h ? I.g_h[r * I.g_h_stride] : 0.0f, inv = s != 0.0f ? 1.0f / s : 0.0f;
    const float lift = s != 0.0f ? H - logf(s) : 0.0f;           // log p + H = z - m + lift
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
    out->per_level = (uint32_t)((0xffffffffull + in->levels) / in->levels);
    return 0;
}

int64_t size_of(int dtype) { return dtype == LRN_F32 ? 4 : 2; }
int tiles(const Rows& R, unsigned* grid) {
    const int64_t n = cdiv(R.rows, group_rows(R.levels));
    if (n > 0x7fffffff) return fail(-1, "rows: %lld are too many for one call", (long long)R.rows);
    *grid = (unsigned)n;
    return 0;
}

int check_workspace(int64_t need, const void* workspace, int64_t bytes, const char* who) {
    if (need && (!workspace || bytes < need)) return fail(-1, "%s: a workspace of %lld bytes is needed, got %lld", who, (long long)need, (long long)bytes);
    return 0;
}

template <class T, bool CHOOSE> int launch_wide(const Rows& R, const ChooseOut& C, const ScoreOut& O, int top, void* workspace, hipStream_t stream, const char* who) {
    const Cut cut = cut_of(R, top, workspace);
    if (R.rows * cut.parts > 0x7fffffff) return fail(-1, "rows: %lld are too many for one call", (long long)R.rows);
    if (R.mask) wide_kernel<T, CHOOSE, true><<<(unsigned)(R.rows * cut.parts), 256, 0, stream>>>(R, C, O, cut);
    else wide_kernel<T, CHOOSE, false><<<(unsigned)(R.rows * cut.parts), 256, 0, stream>>>(R, C, O, cut);
    if (cut.parts > 1) join_kernel<T, CHOOSE><<<(unsigned)R.rows, 64, 0, stream>>>(R, C, O, cut);
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
    if (int rc = check_workspace(cut_bytes(R, 0), workspace, workspace_bytes, "lrn_choose")) return rc;
    LRN_ON_DEVICE(device);
    const ChooseOut O{noise, noise_outer, noise_inner, level_out, logprob_out, entropy_out};
    if (R.levels <= kGroupLevels) {
        unsigned grid;
        if (int rc = tiles(R, &grid)) return rc;
        hipStream_t stream = (hipStream_t)hip_stream;
        if (flat(R, size_of(rows->dtype), noise, noise_outer, noise_inner))
            BY_TYPE(rows->dtype, BY_LEVELS(R.levels, (group_choose_kernel<T, G, E, true><<<grid, 256, 0, stream>>>(R, O))))
        else
            BY_TYPE(rows->dtype, BY_LEVELS(R.levels, (group_choose_kernel<T, G, E, false><<<grid, 256, 0, stream>>>(R, O))))
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
        unsigned grid;
        if (int rc = tiles(R, &grid)) return rc;
        hipStream_t stream = (hipStream_t)hip_stream;
        if (flat(R, size_of(rows->dtype), nullptr, 0, 0))
            BY_TYPE(rows->dtype, BY_LEVELS(R.levels, (group_score_kernel<T, G, E, true><<<grid, 256, 0, stream>>>(R, O))))
        else
            BY_TYPE(rows->dtype, BY_LEVELS(R.levels, (group_score_kernel<T, G, E, false><<<grid, 256, 0, stream>>>(R, O))))
        LRN_LAUNCHED("lrn_score");
        return 0;
    }
    BY_TYPE(rows->dtype, return (launch_wide<T, false>(R, ChooseOut{}, O, top, workspace, (hipStream_t)hip_stream, "lrn_score")));
}

int lrn_score_backward_needs_stat(const lrn_rows* rows) { return rows && rows->levels > kGroupLevels; }

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
        unsigned grid;
        if (int rc = tiles(R, &grid)) return rc;
        hipStream_t stream = (hipStream_t)hip_stream;
        const bool out16 = aligned16(grad_out) && (group_rows(R.levels) * (int64_t)R.levels * size_of(rows->dtype)) % 16 == 0;
        if (flat(R, size_of(rows->dtype), nullptr, 0, 0))
            BY_TYPE(rows->dtype, BY_LEVELS(R.levels, (group_backward_kernel<T, G, E, true><<<grid, 256, 0, stream>>>(R, I, (T*)grad_out, out16))))
        else
            BY_TYPE(rows->dtype, BY_LEVELS(R.levels, (group_backward_kernel<T, G, E, false><<<grid, 256, 0, stream>>>(R, I, (T*)grad_out, out16))))
        LRN_LAUNCHED("lrn_score_backward");
        return 0;
    }
    const int64_t parts = cdiv(R.levels, 256 * kBackPieces * 16 / size_of(rows->dtype));
    if (R.rows * parts > 0x7fffffff) return fail(-1, "rows: %lld are too many for one call", (long long)R.rows);
    BY_TYPE(rows->dtype, (wide_backward_kernel<T><<<(unsigned)(R.rows * parts), 256, 0, (hipStream_t)hip_stream>>>(R, I, (T*)grad_out, (int)parts)));
    LRN_LAUNCHED("lrn_score_backward");
    return 0;
}

}  // extern "C"
