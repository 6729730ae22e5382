// learner_rows.hip — gfx950 kernels of lrn_choose / lrn_score / lrn_score_backward (include/learner_ops.h).
//
// One pass over a row with the running maximum m, s = sum exp(z - m) and t = sum exp(z - m) (z - m): when the maximum moves
// from m to m', c = exp(m - m') rescales s' = c s and t' = c (t + s (m - m')).  log s and t / s are all that the log
// probability and the entropy need.  Sums are float32 whatever the logits' type.
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
};

struct Sums {
    float m, s, t;
    __device__ __forceinline__ void clear() { m = kNegInf; s = 0.0f; t = 0.0f; }
    // one more logit (not -inf)
    __device__ __forceinline__ void add(float z) {
        if (z > m) {
            const float d = m - z, c = s > 0.0f ? fast_exp(d) : 0.0f;
            t = s > 0.0f ? c * (t + s * d) : 0.0f;
            s = c * s + 1.0f;
            m = z;
        } else {
            const float d = z - m, e = fast_exp(d);
            s += e;
            t += e > 0.0f ? e * d : (d != d ? d : 0.0f);
        }
    }
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

// The 64 best of what a wavefront has seen, lane i the i-th (falling, the lowest index first among equals).
struct TopList {
    float v;
    int j;
    __device__ __forceinline__ void clear() { v = kNegInf; j = 0x7fffffff; }
    __device__ __forceinline__ void insert(float x, int i, int lane) {
        const bool ahead = v > x || (v == x && j < i);
        const int at = __popcll(__ballot(ahead));
        const float pv = __shfl_up(v, 1);
        const int pj = __shfl_up(j, 1);
        if (lane > at) { v = pv; j = pj; }
        if (lane == at) { v = x; j = i; }
    }
    // every lane offers one candidate; only those ahead of the top-th entry are put in, one after the other
    __device__ __forceinline__ void offer(float x, int i, int top, int lane) {
        for (;;) {
            const float bound = __shfl(v, top - 1);
            const int bound_j = __shfl(j, top - 1);
            const unsigned long long some = __ballot(x > bound || (x == bound && x > kNegInf && i < bound_j));
            if (!some) return;
            const int src = __ffsll((long long)some) - 1;
            insert(__shfl(x, src), __shfl(i, src), lane);
            if (lane == src) x = kNegInf;
        }
    }
};

__device__ __forceinline__ int64_t row_base(const Rows& R, int64_t r) { return (r / R.inner) * R.so + (r % R.inner) * R.si; }
__device__ __forceinline__ const uint8_t* row_mask(const Rows& R, int64_t r) {
    return R.mask ? R.mask + (r / R.inner) * R.mo + (r % R.inner) * R.mi : nullptr;
}

__device__ __forceinline__ void wave_join(Sums& a) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        Sums b{__shfl_xor(a.m, o), __shfl_xor(a.s, o), __shfl_xor(a.t, o)};
        a.join(b);
    }
}
__device__ __forceinline__ void wave_join(Best& a) {
#pragma unroll
    for (int o = 32; o; o >>= 1) a.add(__shfl_xor(a.v, o), __shfl_xor(a.j, o));
}

// +inf among the allowed logits: no distribution
__device__ __forceinline__ void finish(Sums& a) { if (a.m == -kNegInf) a.s = __builtin_nanf(""); }
__device__ __forceinline__ float entropy_of(const Sums& a, float logs) { return a.s != 0.0f ? logs - a.t / a.s : 0.0f; }

struct ChooseOut { const float* noise; int64_t no, ni; int64_t* level; float* logprob; float* entropy; };
struct ScoreOut { const int64_t* level; float* logprob; float* entropy; float* stat; int top; float* top_logprob; int64_t* top_level; };

// A wavefront to a row.
template <class T>
__global__ __launch_bounds__(256) void choose_kernel(Rows R, ChooseOut O) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < R.rows; r += (int64_t)gridDim.x * 4) {
        const T* z = (const T*)R.logits + row_base(R, r);
        const uint8_t* mk = row_mask(R, r);
        const float* nz = O.noise ? O.noise + (r / R.inner) * O.no + (r % R.inner) * O.ni : nullptr;
        Sums a; a.clear();
        Best b; b.clear();
        float zb = 0.0f;
        for (int j = lane; j < R.levels; j += 64) {
            const float v = mk && !mk[(int64_t)j * R.mask_level] ? kNegInf : to_f32(z[j]);
            if (v == kNegInf) continue;
            a.add(v);
            b.add(nz ? v + nz[j] : v, j);
        }
        wave_join(a);
        wave_join(b);
        finish(a);
        if (lane == 0) {
            const bool some = a.s != 0.0f;
            const int at = b.j < R.levels ? b.j : 0;
            const float logs = logf(a.s);
            zb = to_f32(z[at]);
            O.level[r] = some ? at : 0;
            O.logprob[r] = some ? (b.j < R.levels ? zb - a.m - logs : __builtin_nanf("")) : 0.0f;
            O.entropy[r] = entropy_of(a, logs);
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void score_kernel(Rows R, ScoreOut O) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < R.rows; r += (int64_t)gridDim.x * 4) {
        const T* z = (const T*)R.logits + row_base(R, r);
        const uint8_t* mk = row_mask(R, r);
        Sums a; a.clear();
        TopList list; list.clear();
        for (int j0 = 0; j0 < R.levels; j0 += 64) {
            const int j = j0 + lane;
            float v = kNegInf;
            if (j < R.levels && !(mk && !mk[(int64_t)j * R.mask_level])) v = to_f32(z[j]);
            if (v != kNegInf) a.add(v);
            if (O.top) list.offer(v, j, O.top, lane);
        }
        wave_join(a);
        finish(a);
        const float logs = logf(a.s);
        if (lane == 0) {
            const int64_t l = O.level[r];
            float lp = 0.0f;
            if (l >= R.levels) lp = __builtin_nanf("");
            else if (l >= 0 && a.s != 0.0f) lp = (mk && !mk[l * R.mask_level]) ? kNegInf + 0.0f * a.s : to_f32(z[l]) - a.m - logs;
            O.logprob[r] = lp;
            O.entropy[r] = entropy_of(a, logs);
            if (O.stat) { O.stat[2 * r] = a.m; O.stat[2 * r + 1] = a.s; }
        }
        if (lane < O.top) {
            const bool some = list.v > kNegInf;
            O.top_logprob[r * O.top + lane] = some ? list.v - a.m - logs : (a.s == a.s ? kNegInf : a.s);
            O.top_level[r * O.top + lane] = some ? list.j : -1;
        }
    }
}

struct BackIn { const int64_t* level; const float* stat; const float* entropy; const float* g_lp; const float* g_h; int g_lp_stride, g_h_stride; };

template <class T>
__global__ __launch_bounds__(256) void score_backward_kernel(Rows R, BackIn I, T* grad) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < R.rows; r += (int64_t)gridDim.x * 4) {
        const T* z = (const T*)R.logits + row_base(R, r);
        const uint8_t* mk = row_mask(R, r);
        const float m = I.stat[2 * r], s = I.stat[2 * r + 1], H = I.entropy[r];
        const int64_t l = I.level[r];
        const float g = I.g_lp && l >= 0 ? I.g_lp[r * I.g_lp_stride] : 0.0f, gh = I.g_h ? I.g_h[r * I.g_h_stride] : 0.0f;
        const float logs = logf(s), inv = 1.0f / s;
        for (int j = lane; j < R.levels; j += 64) {
            const float v = mk && !mk[(int64_t)j * R.mask_level] ? kNegInf : to_f32(z[j]);
            float d = 0.0f;
            if (v != kNegInf && s != 0.0f) {
                const float e = fast_exp(v - m), p = e * inv;
                d = (j == l ? g : 0.0f) - p * (g + gh * (e > 0.0f ? v - m - logs + H : 0.0f));
                if (l >= R.levels) d = __builtin_nanf("");
            }
            grad[r * R.levels + j] = (T)d;
        }
    }
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
    return 0;
}

unsigned grid_for(int64_t rows) { const int64_t g = cdiv(rows, 4); return (unsigned)(g < 65536 ? g : 65536); }

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

int64_t lrn_choose_workspace(const lrn_rows*) { return 0; }

int lrn_choose(int32_t device, void* hip_stream, const lrn_rows* rows, const float* noise, int64_t noise_outer,
               int64_t noise_inner, int64_t* level_out, float* logprob_out, float* entropy_out, void*, int64_t) {
    Rows R;
    if (int rc = checked(rows, &R)) return rc;
    if (!R.rows) return 0;
    if (!level_out || !logprob_out || !entropy_out) return fail(-1, "lrn_choose: null output");
    LRN_ON_DEVICE(device);
    const ChooseOut O{noise, noise_outer, noise_inner, level_out, logprob_out, entropy_out};
    BY_TYPE(rows->dtype, (choose_kernel<T><<<grid_for(R.rows), 256, 0, (hipStream_t)hip_stream>>>(R, O)));
    LRN_LAUNCHED("lrn_choose");
    return 0;
}

int64_t lrn_score_workspace(const lrn_rows*, int32_t) { return 0; }

int lrn_score(int32_t device, void* hip_stream, const lrn_rows* rows, const int64_t* level, float* logprob_out,
              float* entropy_out, float* stat_out, int32_t top, float* top_logprob_out, int64_t* top_level_out, void*, int64_t) {
    Rows R;
    if (int rc = checked(rows, &R)) return rc;
    if (top < 0 || top > LRN_MAX_TOP || top > R.levels) return fail(-1, "lrn_score: top %d of %d levels (at most %d)", top, R.levels, LRN_MAX_TOP);
    if (!R.rows) return 0;
    if (!level || !logprob_out || !entropy_out || (top && (!top_logprob_out || !top_level_out))) return fail(-1, "lrn_score: null argument");
    LRN_ON_DEVICE(device);
    const ScoreOut O{level, logprob_out, entropy_out, stat_out, top, top_logprob_out, top_level_out};
    BY_TYPE(rows->dtype, (score_kernel<T><<<grid_for(R.rows), 256, 0, (hipStream_t)hip_stream>>>(R, O)));
    LRN_LAUNCHED("lrn_score");
    return 0;
}

int lrn_score_backward_needs_stat(const lrn_rows*) { return 1; }

int lrn_score_backward(int32_t device, void* hip_stream, const lrn_rows* rows, const int64_t* level, const float* stat,
                       const float* entropy, const float* g_logprob, int32_t g_logprob_stride, const float* g_entropy,
                       int32_t g_entropy_stride, void* grad_out) {
    Rows R;
    if (int rc = checked(rows, &R)) return rc;
    if (!R.rows) return 0;
    if (!level || !stat || !entropy || !grad_out) return fail(-1, "lrn_score_backward: null argument");
    if ((g_logprob_stride & ~1) || (g_entropy_stride & ~1)) return fail(-1, "lrn_score_backward: gradient strides are 0 or 1");
    LRN_ON_DEVICE(device);
    const BackIn I{level, stat, entropy, g_logprob, g_entropy, g_logprob_stride, g_entropy_stride};
    BY_TYPE(rows->dtype, (score_backward_kernel<T><<<grid_for(R.rows), 256, 0, (hipStream_t)hip_stream>>>(R, I, (T*)grad_out)));
    LRN_LAUNCHED("lrn_score_backward");
    return 0;
}

}  // extern "C"
