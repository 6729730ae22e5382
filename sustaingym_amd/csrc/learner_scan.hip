// learner_scan.hip — gfx950 kernels of lrn_scan / lrn_scan_backward / lrn_advantages (include/learner_ops.h).
//
// All three are h_u = a_u h_{u-1} + x_u along an order u of the steps; what differs is what x, a and the outputs are:
//   scan       u runs with the sequence, x and a are read
//   backward   u runs against it: x_u = g_h, a_u = the gate of the step before in this order (1 in front of the first, so
//              that g_final enters as the state), and beside h = grad_x comes grad_gate = h * (the state before the step)
//   advantages u runs against time: x_u = d_t, a_u = gamma lam (1 - end_t), and beside h comes h + V_t
// The state is float32 (float64 for float64 sequences) in a register whatever the type of the elements.
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
    const float* last;          // advantages: V behind the last step
    const void* values;         // advantages (with View before = values)
    void* final;
};

enum Kind { SCAN, BACKWARD, ADVANTAGES };

template <class T> struct State { using type = float; };
template <> struct State<double> { using type = double; };

template <class T> __device__ __forceinline__ T* at(const View& v, int64_t u, int64_t b, int64_t c) {
    return (T*)v.p + u * v.st + b * v.sb + c * v.sc;
}

// One thread walks one column.
template <Kind K, class T>
__global__ __launch_bounds__(256) void walk_kernel(Seq S) {
    using W = typename State<T>::type;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < S.cols; q += (int64_t)gridDim.x * 256) {
        const int64_t b = q / S.channels, c = q % S.channels;
        W h = S.initial ? ((const W*)S.initial)[q] : W(0);
        if constexpr (K == ADVANTAGES) h = W(0);
        W a_next = W(1);                    // BACKWARD: the gate in front of the first step of this order
        float v_next = K == ADVANTAGES ? S.last[q] : 0.0f;
        for (int64_t u = 0; u < S.steps; u++) {
            if constexpr (K == SCAN) {
                W a = S.gate.p ? (W)*at<const T>(S.gate, u, b, c) : (W)S.gate_const;
                const bool anew = S.resets.p && *at<const uint8_t>(S.resets, u, b, 0);
                const W x = (W)*at<const T>(S.x, u, b, c);
                h = anew ? x : a * h + x;
                *at<T>(S.h, u, b, c) = (T)h;
            } else if constexpr (K == BACKWARD) {
                const W g = S.x.p ? (W)*at<const T>(S.x, u, b, c) : W(0);
                h = a_next == W(0) ? g : a_next * h + g;
                if (S.h.p) *at<T>(S.h, u, b, c) = (T)h;
                const bool anew = S.resets.p && *at<const uint8_t>(S.resets, u, b, 0);
                if (S.gate_out.p) {
                    W prev = W(0);
                    if (u + 1 < S.steps) prev = (W)*at<const T>(S.before, u + 1, b, c);
                    else if (S.last) prev = ((const W*)S.last)[q];
                    *at<T>(S.gate_out, u, b, c) = (T)(anew ? W(0) : h * prev);
                }
                a_next = anew ? W(0) : S.gate.p ? (W)*at<const T>(S.gate, u, b, c) : (W)S.gate_const;
            } else {
                const float v = *at<const float>(S.before, u, b, c);
                const bool end = *at<const uint8_t>(S.resets, u, b, 0);
                const W r = (W)*at<const T>(S.x, u, b, c);
                const W d = end ? r - (W)v : r + (W)S.scale * (W)v_next - (W)v;
                h = end ? d : (W)S.gate_const * h + d;
                *at<float>(S.h, u, b, c) = (float)h;
                *at<float>(S.gate_out, u, b, c) = (float)(h + (W)v);
                v_next = v;
            }
        }
        if (S.final) ((W*)S.final)[q] = K == BACKWARD ? (a_next == W(0) ? W(0) : a_next * h) : h;
    }
}

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

template <Kind K, class T> void launch(const Seq& S, hipStream_t stream) {
    const int64_t g = cdiv(S.cols, 256);
    walk_kernel<K, T><<<(unsigned)(g < 65536 ? g : 65536), 256, 0, stream>>>(S);
}

template <Kind K> int run(const Seq& S, int dtype, hipStream_t stream, const char* who) {
    if (dtype == LRN_F32) launch<K, float>(S, stream);
    else if (dtype == LRN_F64) launch<K, double>(S, stream);
    else if constexpr (K != ADVANTAGES) {
        if (dtype == LRN_BF16) launch<K, bf16>(S, stream);
        else launch<K, f16>(S, stream);
    }
    LRN_LAUNCHED(who);
    return 0;
}

}  // namespace
}  // namespace lrn

using namespace lrn;

extern "C" {

int64_t lrn_scan_workspace(const lrn_seq*) { return 0; }

int lrn_scan(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* x, const lrn_view* gate,
             double gate_const, const lrn_view* resets, const void* initial, const lrn_view* h_out, void* final_out, void*, int64_t) {
    if (int rc = checked(seq, "lrn_scan")) return rc;
    if (seq->batch * seq->channels == 0) return 0;
    if (seq->steps && (!x || !x->data || !h_out || !h_out->data)) return fail(-1, "lrn_scan: null x or h");
    LRN_ON_DEVICE(device);
    const bool rev = seq->reverse != 0;
    const int64_t n = bytes_of(seq->dtype);
    Seq S{};
    S.steps = seq->steps; S.cols = seq->batch * seq->channels; S.channels = seq->channels;
    S.x = ordered(x, seq->steps, n, rev); S.gate = ordered(gate, seq->steps, n, rev);
    S.resets = ordered(resets, seq->steps, 1, rev); S.h = ordered(h_out, seq->steps, n, rev);
    S.gate_const = gate_const; S.initial = initial; S.final = final_out;
    return run<SCAN>(S, seq->dtype, (hipStream_t)hip_stream, "lrn_scan");
}

int lrn_scan_backward(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* gate, double gate_const,
                      const lrn_view* resets, const void* initial, const lrn_view* h, const lrn_view* g_h,
                      const void* g_final, const lrn_view* grad_x_out, const lrn_view* grad_gate_out,
                      void* grad_initial_out, void*, int64_t) {
    if (int rc = checked(seq, "lrn_scan_backward")) return rc;
    if (seq->batch * seq->channels == 0) return 0;
    if (grad_gate_out && grad_gate_out->data && seq->steps && (!h || !h->data)) return fail(-1, "lrn_scan_backward: null h");
    LRN_ON_DEVICE(device);
    const bool rev = seq->reverse == 0;
    const int64_t n = bytes_of(seq->dtype);
    Seq S{};
    S.steps = seq->steps; S.cols = seq->batch * seq->channels; S.channels = seq->channels;
    S.x = ordered(g_h, seq->steps, n, rev); S.gate = ordered(gate, seq->steps, n, rev);
    S.resets = ordered(resets, seq->steps, 1, rev); S.before = ordered(h, seq->steps, n, rev);
    S.h = ordered(grad_x_out, seq->steps, n, rev); S.gate_out = ordered(grad_gate_out, seq->steps, n, rev);
    S.gate_const = gate_const; S.initial = g_final; S.last = (const float*)initial; S.final = grad_initial_out;
    return run<BACKWARD>(S, seq->dtype, (hipStream_t)hip_stream, "lrn_scan_backward");
}

int64_t lrn_advantages_workspace(const lrn_seq*) { return 0; }

int lrn_advantages(int32_t device, void* hip_stream, const lrn_seq* seq, const lrn_view* rewards, const lrn_view* values,
                   const lrn_view* ends, const float* last_values, double gamma, double lam, float* advantage_out,
                   float* target_out, void*, int64_t) {
    if (int rc = checked(seq, "lrn_advantages")) return rc;
    if (seq->channels != 1) return fail(-1, "lrn_advantages: %lld channels", (long long)seq->channels);
    if (seq->dtype != LRN_F32 && seq->dtype != LRN_F64) return fail(-1, "lrn_advantages: dtype %d", seq->dtype);
    if (seq->batch == 0 || seq->steps == 0) return 0;
    if (!rewards || !rewards->data || !values || !values->data || !ends || !ends->data || !last_values || !advantage_out || !target_out)
        return fail(-1, "lrn_advantages: null argument");
    LRN_ON_DEVICE(device);
    const lrn_view adv{advantage_out, seq->batch, 1, 0}, tgt{target_out, seq->batch, 1, 0};
    Seq S{};
    S.steps = seq->steps; S.cols = seq->batch; S.channels = 1;
    S.x = ordered(rewards, seq->steps, bytes_of(seq->dtype), true); S.before = ordered(values, seq->steps, 4, true);
    S.resets = ordered(ends, seq->steps, 1, true);
    S.h = ordered(&adv, seq->steps, 4, true); S.gate_out = ordered(&tgt, seq->steps, 4, true);
    S.gate_const = gamma * lam; S.scale = gamma; S.last = last_values;
    return run<ADVANTAGES>(S, seq->dtype, (hipStream_t)hip_stream, "lrn_advantages");
}

}  // extern "C"
