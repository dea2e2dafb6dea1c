// causal_conv.hip -- short depthwise causal convolution with an activation on channels-last tensors (mv_causal_conv).
//
//   y[t, c] = act(bias_c + sum_k w[c, k] x[t - K + 1 + k, c]),  frames before the first from the state
//
// HBM-bound: x once in, y once out; a few kilobytes are bound by the launch.  A thread holds 16 bytes of adjacent channels (the
// widest load) and walks along time, so a frame comes in once per run and its K uses are registers; the activation's exponential
// and reciprocal hide behind the loads.  4 taps, SiLU, bf16: 32 x 861 x 512 16 us (3.5 TB/s), 16 x 8192 x 512 57 us (4.7 TB/s),
// 4 x 16384 x 4096 202 us (5.3 TB/s; a large copy reaches 5.0).
#include "sequence.h"

namespace mv {

template <typename T>
struct CausalParams {
    Rows<const T> x;
    Rows<T> y;
    const void *w, *bias;
    const T* state_in;
    T* state_out;
    const int32_t* lengths;
    int B, Tmax, C, w32;
    float slope;
    unsigned vecs, runs;
    int run, past;  // vectors of a row, threads to a sequence's vector, frames each walks; results past the L2
};

// frames whose loads are in flight together (more taps leave registers for fewer)
template <int K>
constexpr int kConvStep = K <= 4 ? 8 : 4;

// A thread walks `run` frames of V adjacent channels with the K - 1 frames before in registers.  The thread of a sequence's
// first run also moves the state on: it alone reads state_in, before it writes state_out.
template <typename T, int ACT, int K, int V>
__global__ __launch_bounds__(256) void causal_conv_kernel(CausalParams<T> p) {
    typedef typename Unaligned<T, V>::type Vec;
    constexpr int kStep = kConvStep<K>;
    const unsigned id = blockIdx.x * 256 + threadIdx.x, rest = id / p.vecs;
    const int cv = id % p.vecs, r = p.runs == 1 ? 0 : rest % p.runs, b = p.runs == 1 ? rest : rest / p.runs;
    if (b >= p.B) return;
    // The last vector of a row whose channels are no multiple of V reaches back over its neighbour's and writes what that one
    // writes; where the state is moved on, one thread alone may read a channel's and write it, and it has what is left.
    const bool back = cv * V + V > p.C && p.C >= V && !(r == 0 && p.state_out);
    const int c = back ? p.C - V : cv * V, n = min(V, p.C - c), len = seq_frames(p.lengths, b, p.Tmax);
    const int t0 = r * p.run, t1 = min(t0 + p.run, p.Tmax);
    const T* from = p.x.row(b, 0) + c;
    T* to = p.y.row(b, 0) + c;

    Vec carry[K];  // (K - 1 of them)
    if (K > 1 && r == 0) {
        const long long s = (long long)b * (K - 1) * p.C + c;
#pragma unroll
        for (int k = 0; k + 1 < K; ++k) {
            if (p.state_in) {
                carry[k] = load_some<T, V>(p.state_in + s + (long long)k * p.C, n);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) carry[k][e] = (T)0.f;
            }
        }
        if (p.state_out) {
            Vec next[K];
#pragma unroll
            for (int k = 0; k + 1 < K; ++k) {
                const int at = len + k - (K - 1);  // frame that becomes row k, or a row of the state before
                if (at >= 0) {
                    next[k] = load_some<T, V>(from + at * p.x.rs, n);
                } else {
                    next[k] = carry[k];
#pragma unroll
                    for (int q = 1; q + k < K - 1; ++q)
                        if (len == q) next[k] = carry[k + q];
                }
            }
#pragma unroll
            for (int k = 0; k + 1 < K; ++k) store_some<T, V>(p.state_out + s + (long long)k * p.C, next[k], n);
        }
    } else if (K > 1 && t0 < len) {
#pragma unroll
        for (int k = 0; k + 1 < K; ++k) {
            // (a run is no shorter than K - 1 frames unless it is the only one: t0 - (K - 1) >= 0)
            carry[k] = load_some<T, V>(from + (t0 - (K - 1) + k) * p.x.rs, n);
        }
    }

    float w[K * V], bias[V];
    if (t0 < len) {
        // a vector's taps lie side by side: [channel][K]
        if (n == V) {
#pragma unroll
            for (int i = 0; i < K; ++i) {
                if (p.w32) {
                    const auto t = *(const typename Unaligned<float, V>::type*)((const float*)p.w + c * K + i * V);
#pragma unroll
                    for (int e = 0; e < V; ++e) w[i * V + e] = t[e];
                } else {
                    const auto t = *(const Vec*)((const T*)p.w + c * K + i * V);
#pragma unroll
                    for (int e = 0; e < V; ++e) w[i * V + e] = (float)t[e];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < K * V; ++i) w[i] = i < n * K ? load_weight<T>(p.w, p.w32, c * K + i) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) bias[e] = p.bias && e < n ? load_weight<T>(p.bias, p.w32, c + e) : 0.f;
    }
    float x[K - 1 + kStep][V];
#pragma unroll
    for (int k = 0; k + 1 < K; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) x[k][e] = (float)carry[k][e];
    const int live = min(t1, len);
    int t = t0;
    for (; t < live; t += kStep) {
        Vec raw[kStep];
#pragma unroll
        for (int u = 0; u < kStep; ++u)
            if (t + u < live) raw[u] = load_some<T, V>(from + (t + u) * p.x.rs, n);
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
            if (t + u >= live) break;
            Vec y;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x[K - 1 + u][e] = (float)raw[u][e];
                float v = bias[e];
#pragma unroll
                for (int k = 0; k < K; ++k) v += w[e * K + k] * x[u + k][e];
                y[e] = (T)activate<ACT>(v, p.slope);
            }
            store_some<T, V>(to + (t + u) * p.y.rs, y, n, p.past);
        }
#pragma unroll
        for (int k = 0; k + 1 < K; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) x[k][e] = x[k + kStep][e];
    }
    Vec zero;
#pragma unroll
    for (int e = 0; e < V; ++e) zero[e] = (T)0.f;
    for (t = max(t0, len); t < t1; ++t) store_some<T, V>(to + t * p.y.rs, zero, n, p.past);
}

template <typename F>
static int by_taps(int K, F&& f) {
    switch (K) {
        case 1: return f(std::integral_constant<int, 1>());
        case 2: return f(std::integral_constant<int, 2>());
        case 3: return f(std::integral_constant<int, 3>());
        case 4: return f(std::integral_constant<int, 4>());
        case 5: return f(std::integral_constant<int, 5>());
        case 6: return f(std::integral_constant<int, 6>());
        case 7: return f(std::integral_constant<int, 7>());
        default: return f(std::integral_constant<int, 8>());
    }
}

}  // namespace mv

using namespace mv;

extern "C" int mv_causal_conv(const mv_causal_conv_args* a, void* stream) {
    const char* who = "mv_causal_conv";
    if (!a) {
        set_error("%s: null argument", who);
        return MV_EINVAL;
    }
    if (int rc = check_sequence(who, a->B, a->T, a->C, a->dtype)) return rc;
    if (a->K < 1 || a->K > 8 || a->C > 1 << 27) {
        set_error("%s: %d taps (1 to 8), or more than 2^27 channels", who, a->K);
        return MV_EINVAL;
    }
    if (!a->weight || (a->weight_dtype != MV_DTYPE_F32 && a->weight_dtype != a->dtype)) {
        set_error("%s: needs a weight, of MV_DTYPE_F32 or dtype", who);
        return MV_EINVAL;
    }
    if (a->activation < MV_ACT_NONE || a->activation > MV_ACT_TANH) {
        set_error("%s: unknown activation %d", who, a->activation);
        return MV_EINVAL;
    }
    const size_t size = dtype_size(a->dtype), wsize = dtype_size(a->weight_dtype);
    for (auto [p, bytes] : {std::pair<const void*, size_t>{a->weight, wsize}, {a->bias, wsize}, {a->state_in, size},
                            {a->state_out, size}, {a->lengths, 4}})
        if (int rc = check_aligned(who, p, bytes)) return rc;
    const long long states = (long long)a->B * (a->K - 1) * a->C;
    if (int rc = check_states(who, a->state_in, a->state_out, states * (long long)dtype_size(a->dtype))) return rc;
    if (a->B == 0) return MV_OK;
    if (a->T == 0)
        return by_dtype(a->dtype, [&](auto t) {
            using T = decltype(t);
            return carry_state((const T*)a->state_in, (T*)a->state_out, states, (hipStream_t)stream);
        });
    if (int rc = check_rows(who, "x", a->x, a->T, a->dtype)) return rc;
    if (int rc = check_output_rows(who, a->y, a->B, a->T, a->C, a->dtype)) return rc;
    const Span x(a->x, a->C, a->B, a->T, a->dtype), w(a->weight, (long long)a->C * a->K * wsize), bias(a->bias, a->C * (long long)wsize),
        lengths(a->lengths, 4ll * a->B), before(a->state_in, states * (long long)size), after(a->state_out, states * (long long)size);
    if (int rc = check_overlaps(who, Span(a->y, a->C, a->B, a->T, a->dtype), "y", {x, w, bias, lengths, before, after})) return rc;
    if (int rc = check_overlaps(who, after, "state_out", {x, w, bias, lengths})) return rc;
    return by_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int V = 16 / sizeof(T);
        CausalParams<T> p{rows_of<const T>(a->x), rows_of<T>(a->y), a->weight, a->bias, (const T*)a->state_in, (T*)a->state_out,
                        a->lengths, a->B, a->T, a->C, a->weight_dtype == MV_DTYPE_F32, 0.f, (unsigned)(a->C + V - 1) / V, 0, 0, pass_by_l2(a->y, a->B, a->T, a->C, a->dtype)};
        // A run reads K - 1 frames that the one before reads too: runs of 32 frames, halved (to 8) until there are 2^17
        // threads (1 x 861 x 512: 8.0 us with runs of 8, 13.7 with 32).  Two taps, or up to four where the frames read twice
        // are in the block's own cache (up to 16 vectors a row) or weigh little (float32), gain more from threads: runs of 8
        // (4 taps, runs of 8 / 32: bf16 8 x 30000 x 128 26 / 33 us, float32 16 x 8192 x 512 93 / 103, 2 taps bf16 the same
        // 48 / 54; but 4 taps bf16 8 x 8192 x 1023 63 / 53, 8 taps float32 16 x 8192 x 512 171 / 143).
        const bool short_runs = a->K <= 2 || (a->K <= 4 && (sizeof(T) == 4 || p.vecs <= 16));
        for (p.run = short_runs ? 8 : 32; p.run > 8 && (long long)a->B * ((a->T + p.run - 1) / p.run) * p.vecs < 1 << 17;)
            p.run /= 2;
        p.runs = (a->T + p.run - 1) / p.run;
        const long long blocks = ((long long)a->B * p.runs * p.vecs + 255) / 256;
        if (blocks > 0x7fffff) {
            set_error("%s: too many frames for one call", who);
            return MV_EINVAL;
        }
        return by_activation(a->activation, a->slope, &p.slope, [&](auto act) {
            return by_taps(a->K, [&](auto taps) {
                hipLaunchKernelGGL((causal_conv_kernel<T, decltype(act)::value, decltype(taps)::value, V>),
                                   dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p);
                MV_HIP(hipGetLastError());
                return MV_OK;
            });
        });
    });
}
