// causal_conv.hip -- short depthwise causal convolution with an activation on channels-last tensors (mv_causal_conv).
//
//   y[t, c] = act(bias_c + sum_k w[c, k] x[t - K + 1 + k, c]),  frames before the first from the state
//
// HBM-bound: x once in, y once out.
#include "sequence.h"

namespace mv {

// One thread per channel of a sequence, walking its frames: the state is read before it is replaced by the same thread.
template <typename T, int ACT, int K>
__global__ __launch_bounds__(256) void causal_conv_kernel(Rows<const T> x, Rows<T> y, const void* w, const void* bias,
                                                          bool w32, const T* state_in, T* state_out,
                                                          const int32_t* lengths, int B, int Tmax, int C, float slope) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)B * C) return;
    const int b = (int)(i / C), c = (int)(i % C), len = seq_frames(lengths, b, Tmax);
    float win[K], wk[K];
    for (int k = 0; k < K; ++k) {
        wk[k] = load_weight<T>(w, w32, c * K + k);
        win[k] = k && state_in ? (float)state_in[((long long)b * (K - 1) + k - 1) * C + c] : 0.f;
    }
    const float bc = bias ? load_weight<T>(bias, w32, c) : 0.f;
    for (int t = 0; t < Tmax; ++t) {
        float v = 0.f;
        if (t < len) {
            for (int k = 0; k + 1 < K; ++k) win[k] = win[k + 1];
            win[K - 1] = (float)x.row(b, t)[c];
            v = bc;
            for (int k = 0; k < K; ++k) v += wk[k] * win[k];
            v = activate<ACT>(v, slope);
        }
        y.row(b, t)[c] = (T)v;
    }
    if (state_out)
        for (int k = 1; k < K; ++k) state_out[((long long)b * (K - 1) + k - 1) * C + c] = (T)win[k];
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
    if (a->K < 1 || a->K > 8) {
        set_error("%s: %d taps (1 to 8)", who, a->K);
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
    const long long states = (long long)a->B * (a->K - 1) * a->C;
    if (int rc = check_states(who, a->state_in, a->state_out, states * (long long)dtype_size(a->dtype))) return rc;
    if (a->B == 0) return MV_OK;
    if (a->T == 0)
        return by_dtype(a->dtype, [&](auto t) {
            using T = decltype(t);
            return carry_state((const T*)a->state_in, (T*)a->state_out, states, (hipStream_t)stream);
        });
    if (int rc = check_rows(who, "x", a->x, a->dtype)) return rc;
    if (int rc = check_output_rows(who, a->y, a->B, a->T, a->C, a->dtype)) return rc;
    return by_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return by_activation(a->activation, [&](auto act) {
            return by_taps(a->K, [&](auto taps) {
                const long long n = (long long)a->B * a->C;
                hipLaunchKernelGGL((causal_conv_kernel<T, decltype(act)::value, decltype(taps)::value>),
                                   dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                                   rows_of<const T>(a->x), rows_of<T>(a->y), a->weight, a->bias,
                                   a->weight_dtype == MV_DTYPE_F32, (const T*)a->state_in, (T*)a->state_out, a->lengths,
                                   a->B, a->T, a->C, a->slope);
                MV_HIP(hipGetLastError());
                return MV_OK;
            });
        });
    });
}
