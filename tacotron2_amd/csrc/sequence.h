// sequence.h -- what the sequence operators share (group_norm.hip, causal_conv.hip, selective_scan.hip): element types,
// activations, row addressing.  The operators work on channels-last tensors [B][T][C] whose channels are adjacent and
// whose rows and batches lie at any stride (mv_rows); arithmetic is float32, one rounding at the store.
#pragma once
#include "common.h"

namespace mv {

// one tensor of a launch: element (b, t, c) at ptr + b * bs + t * rs + c
template <typename T>
struct Rows {
    T* p;
    long long bs, rs;
    __device__ __forceinline__ T* row(int b, int t) const { return p + b * bs + t * rs; }
};
template <typename T>
inline Rows<T> rows_of(const mv_rows& r) {
    return Rows<T>{(T*)r.ptr, (long long)r.batch_stride, (long long)r.row_stride};
}

// a vector of N elements at any address an element may have (the hardware's vector loads and stores need no more)
template <typename T, int N>
struct Unaligned {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

// V channels at p, or the first `n` of them
template <typename T, int V>
__device__ __forceinline__ typename Unaligned<T, V>::type load_some(const T* p, int n) {
    typename Unaligned<T, V>::type v;
    if (n == V) return *(const typename Unaligned<T, V>::type*)p;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = e < n ? p[e] : (T)0.f;
    return v;
}
// `past`: past the L2, for results that it could not keep for their reader (pass_by_l2 below)
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, typename Unaligned<T, V>::type v, bool past) {
    typedef typename Unaligned<T, V>::type Vec;
    if (past) {
        // (the empty statements keep the compiler from making one ordinary store of the two branches)
        asm volatile("");
        __builtin_nontemporal_store(v, (Vec*)p);
        asm volatile("");
    } else {
        *(Vec*)p = v;
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_some(T* p, typename Unaligned<T, V>::type v, int n, bool past = false) {
    if (n == V) {
        store_vec<T, V>(p, v, past);
        return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (e < n) p[e] = v[e];
}

constexpr float kLog2e = 1.44269504088896341f;

// sigmoid and its relatives on the hardware exp2 and reciprocal (1 ulp each): exp2 overflowing to inf gives the right 0
__device__ __forceinline__ float sigmoidf(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * x));
}
// tanh: (1 - e) / (1 + e) with e = exp(-2|x|) loses x's low bits near 0, where the Taylor series to x^9 takes over
// (its next term is under 1e-8 of the result at 1/4)
__device__ __forceinline__ float tanh_accurate(float x) {
    const float a = fabsf(x);
    if (a < 0.25f) {
        const float q = x * x;
        return x * (1.f + q * (-1.f / 3 + q * (2.f / 15 + q * (-17.f / 315 + q * (62.f / 2835)))));
    }
    const float e = __builtin_amdgcn_exp2f(-2.f * kLog2e * a);
    return copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), x);
}

// the activations of mv_group_norm and mv_causal_conv; a NaN stays a NaN, relu (slope 0) takes -inf to 0
template <int ACT>
__device__ __forceinline__ float activate(float v, float slope) {
    if (ACT == MV_ACT_SILU) return v * sigmoidf(v);
    if (ACT == MV_ACT_LRELU) return v < 0.f ? (slope == 0.f ? 0.f : slope * v) : v;
    return tanh_accurate(v);
}

// weights are float32 or of the data's type
template <typename T>
__device__ __forceinline__ float load_weight(const void* w, bool w32, int i) {
    return w32 ? ((const float*)w)[i] : (float)((const T*)w)[i];
}

// calls f with a value of the element type / of an integral_constant for the activation
template <typename F>
inline int by_dtype(int dtype, F&& f) {
    switch (dtype) {
        case MV_DTYPE_F32: return f(float());
        case MV_DTYPE_BF16: return f(__bf16());
        case MV_DTYPE_F16: return f(_Float16());
    }
    set_error("unknown dtype %d", dtype);
    return MV_EINVAL;
}
// no activation is a leaky_relu of slope 1
template <typename F>
inline int by_activation(int act, float slope, float* use_slope, F&& f) {
    *use_slope = act == MV_ACT_NONE ? 1.f : slope;
    switch (act) {
        case MV_ACT_NONE:
        case MV_ACT_LRELU: return f(std::integral_constant<int, MV_ACT_LRELU>());
        case MV_ACT_SILU: return f(std::integral_constant<int, MV_ACT_SILU>());
        case MV_ACT_TANH: return f(std::integral_constant<int, MV_ACT_TANH>());
    }
    set_error("unknown activation %d", act);
    return MV_EINVAL;
}

inline size_t dtype_size(int dtype) { return dtype == MV_DTYPE_F32 ? 4 : 2; }

// Results leave past the L2 where a call's input and output are more than the L2s hold together (8 x 4 MB) and rows are whole
// 64-byte pieces: 512 channels, 32 utterances 15.1 -> 13.6 us, depthwise 1024 channels 22.6 -> 21.2, 128 channels of 16 x 55104
// rows 119 -> 105 (the next launch finds no dirty lines to wait for); rows that are not whole pieces pay for it (1023 float32
// channels 36.5 -> 38, 32-byte tiles 15 -> 28).
inline bool pass_by_l2(const mv_rows& y, int B, int T, int C, int dtype) {
    const int64_t row = (int64_t)C * (int64_t)dtype_size(dtype);
    auto whole = [&](int64_t bytes) { return bytes % 64 == 0; };
    return whole((int64_t)(uintptr_t)y.ptr) && whole(row) && whole(y.row_stride * (int64_t)dtype_size(dtype)) &&
           whole(y.batch_stride * (int64_t)dtype_size(dtype)) && 2 * row * B * T > 32ll << 20;
}

// rows of an output must not overlap: batches of rows, or rows of batches ([T][B][C] memory)
inline bool rows_disjoint(const mv_rows& r, int B, int T, int C) {
    const int64_t b = r.batch_stride, t = r.row_stride;
    return ((T < 2 || t >= C) && (B < 2 || b >= (T - 1) * t + C)) || ((B < 2 || b >= C) && (T < 2 || t >= (B - 1) * b + C));
}

// a call without frames: the sequences stand where they stood
template <typename T>
__global__ __launch_bounds__(256) void carry_state_kernel(const T* in, T* out, long long n) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256)
        out[i] = in ? in[i] : (T)0.f;
}
template <typename T>
inline int carry_state(const T* in, T* out, long long n, hipStream_t stream) {
    if (!out || in == out || n == 0) return MV_OK;
    const long long blocks = (n + 255) / 256;
    hipLaunchKernelGGL((carry_state_kernel<T>), dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, stream, in,
                       out, n);
    MV_HIP(hipGetLastError());
    return MV_OK;
}

// host-side checks shared by the operators; `who` is the entry point's name
int check_sequence(const char* who, int B, int T, int C, int dtype);
int check_aligned(const char* who, const void* p, size_t bytes);
int check_rows(const char* who, const char* what, const mv_rows& r, int T, int dtype);
int check_states(const char* who, const void* in, const void* out, long long bytes);
int check_output_rows(const char* who, const mv_rows& r, int B, int T, int C, int dtype);

// memory of a call: B x T rows of `width` bytes (of an axis of one the stride is 0)
struct Span {
    const char* p;
    long long width, bs, ts;
    int B, T;
    Span(const void* ptr, long long bytes) : p((const char*)ptr), width(bytes), bs(0), ts(0), B(1), T(1) {}
    Span(const mv_rows& r, long long channels, int B_, int T_, int dtype)
        : p((const char*)r.ptr), width(channels * (long long)dtype_size(dtype)),
          bs(B_ > 1 ? (r.batch_stride < 1ll << 56 ? r.batch_stride : 1ll << 56) * (long long)dtype_size(dtype) : 0),
          ts(T_ > 1 ? r.row_stride * (long long)dtype_size(dtype) : 0), B(B_), T(T_) {}
};
int check_overlaps(const char* who, const Span& output, const char* what, std::initializer_list<Span> inputs);

}  // namespace mv
