// group_norm.hip -- group normalisation with an activation on channels-last tensors (mv_group_norm).
//
//   y = act((x - m) / sqrt(v + eps) * w_c + b_c),  m and v over (t < len, c in group), or over a frame's group alone
//
// HBM-bound: x once in, y once out.
#include "sequence.h"

namespace mv {

int check_sequence(const char* who, int B, int T, int C, int dtype) {
    if (B < 0 || T < 0 || C < 1) {
        set_error("%s: bad sizes (B=%d, T=%d, channels=%d)", who, B, T, C);
        return MV_EINVAL;
    }
    if (dtype != MV_DTYPE_F32 && dtype != MV_DTYPE_BF16 && dtype != MV_DTYPE_F16) {
        set_error("%s: unknown dtype %d", who, dtype);
        return MV_EINVAL;
    }
    return MV_OK;
}

int check_rows(const char* who, const char* what, const mv_rows& r, int dtype) {
    if (!r.ptr || ((uintptr_t)r.ptr % dtype_size(dtype)) != 0 || r.batch_stride < 0 || r.row_stride < 0) {
        set_error("%s: %s needs an aligned pointer and strides >= 0", who, what);
        return MV_EINVAL;
    }
    return MV_OK;
}

// a state may be replaced in place, or by one that lies elsewhere
int check_states(const char* who, const void* in, const void* out, long long bytes) {
    const intptr_t d = (intptr_t)in - (intptr_t)out;
    if (in && out && in != out && (d < 0 ? -d : d) < bytes) {
        set_error("%s: state_in and state_out overlap without being the same", who);
        return MV_EINVAL;
    }
    return MV_OK;
}

int check_output_rows(const char* who, const mv_rows& r, int B, int T, int C, int dtype) {
    if (int rc = check_rows(who, "the output", r, dtype)) return rc;
    if (!rows_disjoint(r, B, T, C)) {
        set_error("%s: the output's rows overlap (batch_stride %lld, row_stride %lld)", who, (long long)r.batch_stride,
                  (long long)r.row_stride);
        return MV_EINVAL;
    }
    return MV_OK;
}

// One block per group of a sequence (or of a frame): mean, then the squared distances from it, then the result.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void group_norm_kernel(Rows<const T> x, Rows<T> y, const void* w, const void* bias,
                                                         bool w32, const int32_t* lengths, int Tmax, int C, int G,
                                                         int per_frame, float slope, float eps) {
    __shared__ float red[256];
    const int Cg = C / G;
    long long item = blockIdx.x;
    const int g = item % G;
    item /= G;
    int t0 = 0, t1 = Tmax;
    if (per_frame) {
        t0 = item % Tmax;
        t1 = t0 + 1;
        item /= Tmax;
    }
    const int b = (int)item, len = seq_frames(lengths, b, Tmax);
    const int c0 = g * Cg, end = min(t1, len);
    const long long n = (long long)max(0, end - t0) * Cg, all = (long long)(t1 - t0) * Cg;
    auto total = [&](float v) {
        red[threadIdx.x] = v;
        __syncthreads();
        for (int s = 128; s; s >>= 1) {
            if (threadIdx.x < s) red[threadIdx.x] += red[threadIdx.x + s];
            __syncthreads();
        }
        const float r = red[0];
        __syncthreads();
        return r;
    };
    float s = 0.f;
    for (long long i = threadIdx.x; i < n; i += 256) s += (float)x.row(b, t0 + (int)(i / Cg))[c0 + i % Cg];
    const float mean = total(s) / (float)n;
    s = 0.f;
    for (long long i = threadIdx.x; i < n; i += 256) {
        const float d = (float)x.row(b, t0 + (int)(i / Cg))[c0 + i % Cg] - mean;
        s += d * d;
    }
    const float r = 1.f / sqrtf(total(s) / (float)n + eps);
    for (long long i = threadIdx.x; i < all; i += 256) {
        const int c = c0 + (int)(i % Cg), t = t0 + (int)(i / Cg);
        float v = 0.f;
        if (i < n) {
            v = ((float)x.row(b, t)[c] - mean) * r;
            v = v * (w ? load_weight<T>(w, w32, c) : 1.f) + (bias ? load_weight<T>(bias, w32, c) : 0.f);
            v = activate<ACT>(v, slope);
        }
        y.row(b, t)[c] = (T)v;
    }
}

}  // namespace mv

using namespace mv;

static int check_group_norm(const mv_group_norm_args* a) {
    const char* who = "mv_group_norm";
    if (!a) {
        set_error("%s: null argument", who);
        return MV_EINVAL;
    }
    if (int rc = check_sequence(who, a->B, a->T, a->C, a->dtype)) return rc;
    if (a->groups < 1 || a->C % a->groups) {
        set_error("%s: %d channels do not split into %d groups", who, a->C, a->groups);
        return MV_EINVAL;
    }
    if (a->weight_dtype != MV_DTYPE_F32 && a->weight_dtype != a->dtype) {
        set_error("%s: weight_dtype must be MV_DTYPE_F32 or dtype", who);
        return MV_EINVAL;
    }
    if (a->activation < MV_ACT_NONE || a->activation > MV_ACT_TANH || !(a->eps >= 0.f) || a->eps > 3e38f) {
        set_error("%s: unknown activation %d or eps not in [0, inf)", who, a->activation);
        return MV_EINVAL;
    }
    return MV_OK;
}

extern "C" {

size_t mv_group_norm_workspace(const mv_group_norm_args* a) {
    if (check_group_norm(a)) return 0;
    return 0;
}

int mv_group_norm(const mv_group_norm_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_group_norm(a)) return rc;
    if (a->B == 0 || a->T == 0) return MV_OK;
    if (int rc = check_rows("mv_group_norm", "x", a->x, a->dtype)) return rc;
    if (int rc = check_output_rows("mv_group_norm", a->y, a->B, a->T, a->C, a->dtype)) return rc;
    const long long items = (long long)a->B * a->groups * (a->per_frame ? a->T : 1);
    if (items > 0xffffff) {
        set_error("mv_group_norm: too many groups");
        return MV_EINVAL;
    }
    return by_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return by_activation(a->activation, [&](auto act) {
            hipLaunchKernelGGL((group_norm_kernel<T, decltype(act)::value>), dim3((unsigned)items), dim3(256), 0,
                               (hipStream_t)stream, rows_of<const T>(a->x), rows_of<T>(a->y), a->weight, a->bias,
                               a->weight_dtype == MV_DTYPE_F32, a->lengths, a->T, a->C, a->groups, a->per_frame, a->slope,
                               a->eps);
            MV_HIP(hipGetLastError());
            return MV_OK;
        });
    });
}

}  // extern "C"
