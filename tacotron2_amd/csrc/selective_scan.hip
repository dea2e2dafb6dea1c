// selective_scan.hip -- the selective state space recurrence on channels-last tensors (mv_selective_scan).
//
//   h[n] = exp(dt A[d, n]) h[n] + dt u B[g, n],   y = (sum_n C[g, n] h[n] + D u) z sigmoid(z)
#include "sequence.h"

namespace mv {

// log(1 + e^x).  log1p(e^-|x|) by its area tangent series: with s = e / (2 + e) <= 1/3, log1p(e) = 2 (s + s^3/3 + ...), so
// that small steps keep their relative precision (the next term is under 1e-8 of the sum).
__device__ __forceinline__ float softplusf(float x) {
    const float e = __builtin_amdgcn_exp2f(-kLog2e * fabsf(x));
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float p = 1.f / 15;
    p = p * q + 1.f / 13;
    p = p * q + 1.f / 11;
    p = p * q + 1.f / 9;
    p = p * q + 1.f / 7;
    p = p * q + 1.f / 5;
    p = p * q + 1.f / 3;
    return fmaxf(x, 0.f) + 2.f * s * (p * q + 1.f);
}

struct ScanParams {
    const float *A, *Dskip, *bias, *state_in;
    float* state_out;
    const int32_t* lengths;
    long long Bg, Cg;
    int B, T, D, N, G, softplus;
};

// One thread per channel of a sequence, its states in registers.
template <typename T>
__global__ __launch_bounds__(64) void scan_kernel(Rows<const T> u, Rows<const T> delta, Rows<const T> z, Rows<const T> Bm,
                                                  Rows<const T> Cm, Rows<T> y, ScanParams p) {
    const long long i = (long long)blockIdx.x * 64 + threadIdx.x;
    if (i >= (long long)p.B * p.D) return;
    const int b = (int)(i / p.D), d = (int)(i % p.D), g = d / (p.D / p.G), len = seq_frames(p.lengths, b, p.T);
    float h[64];
#pragma unroll
    for (int n = 0; n < 64; ++n) h[n] = n < p.N && p.state_in ? p.state_in[i * p.N + n] : 0.f;
    for (int t = 0; t < p.T; ++t) {
        float v = 0.f;
        if (t < len) {
            const float ut = (float)u.row(b, t)[d];
            float dt = (float)delta.row(b, t)[d] + (p.bias ? p.bias[d] : 0.f);
            if (p.softplus) dt = softplusf(dt);
            const T* Bt = Bm.row(b, t) + g * p.Bg;
            const T* Ct = Cm.row(b, t) + g * p.Cg;
#pragma unroll
            for (int n = 0; n < 64; ++n) {
                if (n < p.N) {
                    h[n] = __builtin_amdgcn_exp2f(dt * (p.A[d * p.N + n] * kLog2e)) * h[n] + dt * ut * (float)Bt[n];
                    v += (float)Ct[n] * h[n];
                }
            }
            if (p.Dskip) v += p.Dskip[d] * ut;
            if (z.p) {
                const float zt = (float)z.row(b, t)[d];
                v *= zt * sigmoidf(zt);
            }
        }
        y.row(b, t)[d] = (T)v;
    }
    if (p.state_out)
#pragma unroll
        for (int n = 0; n < 64; ++n)
            if (n < p.N) p.state_out[i * p.N + n] = h[n];
}

}  // namespace mv

using namespace mv;

static int check_scan(const mv_selective_scan_args* a) {
    const char* who = "mv_selective_scan";
    if (!a) {
        set_error("%s: null argument", who);
        return MV_EINVAL;
    }
    if (int rc = check_sequence(who, a->B, a->T, a->D, a->dtype)) return rc;
    if (a->N < 1 || a->N > 64 || a->G < 1 || a->D % a->G) {
        set_error("%s: %d states (1 to 64), or %d channels that do not split into %d groups", who, a->N, a->D, a->G);
        return MV_EINVAL;
    }
    return MV_OK;
}

extern "C" {

size_t mv_selective_scan_workspace(const mv_selective_scan_args* a) {
    if (check_scan(a)) return 0;
    return 0;
}

int mv_selective_scan(const mv_selective_scan_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "mv_selective_scan";
    if (int rc = check_scan(a)) return rc;
    const long long states = (long long)a->B * a->D * a->N;
    if (int rc = check_states(who, a->state_in, a->state_out, 4 * states)) return rc;
    if (a->B == 0) return MV_OK;
    if (a->T == 0) return carry_state(a->state_in, a->state_out, states, (hipStream_t)stream);
    if (!a->A) {
        set_error("%s: needs A", who);
        return MV_EINVAL;
    }
    const struct {
        const char* name;
        const mv_rows* r;
    } ins[] = {{"u", &a->u}, {"delta", &a->delta}, {"z", &a->z}, {"Bm", &a->Bm}, {"Cm", &a->Cm}};
    for (const auto& in : ins)
        if (in.r != &a->z || in.r->ptr)
            if (int rc = check_rows(who, in.name, *in.r, a->dtype)) return rc;
    if (int rc = check_output_rows(who, a->y, a->B, a->T, a->D, a->dtype)) return rc;
    ScanParams p{a->A, a->Dskip, a->delta_bias, a->state_in, a->state_out, a->lengths, (long long)a->Bg_stride,
                 (long long)a->Cg_stride, a->B, a->T, a->D, a->N, a->G, a->delta_softplus};
    return by_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        const long long n = (long long)a->B * a->D;
        hipLaunchKernelGGL((scan_kernel<T>), dim3((unsigned)((n + 63) / 64)), dim3(64), 0, (hipStream_t)stream,
                           rows_of<const T>(a->u), rows_of<const T>(a->delta), rows_of<const T>(a->z),
                           rows_of<const T>(a->Bm), rows_of<const T>(a->Cm), rows_of<T>(a->y), p);
        MV_HIP(hipGetLastError());
        return MV_OK;
    });
}

}  // extern "C"
