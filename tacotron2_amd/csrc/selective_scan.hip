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

constexpr int kLanes = 4;   // lanes that share a channel: lane 4c + j holds states j * NS ... of channel c
constexpr int kTile = 32;   // frames whose B and C rows are in LDS at a time
constexpr int kBlockChannels = 64;  // 4 waves of 16 channels

template <typename T>
struct ScanParams {
    Rows<const T> u, delta, z, Bm, Cm;
    Rows<T> y;
    const float *A, *Dskip, *bias, *state_in;
    float* state_out;
    const int32_t* lengths;
    long long Bg, Cg;
    float *ws_h, *ws_s;  // pieces' states from zero [B][pieces - 1][D][4 * NS] and sums of dt [B][pieces - 1][D]
    int B, Tmax, D, N, G, softplus;
    int blocks_per_group, piece, pieces;  // frames to a piece (a multiple of kTile), number of pieces
};

template <int CTRL>
__device__ __forceinline__ float quad(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int K>
__device__ __forceinline__ float quad_lane(float v) {
    return quad<K * 0x55>(v);
}

// Lane j's NS of the N values at p, as floats; zeros where it has fewer.
template <typename T, int NS>
__device__ __forceinline__ void load_my_states(const T* p, int N, int j, float (&v)[NS]) {
    if (N == kLanes * NS) {
        typedef typename Unaligned<T, NS>::type V;
        const V t = *(const V*)(p + j * NS);
#pragma unroll
        for (int s = 0; s < NS; ++s) v[s] = (float)t[s];
    } else {
#pragma unroll
        for (int s = 0; s < NS; ++s) v[s] = j * NS + s < N ? (float)p[j * NS + s] : 0.f;
    }
}

// The calling thread's channel and states.
template <typename T, int NS>
struct Channel {
    int b, g, d, j, len;
    bool live;   // false: a lane past the group's last channel, which computes on the last one and stores nothing
    float A2[NS];

    __device__ __forceinline__ void init(const ScanParams<T>& p, int b_, int g_, int c) {
        const int Dg = p.D / p.G;
        b = b_, g = g_, j = threadIdx.x & (kLanes - 1);
        live = c < Dg;
        d = g * Dg + min(c, Dg - 1);
        len = seq_frames(p.lengths, b, p.Tmax);
        load_my_states(p.A + (long long)d * p.N, p.N, j, A2);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            // clamped to finite: 0 * inf must not make a NaN of a frame past the end, whose dt is 0
            const float a = A2[s] * kLog2e;
            A2[s] = a < -3e38f ? -3e38f : (a > 3e38f ? 3e38f : a);
        }
    }
    __device__ __forceinline__ void load_state(const ScanParams<T>& p, float (&h)[NS]) const {
        if (p.state_in) {
            load_my_states(p.state_in + ((long long)b * p.D + d) * p.N, p.N, j, h);
        } else {
#pragma unroll
            for (int s = 0; s < NS; ++s) h[s] = 0.f;
        }
    }
    __device__ __forceinline__ void store_state(const ScanParams<T>& p, const float (&h)[NS]) const {
        if (!p.state_out || !live) return;
        float* to = p.state_out + ((long long)b * p.D + d) * p.N;
        if (p.N == kLanes * NS) {
            typedef typename Unaligned<float, NS>::type V;
            V v;
#pragma unroll
            for (int s = 0; s < NS; ++s) v[s] = h[s];
            *(V*)(to + j * NS) = v;
        } else {
#pragma unroll
            for (int s = 0; s < NS; ++s)
                if (j * NS + s < p.N) to[j * NS + s] = h[s];
        }
    }
};

template <int NS>
__device__ __forceinline__ void load_states(const float* p, float (&v)[NS]) {
    if constexpr (NS % 4 == 0) {
#pragma unroll
        for (int s = 0; s < NS; s += 4) *(f32x4*)&v[s] = *(const f32x4*)&p[s];
    } else if constexpr (NS == 2) {
        const float2 t = *(const float2*)p;
        v[0] = t.x, v[1] = t.y;
    } else {
        v[0] = p[0];
    }
}

// One of u, delta, z, y as a channel block walks it: 16 frames at a time, lane j of a channel on frames j, j + 4, j + 8, j + 12
// of them.  The address of a frame is a base that all lanes share (scalar arithmetic) plus an offset that a lane keeps.
template <typename T>
struct Walk {
    T* p;             // channel 0 of frame 0 of the sequence
    long long rs;
    unsigned lane;    // bytes
    __device__ __forceinline__ Walk(const Rows<T>& r, int b, int d, int j)
        : p(r.p ? r.row(b, 0) : nullptr), rs(r.rs), lane((unsigned)(j * r.rs + d) * (unsigned)sizeof(T)) {}
    __device__ __forceinline__ T* at(int t, int i) const { return (T*)((char*)(p + (t + 4 * i) * rs) + lane); }
    // the same with frames from `end` on replaced by frame end - 1
    __device__ __forceinline__ T* at_or_last(int t, int i, int end, int j) const {
        const int r = min(4 * i + j, end - 1 - t) - j;
        return (T*)((char*)(p + t * rs) + (long long)(r * (int)rs) * (int)sizeof(T) + lane);
    }
};

// Frames [t0, t1) of one channel block: h goes from the state before t0 to the state after t1 - 1.  Y: results are stored;
// otherwise only the states move, and the sum of dt is returned.
template <typename T, int NS, bool Y>
__device__ __forceinline__ float scan_frames(const ScanParams<T>& p, const Channel<T, NS>& ch, int t0, int t1, float (&h)[NS],
                                             float* lds) {
    constexpr int NP = kLanes * NS, kMine = kTile * NP / 256 > 0 ? kTile * NP / 256 : 1;
    const int tid = threadIdx.x;
    const float bias = p.bias ? p.bias[ch.d] : 0.f, skip = p.Dskip ? p.Dskip[ch.d] : 0.f;
    const Walk<const T> uw(p.u, ch.b, ch.d, ch.j), dw(p.delta, ch.b, ch.d, ch.j), zw(p.z, ch.b, ch.d, ch.j);
    const Walk<T> yw(p.y, ch.b, ch.d, ch.j);
    const T* Bb = p.Bm.row(ch.b, 0) + ch.g * p.Bg;
    const T* Cb = p.Cm.row(ch.b, 0) + ch.g * p.Cg;
    float sum = 0.f;

    // B and C rows of the next tile on their way to LDS, u, delta and z of the next 16 frames on their way to the lanes;
    // a frame past t1 reads frame t1 - 1 and is replaced by zeros, which leave the state as it is (dt = 0)
    T nb[kMine], nc[kMine], nu[4], nd[4], nz[4];
    auto fetch_maps = [&](int t) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int e = tid + 256 * i, n = min(e % NP, p.N - 1);
            const long long r = min(t + e / NP % kTile, t1 - 1);
            nb[i] = Bb[r * p.Bm.rs + n];
            if (Y) nc[i] = Cb[r * p.Cm.rs + n];
        }
    };
    auto put_maps = [&](int t, float* to) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int e = tid + 256 * i;
            const bool in = e % NP < p.N && t + e / NP < t1;
            if (e < kTile * NP) {
                to[e] = in ? (float)nb[i] : 0.f;
                if (Y) to[kTile * NP + e] = in ? (float)nc[i] : 0.f;
            }
        }
    };
    auto fetch_frames = [&](int t) {
        const bool whole = t + 16 <= t1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            nu[i] = *(whole ? uw.at(t, i) : uw.at_or_last(t, i, t1, ch.j));
            nd[i] = *(whole ? dw.at(t, i) : dw.at_or_last(t, i, t1, ch.j));
        }
        if (Y && zw.p) {
#pragma unroll
            for (int i = 0; i < 4; ++i) nz[i] = *(whole ? zw.at(t, i) : zw.at_or_last(t, i, t1, ch.j));
        }
    };
    fetch_maps(t0);
    fetch_frames(t0);
    int buf = 0;
    for (int t = t0; t < t1; t += kTile, buf ^= 1) {
        float* maps = lds + buf * 2 * kTile * NP;
        put_maps(t, maps);
        __syncthreads();
        if (t + kTile < t1) fetch_maps(t + kTile);
#pragma unroll 1
        for (int q = 0; q < kTile && t + q < t1; q += 16) {
            const bool whole = t + q + 16 <= t1;
            float uv[4], dv[4], xv[4], zv[4], yv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uv[i] = (float)nu[i];
                dv[i] = (float)nd[i] + bias;
                if (Y && zw.p) zv[i] = (float)nz[i];
            }
            if (t + q + 16 < t1) fetch_frames(t + q + 16);
            if (p.softplus) {
#pragma unroll
                for (int i = 0; i < 4; ++i) dv[i] = softplusf(dv[i]);
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t + q + 4 * i + ch.j >= t1) uv[i] = dv[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                xv[i] = dv[i] * uv[i];
                if (!Y) sum += dv[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float out[4];
                auto frame = [&](auto k) {
                    constexpr int K = decltype(k)::value;
                    const float dt = quad_lane<K>(dv[i]), x = quad_lane<K>(xv[i]);
                    const float* row = maps + (q + 4 * i + K) * NP + ch.j * NS;
                    float bn[NS], cn[NS], o = 0.f;
                    load_states<NS>(row, bn);
                    if (Y) load_states<NS>(row + kTile * NP, cn);
#pragma unroll
                    for (int s = 0; s < NS; ++s) {
                        h[s] = __builtin_amdgcn_exp2f(dt * ch.A2[s]) * h[s] + x * bn[s];
                        if (Y) o = s ? o + cn[s] * h[s] : cn[s] * h[s];
                    }
                    out[K] = o;
                };
                frame(std::integral_constant<int, 0>());
                frame(std::integral_constant<int, 1>());
                frame(std::integral_constant<int, 2>());
                frame(std::integral_constant<int, 3>());
                if (Y) {
                    // out[k] of the four lanes added up, frame k's sum to lane k
                    const bool o1 = ch.j & 1, o2 = ch.j & 2;
                    const float a = (o1 ? out[1] : out[0]) + quad<0xB1>(o1 ? out[0] : out[1]);
                    const float b = (o1 ? out[3] : out[2]) + quad<0xB1>(o1 ? out[2] : out[3]);
                    yv[i] = (o2 ? b : a) + quad<0x4E>(o2 ? a : b) + skip * uv[i];
                }
            }
            if (Y) {
                if (zw.p) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) yv[i] *= zv[i] * sigmoidf(zv[i]);
                }
                if (ch.live) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (whole || t + q + 4 * i + ch.j < t1) *yw.at(t + q, i) = (T)yv[i];
                }
            }
        }
        // (the next tile goes to the other buffer; the one after it comes behind the next barrier)
    }
    if (!Y) sum += quad<0xB1>(sum), sum += quad<0x4E>(sum);
    return sum;
}

// zeros for the frames past a sequence's end, by the whole block
template <typename T, int NS>
__device__ __forceinline__ void zero_frames(const ScanParams<T>& p, const Channel<T, NS>& ch, int t0, int t1) {
    T* yb = p.y.row(ch.b, 0) + ch.d;
    if (ch.live)
        for (int t = t0 + ch.j; t < t1; t += kLanes) yb[(long long)t * p.y.rs] = (T)0.f;
}

template <typename T, int NS>
__device__ __forceinline__ float* piece_states(const ScanParams<T>& p, const Channel<T, NS>& ch, int piece) {
    return p.ws_h + (((long long)ch.b * (p.pieces - 1) + piece) * p.D + ch.d) * (kLanes * NS) + ch.j * NS;
}
template <typename T, int NS>
__device__ __forceinline__ float* piece_sum(const ScanParams<T>& p, const Channel<T, NS>& ch, int piece) {
    return p.ws_s + ((long long)ch.b * (p.pieces - 1) + piece) * p.D + ch.d;
}

// Grid (channel blocks of all groups, pieces, sequences).  FIRST: piece 0 from the given state, results and all; every other
// piece but the last from a zero state, for the state it leaves behind.  Second launch: the pieces from 1 on, each from the
// state before it, which it puts together from what the first launch left.
template <typename T, int NS, bool FIRST>
__global__ __launch_bounds__(256) void scan_kernel(ScanParams<T> p) {
    __shared__ float lds[2 * 2 * kTile * kLanes * NS];
    Channel<T, NS> ch;
    const int g = blockIdx.x / p.blocks_per_group, cb = blockIdx.x % p.blocks_per_group;
    const int piece = FIRST ? blockIdx.y : blockIdx.y + 1;
    for (int b = blockIdx.z; b < p.B; b += gridDim.z) {
        ch.init(p, b, g, cb * kBlockChannels + (threadIdx.x >> 2));
        const long long first = (long long)piece * p.piece;
        const int t0 = (int)min(first, (long long)p.Tmax), te = (int)min(first + p.piece, (long long)p.Tmax);
        const int t1 = min(te, ch.len);
        const bool last = ch.len <= te;  // no live frame behind this piece
        float h[NS];
        if (FIRST && piece > 0) {
            if (!last) {
#pragma unroll
                for (int s = 0; s < NS; ++s) h[s] = 0.f;
                const float sum = scan_frames<T, NS, false>(p, ch, t0, t1, h, lds);
                if (ch.live) {
                    float* to = piece_states(p, ch, piece);
#pragma unroll
                    for (int s = 0; s < NS; ++s) to[s] = h[s];
                    if (ch.j == 0) *piece_sum(p, ch, piece) = sum;
                }
            }
        } else if (FIRST || t0 < ch.len) {
            if (FIRST) {
                ch.load_state(p, h);
            } else {
                const float* from = piece_states(p, ch, 0);
#pragma unroll
                for (int s = 0; s < NS; ++s) h[s] = from[s];
                for (int k = 1; k < piece; ++k) {
                    from = piece_states(p, ch, k);
                    const float sum = *piece_sum(p, ch, k);
#pragma unroll
                    for (int s = 0; s < NS; ++s) h[s] = __builtin_amdgcn_exp2f(sum * ch.A2[s]) * h[s] + from[s];
                }
            }
            if (t0 < t1) scan_frames<T, NS, true>(p, ch, t0, t1, h, lds);
            if (last) {
                ch.store_state(p, h);
            } else if (FIRST && ch.live) {
                float* to = piece_states(p, ch, 0);
#pragma unroll
                for (int s = 0; s < NS; ++s) to[s] = h[s];
            }
        }
        if (!FIRST || piece == 0) zero_frames(p, ch, max(t0, ch.len), te);
        __syncthreads();  // the next sequence starts over with the first buffer
    }
}

// A few frames of many sequences (decode steps): no LDS, no barrier; what counts is the state, read and written once.
template <typename T, int NS>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanParams<T> p) {
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) >> 2;
    const long long last = (long long)p.B * p.D - 1;
    const long long at = i < last ? i : last;
    const int Dg = p.D / p.G, b = (int)(at / p.D), d = (int)(at % p.D), g = d / Dg;
    Channel<T, NS> ch;
    ch.init(p, b, g, d - g * Dg);
    ch.live = i <= last;
    float h[NS];
    ch.load_state(p, h);
    const float bias = p.bias ? p.bias[d] : 0.f, skip = p.Dskip ? p.Dskip[d] : 0.f;
    for (int t = 0; t < p.Tmax; ++t) {
        float v = 0.f;
        if (t < ch.len) {
            const float u = (float)p.u.row(b, t)[d];
            float dt = (float)p.delta.row(b, t)[d] + bias;
            float bn[NS], cn[NS];
            load_my_states(p.Bm.row(b, t) + g * p.Bg, p.N, ch.j, bn);
            load_my_states(p.Cm.row(b, t) + g * p.Cg, p.N, ch.j, cn);
            const float z = p.z.p ? (float)p.z.row(b, t)[d] : 0.f;
            if (p.softplus) dt = softplusf(dt);
            const float x = dt * u;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                h[s] = __builtin_amdgcn_exp2f(dt * ch.A2[s]) * h[s] + x * bn[s];
                v += cn[s] * h[s];
            }
            v += quad<0xB1>(v), v += quad<0x4E>(v);  // (the four lanes of a channel are in this branch together)
            v += skip * u;
            if (p.z.p) v *= z * sigmoidf(z);
        }
        if (ch.live && ch.j == 0) p.y.row(b, t)[d] = (T)v;
    }
    ch.store_state(p, h);
}

// Calls of up to this many frames take the step kernel.
constexpr int kStepFrames = 4;

// Pieces that the frames of each sequence are cut into.
static int scan_pieces(int B, int T, int D, int G) {
    const long long waves = (long long)B * G * ((D / G + 15) / 16);
    if (waves >= 1024 || T < 128) return 1;
    long long n = 2048 / waves;
    n = std::min<long long>(n, T / 64);
    n = std::min<long long>(n, 128);
    return n < 3 ? 1 : (int)n;
}

struct ScanPlan {
    int NS, piece, pieces;
    size_t h_bytes, bytes;
};
static ScanPlan scan_plan(const mv_selective_scan_args* a) {
    ScanPlan s{};
    s.NS = 1;
    while (s.NS * kLanes < a->N) s.NS *= 2;
    s.pieces = a->T <= kStepFrames ? 1 : scan_pieces(a->B, a->T, a->D, a->G);
    s.piece = round_up((a->T + s.pieces - 1) / s.pieces, kTile);
    s.pieces = (int)(((long long)a->T + s.piece - 1) / s.piece);
    if (s.pieces > 1) {
        const size_t n = (size_t)a->B * (s.pieces - 1) * a->D;
        s.h_bytes = (n * kLanes * s.NS * 4 + 255) / 256 * 256;
        s.bytes = s.h_bytes + (n * 4 + 255) / 256 * 256;
    }
    return s;
}

template <typename T, int NS>
static int launch_scan(ScanParams<T> p, hipStream_t stream) {
    if (p.Tmax <= kStepFrames) {
        const long long blocks = ((long long)p.B * p.D * kLanes + 255) / 256;
        hipLaunchKernelGGL((scan_step_kernel<T, NS>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
        MV_HIP(hipGetLastError());
        return MV_OK;
    }
    const unsigned z = (unsigned)std::min(p.B, 65535), x = (unsigned)(p.G * p.blocks_per_group);
    hipLaunchKernelGGL((scan_kernel<T, NS, true>), dim3(x, p.pieces > 1 ? p.pieces - 1 : 1, z), dim3(256), 0, stream, p);
    MV_HIP(hipGetLastError());
    if (p.pieces > 1) {
        hipLaunchKernelGGL((scan_kernel<T, NS, false>), dim3(x, p.pieces - 1, z), dim3(256), 0, stream, p);
        MV_HIP(hipGetLastError());
    }
    return MV_OK;
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
    if (a->D > 1 << 22 || (long long)a->B * a->D > 1ll << 29) {
        set_error("%s: more than 2^22 channels, or B * D over 2^29", who);
        return MV_EINVAL;
    }
    return MV_OK;
}

extern "C" {

size_t mv_selective_scan_workspace(const mv_selective_scan_args* a) {
    if (check_scan(a) || a->B == 0 || a->T == 0) return 0;
    return scan_plan(a).bytes;
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
    const ScanPlan plan = scan_plan(a);
    if (plan.bytes && (!workspace || workspace_bytes < plan.bytes || ((uintptr_t)workspace & 255) != 0)) {
        set_error("%s: workspace: need %zu bytes, 256-byte aligned (got %zu)", who, plan.bytes, workspace_bytes);
        return MV_ENOMEM;
    }
    return by_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        ScanParams<T> p{rows_of<const T>(a->u), rows_of<const T>(a->delta), rows_of<const T>(a->z), rows_of<const T>(a->Bm),
                        rows_of<const T>(a->Cm), rows_of<T>(a->y), a->A, a->Dskip, a->delta_bias, a->state_in, a->state_out,
                        a->lengths, (long long)a->Bg_stride, (long long)a->Cg_stride, (float*)workspace,
                        (float*)((char*)workspace + plan.h_bytes), a->B, a->T, a->D, a->N, a->G, a->delta_softplus,
                        (a->D / a->G + kBlockChannels - 1) / kBlockChannels, plan.piece, plan.pieces};
        switch (plan.NS) {
            case 1: return launch_scan<T, 1>(p, (hipStream_t)stream);
            case 2: return launch_scan<T, 2>(p, (hipStream_t)stream);
            case 4: return launch_scan<T, 4>(p, (hipStream_t)stream);
            case 8: return launch_scan<T, 8>(p, (hipStream_t)stream);
            default: return launch_scan<T, 16>(p, (hipStream_t)stream);
        }
    });
}

}  // extern "C"
