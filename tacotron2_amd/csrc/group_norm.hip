// group_norm.hip -- group normalisation with an activation on channels-last tensors (mv_group_norm).
//
//   y = act((x - m) / sqrt(v + eps) * w_c + b_c),  m and v over (t < len, c in group), or over a frame's group alone
//
// HBM-bound: x once in, y once out.  The variance is a sum of squared distances from a mean that is already known (sums of
// squares lose it where the mean is far from zero), so what is normalised has to be looked at twice: it stays in registers
// between the two looks wherever it fits.  32 utterances of up to 861 frames, 512 channels, 32 groups, bf16, SiLU: 12.9 us
// (3.5 TB/s, all in one load and one store phase a block); 16 of up to 55104 x 128, float16, in pieces: 95 - 99 us (statistics 33,
// the second pass 68 at 5.4 TB/s); 64 single frames of 1024 channels: 3.6 us, a launch.
//
//   frame_norm_kernel     per frame, groups of up to 64 * 8 vectors: L lanes hold a group
//   group_norm_kernel     a sequence's group(s) in one block's registers: one read, one write, one launch
//   group_stats_kernel +  a sequence in pieces: count, mean and squared distances of each, batch by batch; then the pieces are
//   group_apply_kernel    put together and x is read a second time
//   wide_norm_kernel      what none of them holds: groups of more channels than a block holds at once, one block to a group and
//                         one element to a load, three times over x (a sequence of 500 x 8200 float32, one group: 13.7 ms, where
//                         500 x 4096 take 16 us; 8 x 861 frames of 8200 bf16 channels, a group each, 129 us)
//
// A vector is as many channels of a group as there are, a power of two of them, 16 bytes at most, at any address.  It never
// holds two groups: where the group is no multiple of it (R), the group's last vector reaches back over the one before; what
// both hold counts once (`skip`), and both write the same.  32 x 861 frames, bf16, C about 512: groups of 17 channels 25 us
// and per frame 24 us (31 and 111 us with the largest vector that divides the group, one channel), of 7 20 and 20 us (59 and
// 60 us), of 16, where nothing overlaps, 15 and 14 us; a group of one channel, a vector of its own, 78 - 99 us.
#include "sequence.h"

namespace mv {

int check_sequence(const char* who, int B, int T, int C, int dtype) {
    if (B < 0 || T < 0 || T > 1 << 30 || C < 1 || C > 1 << 30) {
        set_error("%s: bad sizes (B=%d, T=%d, channels=%d)", who, B, T, C);
        return MV_EINVAL;
    }
    if (dtype != MV_DTYPE_F32 && dtype != MV_DTYPE_BF16 && dtype != MV_DTYPE_F16) {
        set_error("%s: unknown dtype %d", who, dtype);
        return MV_EINVAL;
    }
    return MV_OK;
}

int check_aligned(const char* who, const void* p, size_t bytes) {
    if ((uintptr_t)p % bytes == 0) return MV_OK;
    set_error("%s: a pointer is not aligned to its elements", who);
    return MV_EINVAL;
}

int check_rows(const char* who, const char* what, const mv_rows& r, int T, int dtype) {
    if (!r.ptr || ((uintptr_t)r.ptr % dtype_size(dtype)) != 0 || r.batch_stride < 0 || r.row_stride < 0 ||
        (T > 1 && r.row_stride > 1 << 25)) {
        set_error("%s: %s needs an aligned pointer, strides >= 0 and a row stride of at most 2^25", who, what);
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
    if (int rc = check_rows(who, "the output", r, T, dtype)) return rc;
    if (!rows_disjoint(r, B, T, C)) {
        set_error("%s: the output's rows overlap (batch_stride %lld, row_stride %lld)", who, (long long)r.batch_stride,
                  (long long)r.row_stride);
        return MV_EINVAL;
    }
    return MV_OK;
}

// some i in [i0, i1], k in [k0, k1] with lo < d + i * p + k * q < hi (p, q >= 0)
static bool hits(long long lo, long long hi, long long d, long long i0, long long i1, long long p, long long k0, long long k1,
                 long long q) {
    if (i1 - i0 > k1 - k0) std::swap(i0, k0), std::swap(i1, k1), std::swap(p, q);
    for (long long i = i0; i <= (p ? i1 : i0); ++i) {
        const long long r = d + i * p;
        long long k = k0;
        if (q) {  // the first k past lo
            const long long n = lo - r, below = n / q - (n % q < 0);
            k = std::max(k0, below + 1);
        }
        if (k <= k1 && r + k * q > lo && r + k * q < hi) return true;
    }
    return false;
}

// Whether two pieces of memory have a byte in common, as far as that is decided: of rows with the same strides (halves of one
// buffer), of rows and a piece without gaps, and of any two that start alike.
static bool meet(const Span& a, const Span& b) {
    typedef __int128 wide;
    if (!a.p || !b.p || a.width == 0 || b.width == 0) return false;
    auto extent = [](const Span& s) { return (wide)(s.B - 1) * s.bs + (wide)(s.T - 1) * s.ts + s.width; };
    auto whole = [](const Span& s) {
        return ((s.T == 1 || s.ts == s.width) && (s.B == 1 || (wide)s.bs == (wide)s.T * s.width)) ||
               ((s.B == 1 || s.bs == s.width) && (s.T == 1 || (wide)s.ts == (wide)s.B * s.width));
    };
    const wide ea = extent(a), eb = extent(b), d = (wide)(intptr_t)b.p - (intptr_t)a.p;
    if (d >= ea || -d >= eb) return false;
    if (d == 0) return true;
    if (ea + eb > (wide)1 << 60) return false;  // (no device's memory)
    if (a.bs == b.bs && a.ts == b.ts && a.B == b.B && a.T == b.T)
        return hits(-b.width, a.width, (long long)d, 1 - a.B, a.B - 1, a.bs, 1 - a.T, a.T - 1, a.ts);
    if (whole(a)) return hits(-b.width, (long long)ea, (long long)d, 0, b.B - 1, b.bs, 0, b.T - 1, b.ts);
    return whole(b) && hits(-a.width, (long long)eb, (long long)-d, 0, a.B - 1, a.bs, 0, a.T - 1, a.ts);
}

int check_overlaps(const char* who, const Span& output, const char* what, std::initializer_list<Span> inputs) {
    for (const Span& in : inputs)
        if (meet(output, in)) {
            set_error("%s: %s overlaps another argument of the call", who, what);
            return MV_EINVAL;
        }
    return MV_OK;
}

template <typename T>
struct NormParams {
    Rows<const T> x;
    Rows<T> y;
    const void *w, *b;
    const int32_t* lengths;
    float *n, *mean, *m2;  // pieces' statistics [B][G][pieces]
    int B, Tmax, C, G, w32, past;  // past: results past the L2
    float slope, eps;
    int tile, tiles;     // vectors of a row to a block, blocks to a row
    int piece, pieces;   // frames to a block, blocks to a sequence
};

template <typename T, int V>
__device__ __forceinline__ void load_weights(const void* w, bool w32, int c, float none, float (&v)[V]) {
    if (!w) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = none;
    } else if (w32) {
        const auto t = *(const typename Unaligned<float, V>::type*)((const float*)w + c);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = t[e];
    } else {
        const auto t = *(const typename Unaligned<T, V>::type*)((const T*)w + c);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (float)t[e];
    }
}

// (x - mean) * rstd * w + b of one vector
template <typename T, int V, int ACT>
__device__ __forceinline__ typename Unaligned<T, V>::type normalise(typename Unaligned<T, V>::type x, float mean, float rstd,
                                                                    const float (&w)[V], const float (&b)[V], float slope) {
    typename Unaligned<T, V>::type y;
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = (T)activate<ACT>(((float)x[e] - mean) * rstd * w[e] + b[e], slope);
    return y;
}

// sums over a vector's elements, those from `skip` on where vectors reach back (R)
template <typename T, int V, bool R>
__device__ __forceinline__ float sum_of(typename Unaligned<T, V>::type x, int skip) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) s += !R || e >= skip ? (float)x[e] : 0.f;
    return s;
}
template <typename T, int V, bool R>
__device__ __forceinline__ float squares_of(typename Unaligned<T, V>::type x, float mean, int skip) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float d = !R || e >= skip ? (float)x[e] - mean : 0.f;
        s += d * d;
    }
    return s;
}

// A vector as it was loaded, for the compiler a new value: what is computed from it is computed again rather than kept, and
// the registers that hold a tile hold its 16-bit elements, not their float32 conversions.
template <typename Vec>
__device__ __forceinline__ Vec forget(Vec v) {
    struct Words {
        unsigned w[(sizeof(Vec) + 3) / 4];
    } u{};
    __builtin_memcpy(&u, &v, sizeof(Vec));
#pragma unroll
    for (unsigned& w : u.w) asm volatile("" : "+v"(w));
    __builtin_memcpy(&v, &u, sizeof(Vec));
    return v;
}

// The sum of `v` over the threads of each group of the block.  Threads stand row-major over [rows][tile] vectors, a group is
// `gv` adjacent vectors of every row; a wave adds up a group's values, `red` holds one float a thread and one a group.
// Every thread of the block calls it; the order of additions depends on the layout alone.
__device__ __forceinline__ float group_total(float v, float* red, int rows, int tile, int gv, int mine) {
    const int groups = tile / gv, waves = blockDim.x >> 6, lane = threadIdx.x & 63;
    float* res = red + blockDim.x;
    red[threadIdx.x] = v;
    __syncthreads();
    for (int g = threadIdx.x >> 6; g < groups; g += waves) {
        float s = 0.f;
        for (int i = lane; i < rows * gv; i += 64) s += red[i / gv * tile + g * gv + i % gv];
#pragma unroll
        for (int m = 32; m; m >>= 1) s += __shfl_xor(s, m);
        if (lane == 0) res[g] = s;
    }
    __syncthreads();
    const float r = res[mine];
    __syncthreads();
    return r;
}

// A block's thread on a tile of vectors of a row: which vector, which rows (row, row + rows, ...), which group of the tile.
// Addresses are a base that the block shares plus a 32-bit offset of the thread (the plan sees to it that it fits).
template <typename T, int V, bool R>
struct Place {
    int row, rows, c, skip, mine, gv;
    bool first;  // of its group
    bool in;     // false: a thread without a row, or past the last vector of a row; it loads what its neighbour does

    __device__ __forceinline__ Place(const NormParams<T>& p, int tile) {
        const int tile0 = tile * p.tile, v = threadIdx.x % p.tile;
        const int Cg = p.C / p.G;
        gv = (Cg + V - 1) / V;
        rows = blockDim.x / p.tile;
        row = min((int)threadIdx.x / p.tile, rows - 1);
        in = threadIdx.x < rows * p.tile && tile0 + v < p.G * gv;
        const int at = min(tile0 + v, p.G * gv - 1), k = at % gv;
        c = R ? at / gv * Cg + min(k * V, Cg - V) : at * V;
        skip = R && k == gv - 1 ? gv * V - Cg : 0;
        first = k == 0;
        mine = v / gv;
    }
    // frame t0 + row + i * rows; frames from `end` on: frame end - 1
    template <typename P>
    __device__ __forceinline__ P* at(P* frame0, long long rs, int t0, int i, int end) const {
        const unsigned first = (unsigned)(row * (int)rs + c) * (unsigned)sizeof(T);
        if (t0 + (i + 1) * rows <= end) return (P*)((char*)(frame0 + (t0 + (long long)i * rows) * rs) + first);
        const int r = min(row + i * rows, end - 1 - t0);
        return (P*)((char*)(frame0 + t0 * rs) + (unsigned)(r * (int)rs + c) * (unsigned)sizeof(T));
    }
};

// Frames [t0, t1) of a tile in the block's registers, NI vectors to a thread, and the statistics of the thread's group.
template <typename T, int V, int NI, bool R>
struct Held {
    typedef typename Unaligned<T, V>::type Vec;
    Vec x[NI];
    float mean, m2;

    // count: frames * channels of the group
    __device__ __forceinline__ void take(const NormParams<T>& p, const Place<T, V, R>& at, int b, int t0, int t1, float count,
                                         float* red) {
#pragma unroll
        for (int i = 0; i < NI; ++i) x[i] = *(const Vec*)at.at(p.x.row(b, 0), p.x.rs, t0, i, t1);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (at.in && t0 + at.row + i * at.rows < t1) s += sum_of<T, V, R>(x[i], at.skip);
        mean = group_total(s, red, at.rows, p.tile, at.gv, at.mine) / count;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i) x[i] = forget(x[i]);
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (at.in && t0 + at.row + i * at.rows < t1) s += squares_of<T, V, R>(x[i], mean, at.skip);
        m2 = group_total(s, red, at.rows, p.tile, at.gv, at.mine);
#pragma unroll
        for (int i = 0; i < NI; ++i) x[i] = forget(x[i]);
    }
};

constexpr int kNormThreads = 1024;

// One block to a tile of a sequence: whole groups of it, all frames.  Blocks go to the 8 XCDs in turn; here each XCD gets a
// run of tiles, so that tiles that share a 128-byte line meet in one L2.
template <typename T, int V, int NI, int ACT, bool R>
__global__ __launch_bounds__(kNormThreads) void group_norm_kernel(NormParams<T> p) {
    __shared__ float red[2 * kNormThreads];
    typedef typename Unaligned<T, V>::type Vec;
    const unsigned work = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int b = work / p.tiles;
    if (b >= p.B) return;
    const Place<T, V, R> at(p, work - b * p.tiles);
    Held<T, V, NI, R> h;
    const int len = seq_frames(p.lengths, b, p.Tmax);
    const float count = (float)len * (float)(p.C / p.G);
    if (len) h.take(p, at, b, 0, len, count, red);
    const float rstd = 1.f / sqrtf(h.m2 / count + p.eps);
    float w[V], bias[V];
    load_weights<T, V>(p.w, p.w32, at.c, 1.f, w);
    load_weights<T, V>(p.b, p.w32, at.c, 0.f, bias);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int t = at.row + i * at.rows;
        Vec y;
        if (t < len) {
            y = normalise<T, V, ACT>(h.x[i], h.mean, rstd, w, bias, p.slope);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = (T)0.f;
        }
        if (at.in && t < p.Tmax) store_vec<T, V>(at.at(p.y.row(b, 0), p.y.rs, 0, i, p.Tmax), y, p.past);
        __builtin_amdgcn_sched_barrier(0);  // one vector after the other: the registers hold the tile, not 16 results
    }
}

// Grid (tiles, pieces, sequences): statistics of a piece of a sequence.  A thread takes kStatRows vectors at a time: their
// mean, their squared distances from it, and both into what it has so far (n, mean, m2 of the values seen:
// mean' = mean + d n2 / n', m2' = m2 + q + d^2 n n2 / n' with d the distance of the means); the block's threads are put
// together the same way at the end.
constexpr int kStatRows = 8;
template <typename T, int V, bool R>
__global__ __launch_bounds__(kNormThreads) void group_stats_kernel(NormParams<T> p) {
    __shared__ float red[2 * kNormThreads];
    typedef typename Unaligned<T, V>::type Vec;
    const Place<T, V, R> at(p, blockIdx.x);
    const int Cg = p.C / p.G;
    for (int b = blockIdx.z; b < p.B; b += gridDim.z) {
        const int len = seq_frames(p.lengths, b, p.Tmax);
        const int t0 = blockIdx.y * p.piece, t1 = min(t0 + p.piece, len);
        float n = 0.f, mean = 0.f, m2 = 0.f;
        for (int t = t0; t < t1; t += kStatRows * at.rows) {
            Vec x[kStatRows];
#pragma unroll
            for (int i = 0; i < kStatRows; ++i) x[i] = *(const Vec*)at.at(p.x.row(b, 0), p.x.rs, t, i, t1);
            // this thread's frames of the batch: t + row, t + row + rows, ...
            const int mine = at.in ? min(kStatRows, max(0, (t1 - t - at.row + at.rows - 1) / at.rows)) : 0;
            const float n2 = (float)(mine * (V - at.skip));
            if (mine > 0) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < kStatRows; ++i)
                    if (i < mine) s += sum_of<T, V, R>(x[i], at.skip);
                const float mu = s / n2;
                float q = 0.f;
#pragma unroll
                for (int i = 0; i < kStatRows; ++i)
                    if (i < mine) q += squares_of<T, V, R>(x[i], mu, at.skip);
                const float all = n + n2, d = mu - mean, part = n2 / all;
                mean += d * part;
                m2 += q + d * d * n * part;
                n = all;
            }
        }
        const float count = t1 > t0 ? (float)(t1 - t0) * (float)Cg : 0.f;
        if (t1 > t0) {
            const float mu = group_total(n * mean, red, at.rows, p.tile, at.gv, at.mine) / count, d = mean - mu;
            m2 = group_total(n > 0.f ? m2 + n * d * d : 0.f, red, at.rows, p.tile, at.gv, at.mine);
            mean = mu;
        }
        if (at.in && at.row == 0 && at.first) {
            const long long i = ((long long)b * p.G + at.c / Cg) * p.pieces + blockIdx.y;
            p.n[i] = count;
            p.mean[i] = mean;
            p.m2[i] = m2;
        }
    }
}

// Mean and 1 / sqrt(variance + eps) of a group from its pieces, by one wave: sum n_i m_i / n, then the pieces' own squared
// distances and those of their means.
__device__ __forceinline__ void join_pieces(const float* n, const float* mean, const float* m2, int pieces, float eps,
                                            float* out_mean, float* out_rstd) {
    const int lane = threadIdx.x & 63;
    float N = 0.f, s = 0.f;
    for (int i = lane; i < pieces; i += 64) N += n[i], s += n[i] * mean[i];
#pragma unroll
    for (int m = 32; m; m >>= 1) N += __shfl_xor(N, m), s += __shfl_xor(s, m);
    const float mu = s / N;
    float q = 0.f;
    for (int i = lane; i < pieces; i += 64) {
        const float d = mean[i] - mu;
        q += m2[i] + (n[i] > 0.f ? n[i] * d * d : 0.f);
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) q += __shfl_xor(q, m);
    if (lane == 0) *out_mean = mu, *out_rstd = 1.f / sqrtf(q / N + eps);
}

// Grid (tiles, pieces, sequences).  `piece` is this launch's own, a multiple of 4 * rows frames.
template <typename T, int V, int ACT, bool R>
__global__ __launch_bounds__(kNormThreads) void group_apply_kernel(NormParams<T> p) {
    __shared__ float stat[2 * kNormThreads];
    typedef typename Unaligned<T, V>::type Vec;
    const Place<T, V, R> at(p, blockIdx.x);
    float w[V], bias[V];
    load_weights<T, V>(p.w, p.w32, at.c, 1.f, w);
    load_weights<T, V>(p.b, p.w32, at.c, 0.f, bias);
    const int groups = p.tile / at.gv, g0 = blockIdx.x * groups;
    for (int b = blockIdx.z; b < p.B; b += gridDim.z) {
        const int len = seq_frames(p.lengths, b, p.Tmax);
        const int t0 = blockIdx.y * p.piece, te = min(t0 + p.piece, p.Tmax), live = min(te, len);
        __syncthreads();
        if (t0 < live)
            for (int g = threadIdx.x >> 6; g < groups; g += blockDim.x >> 6)
                if (g0 + g < p.G) {
                    const long long i = ((long long)b * p.G + g0 + g) * p.pieces;
                    join_pieces(p.n + i, p.mean + i, p.m2 + i, p.pieces, p.eps, &stat[g], &stat[kNormThreads + g]);
                }
        __syncthreads();
        const float mean = stat[at.mine], rstd = stat[kNormThreads + at.mine];
        for (int t = t0; t < te; t += 4 * at.rows) {
            Vec x[4];
            if (t < live) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = *(const Vec*)at.at(p.x.row(b, 0), p.x.rs, t, i, live);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int f = t + at.row + i * at.rows;
                Vec y;
                if (f < live) {
                    y = normalise<T, V, ACT>(x[i], mean, rstd, w, bias, p.slope);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) y[e] = (T)0.f;
                }
                if (at.in && f < te) store_vec<T, V>(at.at(p.y.row(b, 0), p.y.rs, t, i, te), y, p.past);
            }
        }
    }
}

// Each frame's groups by themselves: L lanes to a group, NI vectors to a lane.  A slot of L lanes keeps its group (and its
// weights) and walks the frames.
template <typename T, int V, int NI, int ACT, bool R>
__global__ __launch_bounds__(256) void frame_norm_kernel(NormParams<T> p, int L, unsigned slots) {
    typedef typename Unaligned<T, V>::type Vec;
    const unsigned slot = (blockIdx.x * 256 + threadIdx.x) >> (31 - __builtin_clz(L));
    if (slot >= slots) return;  // (whole slots leave: L divides 64)
    const int l = threadIdx.x & (L - 1), Cg = p.C / p.G, nv = (Cg + V - 1) / V, g = slot % p.G;
    auto from_of = [&](int i) { return R ? min((l + i * L) * V, Cg - V) : (l + i * L) * V; };
    auto skip_of = [&](int i) { return R && l + i * L == nv - 1 ? nv * V - Cg : 0; };
    float w[NI][V], bias[NI][V];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int c = g * Cg + min((l + i * L) * V, Cg - V);
        load_weights<T, V>(p.w, p.w32, c, 1.f, w[i]);
        load_weights<T, V>(p.b, p.w32, c, 0.f, bias[i]);
    }
    const unsigned frames = p.B * p.Tmax;
    for (unsigned f = slot / p.G; f < frames; f += slots / p.G) {
        const int b = f / p.Tmax, t = f - b * p.Tmax;
        T* to = p.y.row(b, t) + g * Cg;
        if (t >= seq_frames(p.lengths, b, p.Tmax)) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                Vec y;
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] = (T)0.f;
                if (l + i * L < nv) *(Vec*)(to + from_of(i)) = y;
            }
            continue;
        }
        const T* from = p.x.row(b, t) + g * Cg;
        Vec x[NI];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (l + i * L < nv) x[i] = *(const Vec*)(from + from_of(i));
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (l + i * L < nv) s += sum_of<T, V, R>(x[i], skip_of(i));
        for (int m = L >> 1; m; m >>= 1) s += __shfl_xor(s, m);
        const float mean = s / (float)Cg;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (l + i * L < nv) s += squares_of<T, V, R>(x[i], mean, skip_of(i));
        for (int m = L >> 1; m; m >>= 1) s += __shfl_xor(s, m);
        const float rstd = 1.f / sqrtf(s / (float)Cg + p.eps);
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (l + i * L < nv) *(Vec*)(to + from_of(i)) = normalise<T, V, ACT>(x[i], mean, rstd, w[i], bias[i], p.slope);
    }
}

// One block per group of a sequence (or of a frame), element by element: groups that no block's registers hold.  A thread's sums
// run over all frames, so they are held in 64 bits: a chain of float32 additions loses as many roundings as it has terms (the mean
// of 300 x 10000 values near 3, spread 0.01, was off by enough for 1.3 times the error of a rounded one in the result).
template <typename T, int ACT>
__global__ __launch_bounds__(256) void wide_norm_kernel(NormParams<T> p, int per_frame) {
    __shared__ double red[256];
    const int Cg = p.C / p.G;
    long long item = blockIdx.x;
    const int g = item % p.G;
    item /= p.G;
    int t0 = 0, t1 = p.Tmax;
    if (per_frame) {
        t0 = item % p.Tmax;
        t1 = t0 + 1;
        item /= p.Tmax;
    }
    const int b = (int)item, len = seq_frames(p.lengths, b, p.Tmax), c0 = g * Cg, end = min(t1, len);
    const double count = (double)max(0, end - t0) * (double)Cg;
    auto total = [&](double v) {
        red[threadIdx.x] = v;
        __syncthreads();
        for (int s = 128; s; s >>= 1) {
            if (threadIdx.x < s) red[threadIdx.x] += red[threadIdx.x + s];
            __syncthreads();
        }
        const double r = red[0];
        __syncthreads();
        return r;
    };
    double s = 0.;
    for (int t = t0; t < end; ++t)
        for (int c = threadIdx.x; c < Cg; c += 256) s += (float)p.x.row(b, t)[c0 + c];
    const float mean = (float)(total(s) / count);
    s = 0.;
    for (int t = t0; t < end; ++t)
        for (int c = threadIdx.x; c < Cg; c += 256) {
            const float d = (float)p.x.row(b, t)[c0 + c] - mean;
            s += d * d;
        }
    const float rstd = 1.f / sqrtf((float)(total(s) / count) + p.eps);
    for (int t = t0; t < t1; ++t)
        for (int c = c0 + threadIdx.x; c < c0 + Cg; c += 256) {
            float v = 0.f;
            if (t < end) {
                v = ((float)p.x.row(b, t)[c] - mean) * rstd;
                v = v * (p.w ? load_weight<T>(p.w, p.w32, c) : 1.f) + (p.b ? load_weight<T>(p.b, p.w32, c) : 0.f);
                v = activate<ACT>(v, p.slope);
            }
            p.y.row(b, t)[c] = (T)v;
        }
}

// --- host side -----------------------------------------------------------------------------------------------------
enum { NORM_FRAME, NORM_HELD, NORM_PIECES, NORM_WIDE };
struct NormPlan {
    int kind, V, NI, threads, tile, tiles, piece, pieces, apply_piece, L;
    bool past, reach;
    size_t bytes;
};

static int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
static int pow2_at_least(int v, int most) {
    int p = 1;
    while (p < v && p < most) p *= 2;
    return p;
}

static NormPlan norm_plan(const mv_group_norm_args* a) {
    NormPlan s{};
    const int Cg = a->C / a->groups, size = (int)dtype_size(a->dtype);
    s.V = 16 / size;
    while (s.V > Cg) s.V /= 2;
    // (in place, two vectors that share channels must not be two threads' whose order nothing sets)
    if (!a->per_frame && a->x.ptr == a->y.ptr)
        while (Cg % s.V) s.V /= 2;
    s.reach = Cg % s.V != 0;
    const int gv = ceil_div(Cg, s.V), row = a->groups * gv;
    s.kind = NORM_WIDE;
    auto by_frame = [&] {
        if (gv > 64 * 8) return s;
        s.kind = NORM_FRAME;
        s.L = pow2_at_least(gv, 64);
        s.NI = pow2_at_least(ceil_div(gv, s.L), 8);
        return s;
    };
    if (a->per_frame) return by_frame();
    if (gv > kNormThreads) return s;
    const long long far = a->T > 1 ? std::max(a->x.row_stride, a->y.row_stride) : 0;  // (of a single row the stride says nothing)
    auto fits = [&](long long frames) { return (frames * far + a->C) * size < 1ll << 31; };  // Place's offsets
    // Whole groups side by side.  A tile of a whole sequence: rows of 32 bytes at least, as many blocks as that gives (two
    // and more to a CU, one loading while another reduces or stores); rows of 64 bytes where results pass by the L2
    // (32 x 861 x 512, 32 groups, bf16 14.2 us, with 32 bytes 16.8), full lines where that leaves 384 blocks (float32 19.0 us
    // against 26.9 with 64 bytes; bf16, 256 blocks, 14.6 against 14.2).
    const int most = std::min(row, kNormThreads);
    auto grow = [&](int bytes) {
        while (s.tile * s.V * size < bytes && s.tile + gv <= most) s.tile += gv;
        s.tiles = ceil_div(row, s.tile);
    };
    s.tile = gv;
    s.past = pass_by_l2(a->y, a->B, a->T, a->C, a->dtype);
    grow(s.past ? 64 : 32);
    if (s.past && (long long)a->C * size / 128 * a->B >= 384) grow(128);
    s.past = s.past && !s.reach && (s.tile * s.V * size) % 64 == 0;
    if ((long long)s.tiles * a->B > 4096) grow(128);
    // A block computes 1000 vectors in 1.3 us; the second launch of the pieces costs 4.  So fewer blocks than CUs hold up to
    // 4096 vectors each (bf16: 1 x 2000 x 256, 16 groups, 9.4 us held, 11.9 in pieces; 1 x 4000 14.8 and 11.5; 2 x 8192 24.6
    // and 12.7), more blocks whatever fits (16 x 2000 x 512, 32 groups, 17.9 held, 21.8 in pieces).
    const bool few = (long long)s.tiles * a->B < 256;
    for (s.threads = 64; s.threads <= kNormThreads && !(few && (long long)a->T * s.tile > 4096); s.threads *= 2) {
        if (s.threads < s.tile) continue;
        const int n = ceil_div(a->T, s.threads / s.tile);
        if (n <= (s.threads < kNormThreads ? 8 : 16) && fits(s.threads / s.tile * 16ll) &&
            (long long)s.tiles * a->B * s.threads < 1ll << 31) {
            s.kind = NORM_HELD;
            s.NI = n <= 1 ? 1 : n <= 4 ? 4 : n <= 8 ? 8 : 16;
            return s;
        }
    }
    // a sequence of one frame is that frame: more of them than a grid holds tiles need no pieces and no scratch
    if (a->T == 1) return s.past = false, by_frame();
    // Pieces: full lines, and enough of them for eight blocks to a CU (padded ones leave at once).
    grow(128);
    s.threads = std::max(256, pow2_at_least(s.tile, kNormThreads));
    const int rows = s.threads / s.tile;
    const long long want = std::max(1ll, 2048 / ((long long)s.tiles * a->B));
    s.piece = rows * kStatRows * std::max(1, ceil_div(a->T, want * rows * kStatRows));
    s.pieces = ceil_div(a->T, s.piece);
    // The second pass goes in runs of 4 to 32 rows a thread: long ones put the pieces together less often, short ones give
    // blocks enough (one sequence of 30000 x 128 float32 24.0 us with runs of 32, 15.2 with 4; 16 of 55104 x 128 bf16 123 and 129).
    for (s.apply_piece = rows * 32; s.apply_piece > rows * 4 && (long long)s.tiles * a->B * ceil_div(a->T, s.apply_piece) < 2048;)
        s.apply_piece /= 2;
    if (s.pieces > 65535 || ceil_div(a->T, s.apply_piece) > 65535 || !fits(rows * 16ll)) return s;
    s.kind = NORM_PIECES;
    s.NI = 1;
    s.bytes = ((size_t)a->B * a->groups * s.pieces * 3 * 4 + 255) / 256 * 256;
    return s;
}

template <int N>
using Int = std::integral_constant<int, N>;

// calls f(V, NI, R) with the plan's vector, count and whether vectors reach back as constants
template <typename T, typename F>
static int by_plan(const NormPlan& s, F&& f) {
    auto by_count = [&](auto v, auto r) {
        switch (s.NI) {
            case 1: return f(v, Int<1>(), r);
            case 2: return f(v, Int<2>(), r);
            case 4: return f(v, Int<4>(), r);
            case 8: return f(v, Int<8>(), r);
            default: return f(v, Int<16>(), r);
        }
    };
    auto by_reach = [&](auto v) { return s.reach ? by_count(v, std::true_type()) : by_count(v, std::false_type()); };
    switch (s.V) {
        case 1: return by_count(Int<1>(), std::false_type());
        case 2: return by_reach(Int<2>());
        case 4: return by_reach(Int<4>());
        default: return by_reach(Int<(sizeof(T) == 2 ? 8 : 4)>());
    }
}

template <typename T, int ACT>
static int launch_norm(const mv_group_norm_args* a, const NormPlan& s, NormParams<T> p, hipStream_t stream) {
    const unsigned B16 = (unsigned)std::min(a->B, 65535);
    if (s.kind == NORM_WIDE) {
        const long long items = (long long)a->B * a->groups * (a->per_frame ? a->T : 1);
        if (items > 0xffffff) {
            set_error("mv_group_norm: more than 2^24 groups of over %d channels", a->per_frame || a->T == 1 ? 512 * s.V : kNormThreads * s.V);
            return MV_EINVAL;
        }
        hipLaunchKernelGGL((wide_norm_kernel<T, ACT>), dim3((unsigned)items), dim3(256), 0, stream, p, a->per_frame);
        MV_HIP(hipGetLastError());
        return MV_OK;
    }
    return by_plan<T>(s, [&](auto v, auto n, auto r) {
        constexpr int V = decltype(v)::value, NI = decltype(n)::value;
        constexpr bool R = decltype(r)::value;
        if (s.kind == NORM_FRAME) {
            if constexpr (NI <= 8) {
                const long long frames = (long long)a->B * a->T, most = 2048ll * 256 / s.L / a->groups;
                const long long slots = std::min(frames, std::max(1ll, most)) * a->groups;
                if (frames >= 1ll << 31 || slots * s.L >= 1ll << 31) {
                    set_error("mv_group_norm: more than 2^31 frames, or groups of a frame, in one call");
                    return MV_EINVAL;
                }
                hipLaunchKernelGGL((frame_norm_kernel<T, V, NI, ACT, R>), dim3((unsigned)((slots * s.L + 255) / 256)), dim3(256), 0,
                                   stream, p, s.L, (unsigned)slots);
            }
        } else if constexpr (NI != 2) {
            p.tile = s.tile;
            p.tiles = s.tiles;
            if (s.kind == NORM_HELD) {
                hipLaunchKernelGGL((group_norm_kernel<T, V, NI, ACT, R>), dim3((s.tiles * a->B + 7) / 8 * 8), dim3(s.threads), 0,
                                   stream, p);
            } else if constexpr (NI == 1) {
                p.piece = s.piece;
                p.pieces = s.pieces;
                hipLaunchKernelGGL((group_stats_kernel<T, V, R>), dim3(s.tiles, s.pieces, B16), dim3(s.threads), 0, stream, p);
                MV_HIP(hipGetLastError());
                p.piece = s.apply_piece;
                hipLaunchKernelGGL((group_apply_kernel<T, V, ACT, R>), dim3(s.tiles, ceil_div(a->T, s.apply_piece), B16),
                                   dim3(s.threads), 0, stream, p);
            }
        }
        MV_HIP(hipGetLastError());
        return MV_OK;
    });
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
    if (check_group_norm(a) || a->B == 0 || a->T == 0) return 0;
    return norm_plan(a).bytes;
}

int mv_group_norm(const mv_group_norm_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_group_norm(a)) return rc;
    if (a->B == 0 || a->T == 0) return MV_OK;
    if (int rc = check_rows("mv_group_norm", "x", a->x, a->T, a->dtype)) return rc;
    if (int rc = check_output_rows("mv_group_norm", a->y, a->B, a->T, a->C, a->dtype)) return rc;
    const size_t wsize = dtype_size(a->weight_dtype);
    if (int rc = check_aligned("mv_group_norm", a->weight, wsize)) return rc;
    if (int rc = check_aligned("mv_group_norm", a->bias, wsize)) return rc;
    if (int rc = check_aligned("mv_group_norm", a->lengths, 4)) return rc;
    const bool in_place = a->x.ptr == a->y.ptr && (a->B < 2 || a->x.batch_stride == a->y.batch_stride) &&
                          (a->T < 2 || a->x.row_stride == a->y.row_stride);
    const Span y(a->y, a->C, a->B, a->T, a->dtype), x(in_place ? mv_rows{} : a->x, a->C, a->B, a->T, a->dtype);
    if (int rc = check_overlaps("mv_group_norm", y, "y", {x, {a->weight, a->C * (long long)wsize}, {a->bias, a->C * (long long)wsize},
                                                          {a->lengths, 4ll * a->B}}))
        return rc;
    const NormPlan plan = norm_plan(a);
    if (plan.bytes && (!workspace || workspace_bytes < plan.bytes || ((uintptr_t)workspace & 255) != 0)) {
        set_error("mv_group_norm: workspace: need %zu bytes, 256-byte aligned (got %zu)", plan.bytes, workspace_bytes);
        return MV_ENOMEM;
    }
    return by_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        NormParams<T> p{};
        p.x = rows_of<const T>(a->x);
        p.y = rows_of<T>(a->y);
        p.w = a->weight;
        p.b = a->bias;
        p.lengths = a->lengths;
        const size_t n = (size_t)a->B * a->groups * plan.pieces;
        p.n = (float*)workspace;
        p.mean = p.n + n;
        p.m2 = p.mean + n;
        p.B = a->B;
        p.Tmax = a->T;
        p.C = a->C;
        p.G = a->groups;
        p.w32 = a->weight_dtype == MV_DTYPE_F32;
        p.past = plan.past;
        p.eps = a->eps;
        return by_activation(a->activation, a->slope, &p.slope, [&](auto act) {
            return launch_norm<T, decltype(act)::value>(a, plan, p, (hipStream_t)stream);
        });
    });
}

}  // extern "C"
