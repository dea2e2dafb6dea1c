// selective_scan.hip -- the selective state space recurrence on channels-last tensors (mv_selective_scan).
//
//   h[n] = exp(dt A[d, n]) h[n] + dt u B[g, n],   y = (sum_n C[g, n] h[n] + D u) z sigmoid(z)
//
// What bounds it.  Many frames: the vector unit.  A wave issues 27.3 vector instructions for a frame of 16 channels x 16 states,
// 5.0 of them transcendental (the states' exponentials are 4), and the counters show the unit active for 132 cycles of it (they
// count 4 for an instruction, 8 for a transcendental) while the CU is busy for 170.  With two waves on a SIMD, each spends 55 %
// of its life issuing, 24 % waiting to issue and 20 % for data, and the two blocks of a CU do not end together (a wave lives 86 %
// of the time its CU is busy).  32 utterances of 861 frames, 1024 channels, 16 states, bf16: 130 us, 73 ns a wave's frame (the
// bytes take 45 us); padded ones of 172 - 861 frames: 94 us a call, where that rate alone would give 77.  Frames of a channel are a chain: the parallelism is sequences x channels, four lanes to a channel (scan_kernel), and
// pieces of the frames where that does not fill the chip, at the price of going through them twice (a piece's decay needs no
// more than its sum of dt: exp(A sum dt)).  One sequence of 8192 frames: 76 us, 32 for the first launch (piece 0, whose results
// it makes, takes all of that) and 49 for the second.
// One frame of many sequences: the state, in and out once (scan_step_kernel).  512 sequences, 71 MB: 17.8 us, 4.0 TB/s.
#include "sequence.h"

namespace mv {

// log(1 + e^x) = max(x, 0) + log1p(e^-|x|), to 3e-7 of the result down to x = -80: the exponential gets back what rounding
// its argument cost, and log1p(e) is log(w) + (e - (w - 1)) with w = 1 + e rounded: the second term is what w lost (over w,
// which is 1 wherever the term counts), so small steps keep their relative precision.
__device__ __forceinline__ float softplusf(float x) {
    constexpr float kLn2 = 0.693147180559945309f;
    const float a = fabsf(x), t = a * -kLog2e, lost = __builtin_fmaf(a, -kLog2e, -t);
    float e = __builtin_amdgcn_exp2f(t);
    e = e > 0.f ? __builtin_fmaf(e, lost * kLn2, e) : e;  // (what an infinity lost is no number)
    const float w = 1.f + e;
    return fmaxf(x, 0.f) + __builtin_fmaf(__builtin_amdgcn_logf(w), kLn2, e - (w - 1.f));
}

// Four lanes share a channel; lane j of them holds states `state_of(j, 0 ... NS - 1)`: runs of four that a 16 x 16 outer
// product leaves in a lane (below), or of NS where a channel has fewer than 16.
constexpr int kLanes = 4;
template <int NS>
__device__ __forceinline__ constexpr int state_of(int j, int s) {
    return NS >= 4 ? 16 * (s / 4) + 4 * j + s % 4 : NS * j + s;
}
template <int NS>
constexpr int kRun = NS >= 4 ? 4 : NS;  // adjacent states of a lane

constexpr int kBlockChannels = 64;  // 4 waves of 16 channels

// A tile of frames in LDS: u, delta, z as they are stored, rows of 64 channels padded so that the four rows that a wave reads
// at once (lane 16 j + c is on channel c of a frame of its own) lie in different banks; B and C as float32 [frame][4 * NS];
// beside them, the steps dt by channel, each wave's own.
template <typename T, int NS>
struct Tile {
    static constexpr int frames = 64 / (int)sizeof(T), NP = kLanes * NS;
    static constexpr int vec = 16 / (int)sizeof(T), vecs = kBlockChannels / vec;  // vectors of a row
    static constexpr int row = kBlockChannels + 16;                                // elements
    static constexpr int steps = frames + 4;                                       // floats to a channel, padded
    T rows[3][frames][row];
    float maps[2][frames][NP];
};

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
    int order;  // 0: sequences as they come; otherwise the longest first, in rounds of `order` (below)
    int blocks_per_group, piece, pieces;  // frames to a piece (a multiple of 32), number of pieces
};

template <int CTRL>
__device__ __forceinline__ float quad(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// lane k's value in all four (k is a constant once the loop around it is unrolled)
__device__ __forceinline__ float quad_lane(float v, int k) {
    return k == 0 ? quad<0x00>(v) : k == 1 ? quad<0x55>(v) : k == 2 ? quad<0xAA>(v) : quad<0xFF>(v);
}

// Four lanes hold NP = 4 * NS states; where a channel has N < NP, no place from N on may add to the sum over states.  Zeros in it
// do not see to that: an infinite step or input makes a NaN of them (inf * 0).  scan_step_kernel, which waits for memory, writes
// their h as 0 in every frame.  scan_kernel has no instruction to spare for that; there these places hold the first states once
// more (NP <= 2 N, or all of them the one state there is): a copy goes the way of its original, to an infinity or a NaN too, and
// the C of the two (or four) is half (a quarter), so that together they add what one would.
__device__ __forceinline__ int state_at(int place, int N) { return place < N ? place : N == 1 ? 0 : place - N; }
__device__ __forceinline__ float share_of(int place, int N, int NP) {
    return N == 1 ? 1.f / (float)NP : state_at(place, N) < NP - N ? 0.5f : 1.f;
}

// Lane j's NS of the N values at p, as floats; where it has fewer, zeros or COPIES.
template <bool COPIES, typename T, int NS>
__device__ __forceinline__ void load_my_states(const T* p, int N, int j, float (&v)[NS]) {
    if (N == kLanes * NS) {
        typedef typename Unaligned<T, kRun<NS>>::type V;
#pragma unroll
        for (int s = 0; s < NS; s += kRun<NS>) {
            const V t = *(const V*)(p + state_of<NS>(j, s));
#pragma unroll
            for (int e = 0; e < kRun<NS>; ++e) v[s + e] = (float)t[e];
        }
    } else {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int place = state_of<NS>(j, s);
            v[s] = COPIES ? (float)p[state_at(place, N)] : place < N ? (float)p[place] : 0.f;
        }
    }
}
template <int NS>
__device__ __forceinline__ void store_my_states(float* p, int N, int j, const float (&v)[NS]) {
    if (N == kLanes * NS) {
        typedef typename Unaligned<float, kRun<NS>>::type V;
#pragma unroll
        for (int s = 0; s < NS; s += kRun<NS>) {
            V t;
#pragma unroll
            for (int e = 0; e < kRun<NS>; ++e) t[e] = v[s + e];
            *(V*)(p + state_of<NS>(j, s)) = t;
        }
    } else {
#pragma unroll
        for (int s = 0; s < NS; ++s)
            if (state_of<NS>(j, s) < N) p[state_of<NS>(j, s)] = v[s];
    }
}

// A of channel d for exponentials to base 2.  Clamped to finite: 0 * inf must not make a NaN of a frame past the end, whose dt
// is 0.
template <bool COPIES, typename T, int NS>
__device__ __forceinline__ void load_decays(const ScanParams<T>& p, int d, int j, float (&A2)[NS]) {
    load_my_states<COPIES>(p.A + (long long)d * p.N, p.N, j, A2);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const float a = A2[s] * kLog2e;
        A2[s] = a < -3e38f ? -3e38f : (a > 3e38f ? 3e38f : a);  // (a NaN stays one)
    }
}
template <bool COPIES, int NS>
__device__ __forceinline__ void load_state(const float* from, int N, int j, float (&h)[NS]) {
    if (from) {
        load_my_states<COPIES>(from, N, j, h);
    } else {
#pragma unroll
        for (int s = 0; s < NS; ++s) h[s] = 0.f;
    }
}

// The calling thread's channel.
template <typename T, int NS>
struct Channel {
    int b, g, d, j, len;
    bool live;   // false: a lane past the group's last channel, which computes on the last one and stores nothing
    float A2[NS];

    __device__ __forceinline__ void init(const ScanParams<T>& p, int b_, int g_, int c, int j_) {
        const int Dg = p.D / p.G;
        b = b_, g = g_, j = j_;
        live = c < Dg;
        d = g * Dg + min(c, Dg - 1);
        len = seq_frames(p.lengths, b, p.Tmax);
        load_decays<true>(p, d, j, A2);
    }
};

// a[k] of four values, each spread over the four rows of 16 lanes: row k gets the sum of a[k]
__device__ __forceinline__ float sum_rows(const float (&a)[4]) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    auto both = [](u32x2 v) {
        const unsigned x = v[0], y = v[1];
        return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
    };
    auto bits = [](float v) { return __builtin_bit_cast(unsigned, v); };
    const float lo = both(__builtin_amdgcn_permlane16_swap(bits(a[0]), bits(a[1]), false, false));
    const float hi = both(__builtin_amdgcn_permlane16_swap(bits(a[2]), bits(a[3]), false, false));
    return both(__builtin_amdgcn_permlane32_swap(bits(lo), bits(hi), false, false));
}

// lane j's states of a row of 4 * NS floats in LDS
template <int NS>
__device__ __forceinline__ void load_lane_states(const float* row, int j, float (&v)[NS]) {
    typedef float V __attribute__((ext_vector_type(kRun<NS>)));
#pragma unroll
    for (int s = 0; s < NS; s += kRun<NS>) {
        const V t = *(const V*)&row[state_of<NS>(j, s)];
#pragma unroll
        for (int e = 0; e < kRun<NS>; ++e) v[s + e] = t[e];
    }
}

// Frames [t0, t1) of one channel block: h goes from the state before t0 to the state after t1 - 1.  Y: results are stored;
// otherwise only the states move, and the sum of dt is returned.
template <typename T, int NS, bool Y>
__device__ __forceinline__ float scan_frames(const ScanParams<T>& p, const Channel<T, NS>& ch, int c0, int t0, int t1,
                                             float (&h)[NS], Tile<T, NS>* lds, float* steps) {
    typedef Tile<T, NS> Tl;
    typedef typename Unaligned<T, Tl::vec>::type Vec;
    constexpr int NP = Tl::NP, kMine = Tl::frames * NP / 256 > 0 ? Tl::frames * NP / 256 : 1;
    const int tid = threadIdx.x;
    const float bias = p.bias ? p.bias[ch.d] : 0.f, skip = p.Dskip ? p.Dskip[ch.d] : 0.f;
    const bool gate = Y && p.z.p;
    float sum = 0.f;

    // The next tile on its way: a thread brings one vector of a row of u, delta, z each (256 threads cover a tile) and kMine
    // elements of B and C.  A frame past t1 - 1 is that frame again; nothing reads it but for zeros in its place.  Addresses
    // are a base that all threads share (scalar arithmetic) plus an offset that a thread keeps.
    const int vrow = tid / Tl::vecs;
    int vcol = tid % Tl::vecs * Tl::vec, vn = min(Tl::vec, p.D / p.G - c0 - vcol);  // channels of the vector that the group has
    if (vn > 0 && vn < Tl::vec && vcol >= Tl::vec - vn) {  // reaches back over its neighbour's, which brings the same
        vcol -= Tl::vec - vn;
        vn = Tl::vec;
    }
    const int d0 = ch.g * (p.D / p.G) + c0 + vcol;
    constexpr int kRows = 256 / NP > Tl::frames ? Tl::frames : 256 / NP;  // rows of B and C that the block brings at once
    const int mrow = tid / NP % Tl::frames, mn = state_at(tid % NP, p.N);
    const float share = share_of(tid % NP, p.N, NP);
    const long long Bg = ch.g * p.Bg, Cg = ch.g * p.Cg;
    Vec nv[3];
    T nb[kMine], nc[kMine];
    auto at = [&](const Rows<const T>& r, long long off, int t, int row, int col) {
        const T* base = r.row(ch.b, t) + off;
        return (const T*)((const char*)base + (unsigned)(row * (int)r.rs + col) * (unsigned)sizeof(T));
    };
    auto fetch = [&](int t) {
        const int last = t1 - 1 - t;
        const int r = min(vrow, last);
        if (vn > 0) {
            nv[0] = load_some<T, Tl::vec>(at(p.u, 0, t, r, d0), vn);
            nv[1] = load_some<T, Tl::vec>(at(p.delta, 0, t, r, d0), vn);
            if (gate) nv[2] = load_some<T, Tl::vec>(at(p.z, 0, t, r, d0), vn);
        }
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int m = min(mrow + i * kRows, last);
            nb[i] = *at(p.Bm, Bg, t, m, mn);
            if (Y) nc[i] = *at(p.Cm, Cg, t, m, mn);
        }
    };
    auto put = [&](int t, Tl& to) {
        *(Vec*)&to.rows[0][vrow][vcol] = nv[0];
        *(Vec*)&to.rows[1][vrow][vcol] = nv[1];
        if (gate) *(Vec*)&to.rows[2][vrow][vcol] = nv[2];
        const bool whole = t + Tl::frames <= t1;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int e = tid + 256 * i;
            float vb = (float)nb[i], vc = Y ? (float)nc[i] * share : 0.f;
            if (!whole && t + e / NP >= t1) vb = vc = 0.f;
            if (256 * (i + 1) <= Tl::frames * NP || e < Tl::frames * NP) {
                to.maps[0][0][e] = vb;
                if (Y) to.maps[1][0][e] = vc;
            }
        }
    };
    const int lane = tid & 63, wave = tid >> 6, cl = wave * 16 + (lane & 15);  // the lane's channel of the block's 64
    const bool idle = __builtin_amdgcn_readfirstlane(c0 + wave * 16) >= p.D / p.G;  // a wave past the group's last channel only loads
    float* mine = steps + cl * Tl::steps;
    // results leave 16 bytes a lane: 16 channels of a frame on two or four lanes
    constexpr int kOut = 16 / Tl::vec, kOutRows = 64 / kOut;
    const int orow = lane / kOut, ocol = wave * 16 + lane % kOut * Tl::vec;
    const int on = min(Tl::vec, p.D / p.G - c0 - ocol);
    fetch(t0);
    int buf = 0;
    for (int t = t0; t < t1; t += Tl::frames, buf ^= 1) {
        Tl& tile = lds[buf];
        put(t, tile);
        __syncthreads();
        if (t + Tl::frames < t1) fetch(t + Tl::frames);
        if (idle) continue;
        // A lane's frames of the tile are j, j + 4, ...: their steps dt, which all four lanes of a channel need, go to LDS.
        constexpr int L = Tl::frames / 4;
        float uv[L], xv[L], zv[L], yv[L];
        {
            float dv[L];
#pragma unroll
            for (int i = 0; i < L; ++i) {
                uv[i] = (float)tile.rows[0][4 * i + ch.j][cl];
                dv[i] = (float)tile.rows[1][4 * i + ch.j][cl] + bias;
                if (gate) zv[i] = (float)tile.rows[2][4 * i + ch.j][cl];
            }
            if (p.softplus) {
#pragma unroll
                for (int i = 0; i < L; ++i) dv[i] = softplusf(dv[i]);
            }
            if (t + Tl::frames > t1) {  // frames past the end leave the state as it is: dt = 0
#pragma unroll
                for (int i = 0; i < L; ++i)
                    if (t + 4 * i + ch.j >= t1) uv[i] = dv[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < L; ++i) {
                xv[i] = dv[i] * uv[i];
                if (!Y) sum += dv[i];
                mine[4 * i + ch.j] = dv[i];
                if (NS < 4) mine[kBlockChannels * Tl::steps + 4 * i + ch.j] = xv[i];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();

        // F frames at a time, one unit ahead: while the chain through h runs for one unit, the exponentials of the next,
        // which depend on nothing, fill its gaps, C values come out of LDS, and the matrix unit makes dt u B: of four frames,
        // four outer products of 16 channels by 16 states.
        constexpr int F = NS >= 16 ? 1 : NS == 8 ? 2 : 4, units = Tl::frames / F;
        constexpr int XB = NS >= 16 ? 1 : 2;  // (16 states a lane: no registers for two)
        float cn[2][F][NS], decay[2][F][NS], out[4];
        f32x4 xb[XB][4][NS >= 4 ? NS / 4 : 1], dt4[2];
        auto inputs = [&](int i) {  // of frames 4 i ... 4 i + 3
            if constexpr (NS >= 4) {
#pragma unroll
                for (int m = 0; m < NS / 4; ++m) {
                    typedef float f32x16 __attribute__((ext_vector_type(16)));
                    const float bn = tile.maps[0][4 * i + ch.j][16 * m + (lane & 15)];
                    const f32x16 v = __builtin_amdgcn_mfma_f32_16x16x1f32(bn, xv[i], f32x16{}, 0, 0, 0);
#pragma unroll
                    for (int k = 0; k < 4; ++k) xb[i % XB][k][m] = f32x4{v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
                }
            } else {
                const f32x4 x4 = *(const f32x4*)&mine[kBlockChannels * Tl::steps + 4 * i];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float bn[NS];
                    load_lane_states<NS>(tile.maps[0][4 * i + k], ch.j, bn);
#pragma unroll
                    for (int s = 0; s < NS; ++s) xb[i % XB][k][0][s] = x4[k] * bn[s];
                }
            }
        };
        auto prepare = [&](int unit) {
            if (XB == 2 && unit * F % 4 == 0) inputs(unit * F / 4);
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const int k = unit * F + f;
                if (Y) load_lane_states<NS>(tile.maps[1][k], ch.j, cn[unit & 1][f]);
#pragma unroll
                for (int s = 0; s < NS; ++s) decay[unit & 1][f][s] = __builtin_amdgcn_exp2f(dt4[k / 4 % 2][k % 4] * ch.A2[s]);
            }
        };
        dt4[0] = *(const f32x4*)&mine[0];
        if (F == 4) dt4[1] = *(const f32x4*)&mine[4];
        prepare(0);
#pragma unroll
        for (int unit = 0; unit < units; ++unit) {
            if (unit * F == 16 && t + 16 >= t1) break;
            const int i = unit * F / 4;
            __builtin_amdgcn_sched_barrier(0);
            if (XB == 1 && unit * F % 4 == 0) inputs(i);
            if (unit + 1 < units) prepare(unit + 1);
            if ((unit + 2) * F % 4 == 0 && unit + 2 < units) dt4[(unit + 2) * F / 4 % 2] = *(const f32x4*)&mine[(unit + 2) * F];
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const int k = (unit * F + f) % 4;
                float o = 0.f;
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    h[s] = __builtin_fmaf(decay[unit & 1][f][s], h[s], xb[i % XB][k][s / 4][s % 4]);
                    if (Y) o = s ? __builtin_fmaf(cn[unit & 1][f][s], h[s], o) : cn[unit & 1][f][s] * h[s];
                }
                out[k] = o;
            }
            if (Y && (unit * F + F) % 4 == 0) yv[i] = sum_rows(out) + skip * uv[i];
        }
        __builtin_amdgcn_sched_barrier(0);
        if (Y) {
            if (gate) {
#pragma unroll
                for (int i = 0; i < L; ++i) yv[i] *= zv[i] * sigmoidf(zv[i]);
            }
            // the results take the place of the u that they came from (the same lane's, read above)
#pragma unroll
            for (int i = 0; i < L; ++i) tile.rows[0][4 * i + ch.j][cl] = (T)yv[i];
        }
        if (Y) {
            // a wave reads back what its own lanes wrote: LDS serves a wave's operations in their order
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int r = orow; r < Tl::frames; r += kOutRows)
                if (on > 0 && t + r < t1)
                    store_some<T, Tl::vec>(p.y.row(ch.b, t + r) + ch.g * (p.D / p.G) + c0 + ocol, *(const Vec*)&tile.rows[0][r][ocol], on);
        }
        // (the next tile goes to the other buffer; the one after it comes behind the next barrier)
    }
    if (!Y) sum += __shfl_xor(sum, 16), sum += __shfl_xor(sum, 32);
    return sum;
}

// zeros for the frames past a sequence's end
template <typename T, int NS>
__device__ __forceinline__ void zero_frames(const ScanParams<T>& p, const Channel<T, NS>& ch, int t0, int t1) {
    T* yb = p.y.row(ch.b, 0) + ch.d;
    if (ch.live)
        for (int t = t0 + ch.j; t < t1; t += kLanes) yb[(long long)t * p.y.rs] = (T)0.f;
}

// (4 * NS floats)
template <typename T, int NS>
__device__ __forceinline__ float* piece_states(const ScanParams<T>& p, const Channel<T, NS>& ch, int piece) {
    return p.ws_h + (((long long)ch.b * (p.pieces - 1) + piece) * p.D + ch.d) * (kLanes * NS);
}
template <typename T, int NS>
__device__ __forceinline__ float* piece_sum(const ScanParams<T>& p, const Channel<T, NS>& ch, int piece) {
    return p.ws_s + ((long long)ch.b * (p.pieces - 1) + piece) * p.D + ch.d;
}

// The sequence that the block at place z takes: by falling length, every second round of `order` places backwards.  A round is
// what fills the CUs once, so that the block that comes second to a CU has the shorter sequence the longer the first one's
// is.  (32 utterances of 172 to 861 frames, D 1024: 94 - 98 us; as they come 118.)
__device__ __forceinline__ int place_to_sequence(const int32_t* lengths, int B, int Tmax, int order, int z, int* found) {
    const int round = z / order, first = round * order;
    const int rank = round & 1 ? first + min(order, B - first) - 1 - (z - first) : z;
    for (int i = threadIdx.x; i < B; i += 256) {
        const int mine = seq_frames(lengths, i, Tmax);
        int before = 0;
        for (int k = 0; k < B; ++k) {
            const int other = seq_frames(lengths, k, Tmax);
            before += other > mine || (other == mine && k < i);
        }
        if (before == rank) *found = i;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(*found);
}

// A state after frames whose decays multiply to 2^e, none of them 0 where e is finite: zero and infinities stay what they are
// however far the factor by itself overflows or underflows, and what the product can hold goes through two halves that float32
// can hold too.
__device__ __forceinline__ float decayed(float h, float e) {
    constexpr int kZero = 0x060, kInf = 0x204, kFinite = 0x1f8;  // classes of both signs
    const float half = __builtin_amdgcn_exp2f(0.5f * e);
    const int kept = __builtin_amdgcn_classf(e, kFinite) ? kZero | kInf : kZero;
    return __builtin_amdgcn_classf(h, kept) ? h : h * half * half;
}

// Grid (channel blocks of all groups, pieces, sequences).  FIRST: piece 0 from the given state, results and all; every other
// piece but the last from a zero state, for the state it leaves behind.  Second launch: the pieces from 1 on, each from the
// state before it, which it puts together from what the first launch left.
template <typename T, int NS, bool FIRST>
__global__ __launch_bounds__(256) void scan_kernel(ScanParams<T> p) {
    __shared__ __align__(16) Tile<T, NS> lds[2];
    __shared__ __align__(16) float steps[(NS < 4 ? 2 : 1) * kBlockChannels * Tile<T, NS>::steps];
    Channel<T, NS> ch;
    const int g = blockIdx.x / p.blocks_per_group, cb = blockIdx.x % p.blocks_per_group;
    const int piece = FIRST ? blockIdx.y : blockIdx.y + 1;
    __shared__ int found;
    for (int z = blockIdx.z; z < p.B; z += gridDim.z) {
        const int b = FIRST && p.order ? place_to_sequence(p.lengths, p.B, p.Tmax, p.order, z, &found) : z;
        const int c0 = cb * kBlockChannels;
        ch.init(p, b, g, c0 + threadIdx.x / 64 * 16 + threadIdx.x % 16, threadIdx.x % 64 / 16);
        const long long first = (long long)piece * p.piece;
        const int t0 = (int)min(first, (long long)p.Tmax), te = (int)min(first + p.piece, (long long)p.Tmax);
        const int t1 = min(te, ch.len);
        const bool last = ch.len <= te;  // no live frame behind this piece
        float h[NS];
        if (FIRST && piece > 0) {
            if (!last) {
#pragma unroll
                for (int s = 0; s < NS; ++s) h[s] = 0.f;
                const float sum = scan_frames<T, NS, false>(p, ch, c0, t0, t1, h, lds, steps);
                if (ch.live) {
                    store_my_states(piece_states(p, ch, piece), kLanes * NS, ch.j, h);
                    if (ch.j == 0) *piece_sum(p, ch, piece) = sum;
                }
            }
        } else if (FIRST || t0 < ch.len) {
            if (FIRST) {
                load_state<true>(p.state_in ? p.state_in + ((long long)b * p.D + ch.d) * p.N : nullptr, p.N, ch.j, h);
            } else {
                load_my_states<false>(piece_states(p, ch, 0), kLanes * NS, ch.j, h);
                constexpr int kBatch = NS >= 16 ? 2 : 8;  // pieces whose loads are in flight together
                for (int k = 1; k < piece; k += kBatch) {
                    float sum[kBatch], end[kBatch][NS];
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        const int at = min(k + i, piece - 1);
                        load_my_states<false>(piece_states(p, ch, at), kLanes * NS, ch.j, end[i]);
                        sum[i] = *piece_sum(p, ch, at);
                    }
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                        if (k + i < piece)
#pragma unroll
                            for (int s = 0; s < NS; ++s) h[s] = decayed(h[s], sum[i] * ch.A2[s]) + end[i][s];
                }
            }
            if (t0 < t1) scan_frames<T, NS, true>(p, ch, c0, t0, t1, h, lds, steps);
            if (last) {
                if (p.state_out && ch.live) store_my_states(p.state_out + ((long long)b * p.D + ch.d) * p.N, p.N, ch.j, h);
            } else if (FIRST && ch.live) {
                store_my_states(piece_states(p, ch, 0), kLanes * NS, ch.j, h);
            }
        }
        if (!FIRST || piece == 0) zero_frames(p, ch, max(t0, ch.len), te);
        __syncthreads();  // the next sequence starts over with the first buffer
    }
}

// a[k] of four values, each spread over a quad's four lanes: lane k gets the sum of a[k]
__device__ __forceinline__ float sum_quad(const float (&a)[4], int j) {
    const bool o1 = j & 1, o2 = j & 2;
    const float x = (o1 ? a[1] : a[0]) + quad<0xB1>(o1 ? a[0] : a[1]);
    const float y = (o1 ? a[3] : a[2]) + quad<0xB1>(o1 ? a[2] : a[3]);
    return (o2 ? y : x) + quad<0x4E>(o2 ? x : y);
}

// A few frames of many sequences (decode steps): no LDS, no barrier; what counts is the state, read and written once.  Here
// the four lanes of a channel stand side by side, so that a wave's states are one piece of memory, and a quad of lanes has Q
// channels: with Q = 4, lane j brings u, delta and z of the quad's channel j, makes its step and hands it around, and B and C
// are loaded once for the four (a wave's memory instructions, not its bytes, are what a call of 16 states waits for: 14
// instead of 32 for 64 channels).  With 8 and more states a lane, one channel fills the registers.  Grid
// (channels, sequences): a block keeps its channels' A and walks sequences.
template <int NS>
constexpr int kQuadChannels = NS <= 4 ? 4 : 1;

template <typename T, int NS>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanParams<T> p) {
    constexpr int Q = kQuadChannels<NS>;
    const int j = threadIdx.x & (kLanes - 1), c0 = (blockIdx.x * 64 + (threadIdx.x >> 2)) * Q, Dg = p.D / p.G;
    if (__builtin_amdgcn_readfirstlane(c0) >= p.D) return;
    const int mine = Q == 4 ? c0 + j : c0, d = min(mine, p.D - 1);  // the channel whose u, delta, z and y are this lane's
    const bool live = mine < p.D, together = p.G == 1 || (Q == 4 && Dg % 4 == 0);
    int dk[Q], gk[Q];
    float A2[Q][NS];
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        dk[k] = min(c0 + k, p.D - 1);
        gk[k] = p.G == 1 ? 0 : dk[k] / Dg;
        load_decays<false>(p, dk[k], j, A2[k]);
    }
    const float bias = p.bias ? p.bias[d] : 0.f, skip = p.Dskip ? p.Dskip[d] : 0.f;
    for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
        const int len = seq_frames(p.lengths, b, p.Tmax);
        const long long state = (long long)b * p.D * p.N;
        float h[Q][NS];
#pragma unroll
        for (int k = 0; k < Q; ++k) load_state<false>(p.state_in ? p.state_in + state + dk[k] * p.N : nullptr, p.N, j, h[k]);
        for (int t = 0; t < p.Tmax; ++t) {
            float v = 0.f;
            if (t < len) {
                const float u = (float)p.u.row(b, t)[d], raw = (float)p.delta.row(b, t)[d] + bias;
                const float z = p.z.p ? (float)p.z.row(b, t)[d] : 0.f;
                float bn[NS], cn[NS], out[Q];
                auto maps = [&](int k) {
                    load_my_states<false>(p.Bm.row(b, t) + gk[k] * p.Bg, p.N, j, bn);
                    load_my_states<false>(p.Cm.row(b, t) + gk[k] * p.Cg, p.N, j, cn);
                };
                maps(0);
                const float dt = p.softplus ? softplusf(raw) : raw, x = dt * u;
#pragma unroll
                for (int k = 0; k < Q; ++k) {
                    const float dtk = Q == 4 ? quad_lane(dt, k) : dt, xk = Q == 4 ? quad_lane(x, k) : x;
                    if (k && !together) maps(k);
                    out[k] = 0.f;
#pragma unroll
                    for (int s = 0; s < NS; ++s) {
                        const float hn = __builtin_fmaf(__builtin_amdgcn_exp2f(dtk * A2[k][s]), h[k][s], xk * bn[s]);
                        h[k][s] = state_of<NS>(j, s) < p.N ? hn : 0.f;
                        out[k] += cn[s] * h[k][s];
                    }
                }
                if constexpr (Q == 4) {
                    v = sum_quad(out, j);
                } else {
                    v = out[0] + quad<0xB1>(out[0]);
                    v += quad<0x4E>(v);
                }
                v += skip * u;
                if (p.z.p) v *= z * sigmoidf(z);
            }
            if (live && (Q == 4 || j == 0)) p.y.row(b, t)[d] = (T)v;
        }
        if (p.state_out) {
#pragma unroll
            for (int k = 0; k < Q; ++k)
                if (c0 + k < p.D) store_my_states(p.state_out + state + dk[k] * p.N, p.N, j, h[k]);
        }
    }
}

constexpr int kStepBlocks = 2048;  // of the step kernel: eight to a CU, each then walks B * D / 64 / 2048 sequences

// Calls of up to this many frames take the step kernel, whose frames cost their own memory instructions; the other one computes
// 16 at a time (D 1024, 64 / 512 sequences: 8 frames 12.2 / 40 us against 14.5 / 91; 16 frames of 64 sequences 21.6 against 14.5).
constexpr int kStepFrames = 8;

// Pieces that the frames of each sequence are cut into: as many as give every SIMD two waves (which is what the registers
// hold), of 32 frames at least.  The work doubles, so two pieces gain nothing (1 x 8192 frames, D 1024: 109 us with waves for
// one a SIMD, 76 for two, 88 - 90 for three or four; 8 x 861: 71 cut in four, 87 whole; 12 x 861: 87 whole, 92 in three), and a
// launch takes what 30 frames take (1 x 861, D 256: 17.9 us in 27 pieces of 32, 21.7 in 14 of 64).
static int scan_pieces(int B, int T, int D, int G) {
    const long long waves = (long long)B * G * ((D / G + 15) / 16);
    if (waves >= 1024 || T < 96) return 1;
    long long n = 2048 / waves;
    n = std::min<long long>(n, (T + 31) / 32);
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
    s.piece = round_up((a->T + s.pieces - 1) / s.pieces, 32);
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
        const int x = (p.D + 64 * kQuadChannels<NS> - 1) / (64 * kQuadChannels<NS>);
        const dim3 grid(x, (unsigned)std::min(p.B, std::max(1, std::min(65535, kStepBlocks / x))));
        hipLaunchKernelGGL((scan_step_kernel<T, NS>), grid, dim3(256), 0, stream, p);
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
    for (const void* f : {(const void*)a->A, (const void*)a->Dskip, (const void*)a->delta_bias, (const void*)a->state_in,
                          (const void*)a->state_out, (const void*)a->lengths})
        if (int rc = check_aligned(who, f, 4)) return rc;
    if (a->Bg_stride < 0 || a->Cg_stride < 0) {
        set_error("%s: group strides must be >= 0", who);
        return MV_EINVAL;
    }
    const struct {
        const char* name;
        const mv_rows* r;
    } ins[] = {{"u", &a->u}, {"delta", &a->delta}, {"z", &a->z}, {"Bm", &a->Bm}, {"Cm", &a->Cm}};
    for (const auto& in : ins)
        if (in.r != &a->z || in.r->ptr)
            if (int rc = check_rows(who, in.name, *in.r, a->T, a->dtype)) return rc;
    if (int rc = check_output_rows(who, a->y, a->B, a->T, a->D, a->dtype)) return rc;
    auto rows = [&](const mv_rows& r, long long channels) { return Span(r, channels, a->B, a->T, a->dtype); };
    const Span y = rows(a->y, a->D), before(a->state_in, 4 * states), after(a->state_out, 4 * states);
    auto apart = [&](const Span& out, const char* what, std::initializer_list<Span> states_of_call) {
        if (int rc = check_overlaps(who, out, what, states_of_call)) return rc;
        if (int rc = check_overlaps(who, out, what, {rows(a->u, a->D), rows(a->delta, a->D), rows(a->z, a->D), {a->A, 4ll * a->D * a->N},
                                                     {a->Dskip, 4ll * a->D}, {a->delta_bias, 4ll * a->D}, {a->lengths, 4ll * a->B}}))
            return rc;
        for (auto [m, step] : {std::pair<mv_rows, int64_t>{a->Bm, a->Bg_stride}, {a->Cm, a->Cg_stride}}) {
            // all groups and what lies between them; only what touches that is looked at group by group
            if (a->G > 1 && step > 1ll << 38) continue;  // (no device's memory, and no product of 64 bits)
            int rc = check_overlaps(who, out, what, {rows(m, a->G == 1 ? a->N : (a->G - 1) * step + a->N)});
            if (!rc) continue;
            if (a->G == 1 || step == a->N) return rc;
            for (int g = 0; g < a->G; ++g, m.ptr = (char*)m.ptr + step * (int64_t)dtype_size(a->dtype))
                if ((rc = check_overlaps(who, out, what, {rows(m, a->N)}))) return rc;
        }
        return MV_OK;
    };
    if (int rc = apart(y, "y", {before, after})) return rc;
    if (int rc = apart(after, "state_out", {})) return rc;
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
                        (float*)((char*)workspace + plan.h_bytes), a->B, a->T, a->D, a->N, a->G, a->delta_softplus, 0,
                        (a->D / a->G + kBlockChannels - 1) / kBlockChannels, plan.piece, plan.pieces};
        if (a->lengths && plan.pieces == 1 && a->B <= 256) p.order = std::max(1, 256 / (a->G * p.blocks_per_group));
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
